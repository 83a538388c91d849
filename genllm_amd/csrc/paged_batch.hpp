// paged_batch.hpp -- what the kernels of paged_attention_batch share: the launch's
// parameters, how a padded batch of unlike lengths is divided among workgroups, the
// pages that a row tile visits, and the form that takes one key after another.
#pragma once

#include <climits>

#include "common.hpp"

namespace genllm {

struct BatchAttn {
    const int32_t* n_cached = nullptr;  // [B]
    const int32_t* q_lens = nullptr;    // [B], or null: S each
    const uint16_t* q = nullptr;
    int64_t q_batch = 0, q_tok = 0, q_head = 0;  // elements
    const char* k_pool = nullptr;
    const char* v_pool = nullptr;
    int64_t k_block = 0, v_block = 0;                    // bytes
    int32_t k_tok = 0, k_head = 0, v_tok = 0, v_head = 0;  // bytes within a block
    const uint8_t* k_scales = nullptr;  // [blocks][Hkv], 2^(byte - 127); null with 16-bit pools
    const uint8_t* v_scales = nullptr;
    const int32_t* k_ids = nullptr;
    const int32_t* v_ids = nullptr;
    int64_t k_ids_row = 0, v_ids_row = 0;
    uint16_t* out = nullptr;
    int64_t o_batch = 0, o_tok = 0, o_head = 0;
    int32_t B = 0, S = 0, Hq = 0, Hkv = 0, G = 0;
    int32_t blocks = 0;    // ids outside [0, blocks) are no pages: NaN for the rows that see them
    int32_t capacity = 0;  // tokens that a row of the tables holds
    int32_t window = 0;    // keys a query sees up to itself; kNoWindow: all
    int32_t sinks = 0;     // first tokens that stay visible behind a window
    int32_t causal = 1;
    float c = 0.0f;        // scale * log2(e), at least FLT_MIN
    // division of the work
    int32_t tiles_max = 1; // row tiles of an entry at most
    int32_t target = 1;    // workgroups to fill the GPU with
    int32_t least = 1;     // steps that a split takes at least
    int32_t can_split = 0; // else every row tile has one workgroup
    int32_t paired = 0;    // row tiles in the order last, last but one, .., then first, second, ..
    float* partial = nullptr;  // headers [unit], then o [workgroup][tile row][D], then {m, l} [workgroup][tile row]
    int32_t slots = 0;         // workgroups that the partials have room for
};

constexpr int32_t kNoWindow = 1 << 30;
constexpr int kDecodeStep = 2, kPrefillStep = 4;  // pages of a step

// Keys in pages: the first `sink_pages` of a sequence, then from sink_pages + skip on.
struct Span {
    int sink_pages, skip, pages;
    __device__ __forceinline__ int page(int j) const { return j + (j >= sink_pages ? skip : 0); }
};

// The pages that hold a key for some query of positions first_pos.. (negative: before
// the sequence) with keys before `end`.
__device__ __forceinline__ Span span_of(const BatchAttn& p, int first_pos, int end) {
    const int total = (end + kPage - 1) / kPage;
    const int w0 = max(0, first_pos - p.window + 1) / kPage;
    const int sinks = (min(p.sinks, end) + kPage - 1) / kPage;
    if (w0 <= sinks) return {total, 0, total};
    return {sinks, w0 - sinks, total - (w0 - sinks)};
}

// Quotients of numbers from 0 on, rounded down, by a divisor that the lanes have in common:
// by its reciprocal in fp32, once more for what the first (within 2^-21 of itself) leaves,
// and a step up or down.  (The compiler's integer division takes about 40 instructions; a
// plan of 32 row tiles took 8800 cycles with it.)
struct Divisor {
    int d;
    float r;
    __device__ __forceinline__ explicit Divisor(int d_) : d(d_), r(__builtin_amdgcn_rcpf(float(d_))) {}
    __device__ __forceinline__ int operator()(int x) const {
        int q = int(float(x) * r), rest = x - q * d;
        const int more = int(float(rest) * r);
        q += more, rest -= more * d;
        return q + (rest >= d ? 1 : 0) - (rest < 0 ? 1 : 0);
    }
};

struct Entry {
    int n, ql;  // keys cached, queries
};
__device__ __forceinline__ Entry entry_of(const BatchAttn& p, int b) {
    const int n = p.n_cached[b], ql = p.q_lens ? p.q_lens[b] : p.S;
    return {min(max(n, 0), p.capacity), min(max(ql, 0), p.S)};
}

// Positions of a row tile's first and last query, and how many keys it has: up to its last
// query's own.
struct TileKeys {
    int first, end;
};
template <int ROWS>
__device__ __forceinline__ TileKeys tile_keys(const BatchAttn& p, const Entry& e, int tile) {
    if (!p.causal) return {e.n - 1, e.n};
    const int rows = e.ql * p.G, at = e.n - e.ql;
    const Divisor by_g(p.G);
    return {at + by_g(tile * ROWS), max(min(at + by_g(min((tile + 1) * ROWS, rows) - 1) + 1, e.n), 0)};
}

// The work is divided by units, row tile `tile` of entry b being unit b * tiles_max + tile:
// a unit has steps of STEP pages for each kv head, and its splits share them.
template <int ROWS, int STEP>
__device__ __forceinline__ bool unit_steps(const BatchAttn& p, const Entry& e, int tile, int& steps) {
    if (tile * ROWS >= e.ql * p.G) return false;  // no such tile
    const TileKeys k = tile_keys<ROWS>(p, e, tile);
    steps = (span_of(p, k.first, k.end).pages + STEP - 1) / STEP;
    return true;
}

struct Work {
    int b, tile, sp, h, ns;
    int unit, base;  // the unit's first workgroup
    Entry e;
};

// The sums of x over the lanes up to this one, all of them active
__device__ __forceinline__ int wave_sums(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // from the lanes 1, 2, 4, 8 before in a row of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // a row's last to the next row
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // the second row's last to the last two
    return x;
}

constexpr int kQuanta = 4;  // quanta tried: 1, 1 1/4, 1 1/2, 1 3/4 times the share

// What workgroup w does; false: nothing.  Without splits, entry by entry, [tile][kv head],
// the last tiles, which have the most keys, first.  With them all units of the batch are
// cut into pieces of as many steps as a target of workgroups leaves for each: the waves of
// every workgroup come to the same sum (a whole number below 2^53, exact in whatever
// order), and find theirs by the pieces before it, [unit][split][kv head].  With 8 kv heads
// those of one head run on one XCD.
template <int ROWS, int STEP>
__device__ __forceinline__ bool find_work(const BatchAttn& p, int w, Work& r) {
    const int lane = threadIdx.x & 63;
    const Divisor by_heads(p.Hkv), by_tiles(p.tiles_max);
    if (!p.can_split) {
        const int rest = by_heads(w), b = by_tiles(rest), rank = rest - b * p.tiles_max;
        if (b >= p.B) return false;
        r.b = __builtin_amdgcn_readfirstlane(b);
        r.e = entry_of(p, r.b);
        r.h = __builtin_amdgcn_readfirstlane(w - rest * p.Hkv);
        const int tiles = (r.e.ql * p.G + ROWS - 1) / ROWS, half = (tiles + 1) / 2;
        if (rank >= tiles) return false;
        r.tile = __builtin_amdgcn_readfirstlane(p.paired && rank >= half ? rank - half : tiles - 1 - rank);
        r.ns = 1, r.sp = 0, r.unit = 0, r.base = w;
        return true;
    }
    const int units = p.B * p.tiles_max;
    // what lane u % 64 knows of unit u, the first 64 once and for all
    struct Unit {
        int steps = -1;  // none: the entry has no such tile
        Entry e{0, 0};
    };
    const auto unit = [&](int u) {
        Unit r;
        if (u < units) {
            const int b = by_tiles(u);
            r.e = entry_of(p, b);
            if (!unit_steps<ROWS, STEP>(p, r.e, u - b * p.tiles_max, r.steps)) r.steps = -1;
        }
        return r;
    };
    const Unit first = unit(lane);
    int64_t mine = max(first.steps, 0);
    for (int u = lane + 64; u < units; u += 64) mine += max(unit(u).steps, 0);
    // of at most 2^48 in a lane, exact
    const double sum = double(__builtin_amdgcn_readlane(wave_sums(int(mine & 0xffffff)), 63)) +
                       (units > 64 ? double(__builtin_amdgcn_readlane(wave_sums(int(mine >> 24)), 63)) * (1 << 24) : 0.0);
    const double share = ceil(sum * p.Hkv * (1.0 / p.target));  // every workgroup's the same, whatever the last bit is
    int quantum = max(p.least, __builtin_amdgcn_readfirstlane(int(fmin(share, double(1 << 28)))));
    // pieces that are no whole quantum may leave a few workgroups more than the target,
    // which would run after all the others: up to twice the quantum where that avoids it
    if (STEP == kPrefillStep && units * p.Hkv <= p.target) {
        int chosen = 2 * quantum;
#pragma unroll
        for (int k = kQuanta - 1; k >= 0; --k) {
            const int q = quantum * (kQuanta + k) / kQuanta;
            const Divisor by(q);
            int pieces = first.steps < 0 ? 0 : max(1, by(first.steps + q - 1));
            for (int u = lane + 64; u < units; u += 64) {
                const int steps = unit(u).steps;
                pieces += steps < 0 ? 0 : max(1, by(steps + q - 1));
            }
            if (__builtin_amdgcn_readlane(wave_sums(pieces), 63) * p.Hkv <= p.target) chosen = q;
        }
        quantum = chosen;
    }
    const Divisor by_quantum(quantum);
    int base = 0;
    for (int u0 = 0; u0 < units; u0 += 64) {
        const Unit at = u0 == 0 ? first : unit(u0 + lane);
        const Entry e = at.e;
        const int ns = at.steps < 0 ? 0 : max(1, by_quantum(at.steps + quantum - 1));
        const int upto = wave_sums(ns * p.Hkv);
        const unsigned long long hit = __ballot(w >= base + upto - ns * p.Hkv && w < base + upto);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            r.unit = u0 + src;
            r.b = __builtin_amdgcn_readfirstlane(by_tiles(r.unit)), r.tile = r.unit - r.b * p.tiles_max;
            r.ns = __builtin_amdgcn_readlane(ns, src);
            r.base = base + __builtin_amdgcn_readlane(upto, src) - r.ns * p.Hkv;
            r.e = {__builtin_amdgcn_readlane(e.n, src), __builtin_amdgcn_readlane(e.ql, src)};
            r.sp = __builtin_amdgcn_readfirstlane(by_heads(w - r.base));
            r.h = w - r.base - r.sp * p.Hkv;
            return true;
        }
        base += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// What the merge needs of a unit, left in the workspace by the unit's first workgroup (one
// without rows has none, nor needs it).
struct Header {
    int base, ns;
};

// What a row sees: keys up to `pos`, of those from `from` on and those before p.sinks.
struct Sight {
    int pos, from;
    bool any;  // the row has a key at all
    __device__ __forceinline__ bool operator()(const BatchAttn& p, int t) const { return t <= pos && (t >= from || t < p.sinks); }
};
__device__ __forceinline__ Sight sight_of(const BatchAttn& p, const Entry& e, int query) {
    const int pos = p.causal ? min(e.n - e.ql + query, e.n - 1) : e.n - 1;
    return {pos, pos - p.window + 1, pos >= 0};
}

// 2^(byte - 127), NaN for 255
__device__ __forceinline__ float scale_value(int byte) {
    return byte == 255 ? __builtin_nanf("") : __uint_as_float(byte ? uint32_t(byte) << 23 : 0x00400000u);
}
// 2^e for e from -126 to 127, 2^-126 below
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(uint32_t(max(e, -126) + 127) << 23); }

// behind the headers, two ints each, in whole 16 bytes
__device__ __forceinline__ float* partial_rows(const BatchAttn& p) { return p.partial + (2 * int64_t(p.B) * p.tiles_max + 3 & ~int64_t(3)); }

__device__ __forceinline__ void put_header(const BatchAttn& p, const Work& w) {
    if (p.can_split && int(blockIdx.x) == w.base && threadIdx.x == 0) reinterpret_cast<Header*>(p.partial)[w.unit] = {w.base, w.ns};
}

// A page as the lane that looked it up holds it.  The scales' bytes are not looked at
// before they are needed: they arrive with the page's rows, not ahead of them.
struct PageInfo {
    int kid = -1, vid = -1;  // block ids; -1, -1: no page; -1, -2: an id that is none
    int kb = 127, vb = 0;    // bytes of the scales; no page: the least, which raises no reference
};
template <bool Q8>
__device__ __forceinline__ PageInfo page_info(const BatchAttn& p, int b, int h, int page, bool there) {
    PageInfo r;
    if (there) {
        r.kid = p.k_ids[b * p.k_ids_row + page];
        r.vid = p.v_ids[b * p.v_ids_row + page];
        if (unsigned(r.kid) >= unsigned(p.blocks) || unsigned(r.vid) >= unsigned(p.blocks)) r.kid = -1, r.vid = -2;
        if constexpr (Q8) {
            r.kb = p.k_scales[int64_t(max(r.kid, 0)) * p.Hkv + h];
            r.vb = p.v_scales[int64_t(max(r.vid, 0)) * p.Hkv + h];
        }
    }
    return r;
}
// What takes a page's scores to log2 units; NaN where an id or a scale is none.
template <bool Q8>
__device__ __forceinline__ float score_factor(const BatchAttn& p, int vid, int kb, int vb) {
    if (vid == -2 || (Q8 && (kb == 255 || vb == 255))) return __builtin_nanf("");
    return Q8 ? fmaxf(scale_value(kb) * p.c, __FLT_MIN__) : p.c;
}

// Waits for the loads of x and makes the compiler take it from here on as what it is: no
// load's result, whose first use inside a loop would wait for the loads issued there.
__device__ __forceinline__ void landed(uint4& x) { __asm__ volatile("" : "+v"(x.x), "+v"(x.y), "+v"(x.z), "+v"(x.w)); }

// Two e4m3 codes (the low or the high half of w) as a packed pair of elements
template <bool F16, bool kHigh>
__device__ __forceinline__ uint32_t f8_pair(uint32_t w, float scale) {
    if constexpr (F16)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, kHigh));
    else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, kHigh));
}
// eight codes as an MFMA operand
template <bool F16>
__device__ __forceinline__ uint4 f8_octet(uint32_t w0, uint32_t w1, float s0, float s1) {
    return make_uint4(f8_pair<F16, false>(w0, s0), f8_pair<F16, true>(w0, s0), f8_pair<F16, false>(w1, s1), f8_pair<F16, true>(w1, s1));
}

// V's pages are taken relative to a reference scale 2^ref, at least a 64th of the largest so
// far.  That is exact for a page at most 15 binades below it: a code's last bit, 2^-9, is
// fp16's, 2^-24.  Where there are lower ones, or sums might leave fp32's range, rows are
// computed by exact_keys in the end: the scale of another page, of keys that a row may not
// even see, costs no row its precision.  Pages of zeros alone, which have the least scale, do
// not count.  low: a lane's least; next(i): the i-th page, -1 behind the last.
constexpr int kScaleReach = 15, kMostScale = 90;
struct ScaleRange {
    int low = 1 << 20;
    __device__ __forceinline__ void add(const PageInfo& info) { low = info.kid >= 0 ? min(low, info.vb - 127) : low; }
    template <int D, class Next>
    __device__ __forceinline__ bool left(const BatchAttn& p, int b, int h, int ref, const Next& next) const {
        if (ref == INT_MIN) return false;
        if (ref > kMostScale) return true;
        if (!__any(low < ref - kScaleReach)) return false;
        const int lane = threadIdx.x & 63;
        for (int i = 0;; ++i) {
            const int page = next(i);
            if (page < 0) return false;
            const PageInfo info = page_info<true>(p, b, h, page, true);
            if (info.kid < 0 || info.vb - 127 >= ref - kScaleReach) continue;
            if (info.vb - 127 > -100) return true;
            uint32_t any = 0;
            const char* const row = p.v_pool + info.vid * p.v_block + int64_t(h) * p.v_head + int64_t(lane >> 2) * p.v_tok;
            for (int d = 16 * (lane & 3); d < D; d += 64) {
                const uint4 u = *reinterpret_cast<const uint4*>(row + d);
                any |= u.x | u.y | u.z | u.w;
            }
            if (__any((any & 0x7f7f7f7f) != 0)) return true;
        }
    }
};

// One key after another, in fp32, each row with only the keys it sees: what a wave runs
// again whose tiles came out NaN or infinite.  (In the tiles a key that a row does not
// see meets a probability of zero, and 0 x NaN is NaN.)  The lane's row is lane % 16;
// acc: dims 16 db + 4 g + i, in V's own units; m in log2 units.  next(i): the i-th page
// of the wave, or -1 at the end.
template <int D, bool F16, bool Q8, typename Next>
__device__ __forceinline__ void exact_keys(const BatchAttn& p, int b, int h, const uint16_t* qrow, const Sight& see, const Next& next,
                                           f32x4_t (&acc)[D / 16], float& m, float& l) {
    using E = Elem<F16>;
    const int g = (threadIdx.x & 63) >> 4;
    m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) acc[db] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0;; ++i) {
        const int page = next(i);
        if (page < 0) break;
        const PageInfo info = page_info<Q8>(p, b, h, page, true);
        const bool there = info.kid >= 0;
        const char* const kb = p.k_pool + (there ? info.kid : 0) * p.k_block + int64_t(h) * p.k_head;
        const char* const vb = p.v_pool + (there ? info.vid : 0) * p.v_block + int64_t(h) * p.v_head;
        const float kf = score_factor<Q8>(p, info.vid, info.kb, info.vb), vs = Q8 ? scale_value(info.vb) : 1.0f;
        for (int j = 0; j < kPage; ++j) {
            const int t = page * kPage + j;
            const bool vis = see(p, t);
            if (!__any(vis)) continue;
            float x = 0.0f;
#pragma unroll 1
            for (int d = 8 * g; d < D; d += 32) {
                const uint4 qq = *reinterpret_cast<const uint4*>(qrow + d);
                const uint32_t qw[4] = {qq.x, qq.y, qq.z, qq.w};
                uint32_t kw[4] = {0, 0, 0, 0};
                if (there) {
                    if constexpr (Q8) {
                        const uint2 u = *reinterpret_cast<const uint2*>(kb + int64_t(j) * p.k_tok + d);
                        const uint4 o = f8_octet<F16>(u.x, u.y, 1.0f, 1.0f);
                        kw[0] = o.x, kw[1] = o.y, kw[2] = o.z, kw[3] = o.w;
                    } else {
                        const uint4 o = *reinterpret_cast<const uint4*>(kb + int64_t(j) * p.k_tok + 2 * d);
                        kw[0] = o.x, kw[1] = o.y, kw[2] = o.z, kw[3] = o.w;
                    }
                }
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    x = __builtin_fmaf(E::lo(qw[w]), E::lo(kw[w]), x);
                    x = __builtin_fmaf(E::hi(qw[w]), E::hi(kw[w]), x);
                }
            }
            x += __shfl_xor(x, 16);
            x += __shfl_xor(x, 32);
            x *= kf;
            const float mn = vis ? __builtin_elementwise_maximum(m, x) : m;
            const float alpha = m == -INFINITY ? 0.0f : mn == m ? 1.0f : exp2_fast(m - mn);
            const float e = mn == -INFINITY ? 0.0f : exp2_fast(x - mn);
            if (vis) l = __builtin_fmaf(l, alpha, e);
#pragma unroll
            for (int db = 0; db < D / 16; ++db) {
                float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (there) {
                    if constexpr (Q8) {
                        const uint32_t u = *reinterpret_cast<const uint32_t*>(vb + int64_t(j) * p.v_tok + 16 * db + 4 * g);
                        // as read back, in fp16 (a code's value fits whole), then its scale
                        const uint32_t lo = f8_pair<true, false>(u, 1.0f), hi = f8_pair<true, true>(u, 1.0f);
                        v[0] = Elem<true>::lo(lo) * vs, v[1] = Elem<true>::hi(lo) * vs, v[2] = Elem<true>::lo(hi) * vs, v[3] = Elem<true>::hi(hi) * vs;
                    } else {
                        const uint2 u = *reinterpret_cast<const uint2*>(vb + int64_t(j) * p.v_tok + 2 * (16 * db + 4 * g));
                        v[0] = E::lo(u.x), v[1] = E::hi(u.x), v[2] = E::lo(u.y), v[3] = E::hi(u.y);
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[db][k] = vis ? __builtin_fmaf(e, v[k], acc[db][k] * alpha) : acc[db][k];
            }
            m = mn;
        }
    }
}

int launch_batch_decode(const BatchAttn& p, int head_dim, bool f16, hipStream_t stream);
int launch_batch_prefill(const BatchAttn& p, int tile_rows, int head_dim, bool f16, hipStream_t stream);  // tiles of 64 or 128 rows

// Which kernel a call runs and how its work is divided at most.
struct BatchPlan {
    bool decode;
    int rows;           // of a tile
    int step;           // pages of a step
    int64_t tiles_max;  // row tiles of an entry and kv head at most
    int64_t tiles;      // of the batch
    int64_t slots;  // workgroups at most; as many partials where can_split
    int target, least;
    bool can_split, paired;
};

}  // namespace genllm
