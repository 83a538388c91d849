// batch_work.hpp -- how a padded batch of unlike lengths is divided among workgroups:
// the launch's parameters, the pages that a row tile visits, what a workgroup does
// (device), and the sizes of a call (host).
//
// No HIP header is needed here, and of HIP only lanes, moves between them, ballots and
// min and max: a program on the host that stands in for those can run it.  kPage comes
// from common.hpp, or likewise.
#pragma once

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstddef>
#include <cstdint>

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
constexpr int kDecodeRows = 16;                   // of a tile; a prefill tile has 64 or 128
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
    // in halves: with few rows one unit alone has up to 2^25 steps, a lane's share of the units up to 2^41
    const double sum = double(__builtin_amdgcn_readlane(wave_sums(int(mine & 0xffffff)), 63)) +
                       double(__builtin_amdgcn_readlane(wave_sums(int(mine >> 24)), 63)) * (1 << 24);
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

constexpr int kCus = 256;
// The times beside the rules below are of whole calls over three sets of inputs in turn, both sides on one GPU.
// steps of a split at least, times head_dim (one token, 32 and 8 heads of 128, 8-bit pages: after
// 8192 12.8 us with 8 steps, 13.4 with 12, 14.4 with 16; after 1500 11.9, 12.8 and 15.6)
constexpr int kDecodeLeast = 1024;
constexpr int kPrefillLeast = 4;
constexpr int prefill_resident(int D) { return D == 256 ? 1 : 2; }
// Workgroups that a CU holds.  Each is four waves, one on a SIMD: 512 registers over them.
// Three at D = 128 in place of two, 8-bit pages: 64 sequences of up to 4096 tokens 63.4 -> 55.3 us,
// 200 of up to 500 31.8 -> 27.4 (32 windows of 1024 tokens over 16-bit pages 32.8 both ways, one
// sequence of 32768 34.9 -> 36.1).
constexpr int resident(int D) { return D == 64 ? 4 : D == 128 ? 3 : 2; }

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

// The sizes of a call: which kernel, how its work is divided at most.
struct BatchSizes {
    int32_t batch, seq_len, n_q_heads, n_kv_heads, head_dim, max_pages;
    bool empty() const { return batch <= 0 || seq_len <= 0 || n_q_heads <= 0 || n_kv_heads <= 0; }
    const char* refused() const {
        if (batch < 0 || seq_len < 0 || n_q_heads < 0 || n_kv_heads < 0 || max_pages < 0) return "negative size";
        if (n_kv_heads == 0 ? n_q_heads != 0 : n_q_heads % n_kv_heads != 0) return "n_q_heads must be a multiple of n_kv_heads";
        if (max_pages > 1 << 26) return "tables of up to 2^26 pages";
        if (int64_t(seq_len) * (n_kv_heads ? n_q_heads / n_kv_heads : 1) > 1 << 30) return "up to 2^30 rows for a kv head";
        return nullptr;
    }
};

// Decode rows: one 16-row tile.  More rows: tiles of 64 or 128.
inline BatchPlan plan_of(const BatchSizes& z) {
    BatchPlan r;
    const int64_t rows = int64_t(z.seq_len) * (z.n_q_heads / z.n_kv_heads);
    // no more than 2^31, so that 2^30 rows of each make no product of more than 64 bits: above
    // kMostWorkgroups the call is refused
    const int64_t heads = std::min<int64_t>(int64_t(z.batch) * z.n_kv_heads, int64_t(1) << 31);
    r.decode = rows <= kDecodeRows;
    r.target = kCus * (r.decode ? resident(z.head_dim) : prefill_resident(z.head_dim));
    // Prompts over little more than their own rows whose tiles of 64 are all there at once and
    // leave few places: eight waves to each, a long tile beside a short one, no split (16 q and
    // 8 kv heads of 128, 2048 tokens: 43.5 us, with tiles of 128 in splits 45.0; 1800: 37.6 and
    // 41.4; 2 x 1024: 31.2 and 34.0).  Not for short ones (4 x 512: 22.0 and 20.5), nor for chunks on a long
    // context, which splits divide evenly (2048 on 8192: 167 and 144), nor at head_dim 256, one workgroup
    // to a CU (8 and 2 heads, 2048 tokens: 56.6 and 48.6).
    const int64_t fine = (rows + 63) / 64 * heads;
    const bool fits = !r.decode && rows > 64 && z.head_dim <= 128 && z.seq_len >= 1024 && int64_t(z.max_pages) * kPage < 2 * int64_t(z.seq_len) && fine <= r.target &&
                      fine >= r.target / 4 * 3;
    r.rows = r.decode ? kDecodeRows : rows <= 64 || fits ? 64 : 128;
    r.step = r.decode ? kDecodeStep : kPrefillStep;
    r.tiles_max = (rows + r.rows - 1) / r.rows;
    r.tiles = r.tiles_max * heads;
    r.least = r.decode ? kDecodeLeast / z.head_dim : kPrefillLeast;
    // a merge is worth it for contexts of more than two such splits, three of one tile (one
    // token, 32 and 8 heads of 128, after 600: 9.3 us in one launch, 11.7 split; after 800:
    // 10.9 and 11.2; after 2048: 19.2 and 11.4).  Where the tiles alone keep the workgroups busy
    // in turn, only for contexts that are long beside the others: every workgroup looks through
    // all units to find its own (one token each, ragged, unsplit and split: 1024 entries of up
    // to 2048 tokens, 8 and 2 heads, 90 and 135 us; 256 of up to 4096, 32 and 8, 173 and 179).
    // A long entry among many then is one workgroup for each kv head, and takes as long as its tokens
    // after each other.  So it does with more rows as soon as the padded tiles fill the GPU, whatever rows
    // are there: a token at the end of a long context is better off in a call of few rows each.
    const int64_t turns = std::max<int64_t>(1, std::min<int64_t>(r.tiles / r.target, 1 << 20));
    r.can_split = (z.max_pages + r.step - 1) / r.step > (!r.decode ? 2 : turns > 1 ? 12 : 3) * r.least * turns && (r.decode || r.tiles < r.target) && !fits;
    r.least = int(r.least * turns);
    // all workgroups there at once, two to a CU: a long one beside a short one
    r.paired = !r.decode && !r.can_split && prefill_resident(z.head_dim) == 2 && r.tiles > kCus && r.tiles <= 2 * kCus;
    r.slots = r.tiles + (r.can_split ? r.target + 8 : 0);
    return r;
}
inline size_t workspace_of(const BatchPlan& r, int batch, int D) {
    return r.can_split ? size_t(r.slots) * r.rows * (D + 2) * 4 + (size_t(batch) * r.tiles_max * sizeof(Header) + 15 & ~size_t(15)) : 0;
}
constexpr int64_t kMostWorkgroups = INT_MAX / 512;  // of 512 threads, in a launch of fewer than 2^32; a merge has up to 16 of 64 for each

}  // namespace genllm
