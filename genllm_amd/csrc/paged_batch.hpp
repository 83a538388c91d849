// paged_batch.hpp -- what the kernels of paged_attention_batch share: pages and their
// scales, what a row sees, and the form that takes one key after another.
#pragma once

#include <climits>

#include "common.hpp"

#include "batch_work.hpp"  // takes kPage from the other

namespace genllm {

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

typedef __attribute__((address_space(3))) char lds_char;
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ s16x4_t ds_read_tr16(const lds_char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4_t*>(const_cast<lds_char*>(p)));
}

// V's pages are taken relative to a reference scale 2^ref, at least a 64th of the largest so
// far.  That is exact for a page at most 15 binades below it: a code's last bit, 2^-9, is
// fp16's, 2^-24.  Where there are lower ones, or sums might leave fp32's range, rows are
// computed by exact_keys in the end: the scale of another page, of keys that a row may not
// even see, costs no row its precision.  Pages of zeros alone, which have the least scale, do
// not count.  low: a lane's least; next(i): the i-th page, -1 behind the last.
// kScaleLead: how far a page may be above the reference.
constexpr int kScaleReach = 15, kScaleLead = 6, kMostScale = 64;

// A row's maximum may lag its scores by kLazy (log2), so a wave's sums may be 2^kLazy times
// those of probabilities of at most one.  Where all waves and splits (at most 2^13) might not add up
// within fp32's range, exact_keys takes its keys, with probabilities of at most one: sums of
// products above kMostSum, and 8-bit pages whose reference is above kMostScale (2^15 of a
// code and its lead, 2^15 of a probability, 2^30 keys: sums of up to 2^(60 + 64)).
constexpr float kLazy = 8.0f, kMostSum = 0x1p100f;

// A row's probabilities are formed relative to a reference, this much (log2) below its maximum.
// Relative to the maximum itself fp16, whose last bit is 2^-24, would make zeros of all keys
// 25 binades below it, which at the end of a long context can be 0.4 % of the weight (131072
// keys).  7 is what fp16's range leaves: 2^(kLazy + 7); the last bit is 2^-31 of the maximum.  bf16 has
// fp32's range.
template <bool kFp16>
constexpr float kHead = kFp16 ? 7.0f : 0.0f;
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

}  // namespace genllm
