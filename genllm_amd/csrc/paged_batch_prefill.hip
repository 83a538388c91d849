// paged_batch_prefill.hip -- attention of a padded batch over paged caches, for more than
// 16 rows per kv head: prompts, chunks on top of a cache, drafts of many heads.
//
// Rows are the (query, q head) pairs of a kv head, q heads fastest, in tiles of 64 or 128;
// wave w of four has 16 or 32 of them, as columns of the MFMA tiles (RB blocks of 16), and
// all keys of a step: four pages, 64 keys.  Wave w stages page w of the next step: 16-byte
// loads into registers while this step is computed, then to LDS as 16-bit rows whose
// 16-byte chunks are swizzled.  8-bit codes are converted once here, for all waves: K's to
// q's type (without loss; the page's scale is in the factor of the scores), V's to fp16
// relative to a reference scale that follows the largest, so that P is rounded to fp16 (11
// bits) whatever q's type is.  From 16-bit pages P has the elements' type.  Per step:
//   S^T = K Q^T   v_mfma 16x16x32, K's operand read once for the RB row blocks
//   O^T += V^T P^T  with V^T by transposing LDS reads; the sum of a row's probabilities
//        by one more MFMA with ones, from the same rounded values
// Lane (row, g) has the scores of keys 4g..4g+3 of each page: the running maximum and the
// rescaling stay in the lane.  Two LDS buffers, one barrier a step.
#include "paged_batch.hpp"

namespace genllm {

namespace {

constexpr float kLazy = 8.0f;  // log2: a row's maximum may lag its scores by this much
constexpr int kScaleLead = 6;  // a page's scale may be this many binades above the reference
constexpr int kKeys = kPrefillStep * kPage;

typedef __attribute__((address_space(3))) char lds_char;
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) u32x4_t lds_u32x4;

__device__ __forceinline__ s16x4_t ds_read_tr16(const lds_char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4_t*>(const_cast<lds_char*>(p)));
}

// Place of 16-byte chunk c in the LDS row of token r (of 16): K's reads (16 rows, one
// chunk) and the halves of a transposing read (rows 0-3 and 8-11, or 4-7 and 12-15, two
// neighbouring chunks) cover all banks once.
template <int D>
__device__ __forceinline__ int place(int r, int c) {
    if constexpr (D == 64) return c ^ (((r >> 2) & 1) | ((r >> 1) & 1) << 1 | (r >> 3) << 2);
    return (c & ~15) | ((c & 15) ^ ((((r & 7) ^ ((r >> 1) & 4)) << 1) | (r >> 3)));
}

template <int D, bool F16, bool Q8, int RB>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void batch_prefill_kernel(BatchAttn p) {
    using E = Elem<F16>;
    using EV = Elem<F16 || Q8>;
    constexpr int ES = Q8 ? 1 : 2, KS = D / 32, DB = D / 16;
    constexpr int ROWS = 64 * RB;
    constexpr int ROWB = 2 * D;          // bytes of a token's row in LDS
    constexpr int SRC = D * ES / 16;     // 16-byte chunks of a token's row in memory
    constexpr int LD = SRC / 4;          // 16-byte loads of a lane for a page
    constexpr int TILE = kKeys * ROWB;
    __shared__ __attribute__((aligned(16))) char lds_k0[TILE], lds_k1[TILE], lds_v0[TILE], lds_v1[TILE];

    prefetch_kernargs<sizeof(BatchAttn)>();
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, g = lane >> 4;
    Work w;
    if (!find_work<ROWS, kPrefillStep>(p, int(blockIdx.x), w)) return;
    put_header(p, w);
    const int rows = w.e.ql * p.G, row0 = w.tile * ROWS + 16 * RB * wv;  // of the entry; the wave's first

    uint4 qb[RB][KS];
    Sight see[RB];
    const uint16_t* qrow[RB];
    int64_t orow[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int row = min(row0 + 16 * rb + n16, rows - 1), query = row / p.G, head = w.h * p.G + row - query * p.G;
        see[rb] = sight_of(p, w.e, query);
        qrow[rb] = p.q + w.b * p.q_batch + query * p.q_tok + head * p.q_head;
        orow[rb] = w.b * p.o_batch + query * p.o_tok + head * p.o_head;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qb[rb][ks] = *reinterpret_cast<const uint4*>(qrow[rb] + 32 * ks + 8 * g);
    }
    // positions of the tile's, and of the wave's, first and last row
    const auto pos_of = [&](int row) { return p.causal ? w.e.n - w.e.ql + min(row, rows - 1) / p.G : w.e.n - 1; };
    const int tile_first = pos_of(w.tile * ROWS), tile_last = pos_of(w.tile * ROWS + ROWS - 1);
    const bool has_rows = row0 < rows;
    const int pos_a = pos_of(row0), pos_b = pos_of(row0 + 16 * RB - 1);

    const Span span = span_of(p, tile_first, min(tile_last + 1, w.e.n));
    const int steps = (span.pages + kPrefillStep - 1) / kPrefillStep;
    const int s0 = int(int64_t(steps) * w.sp / w.ns), s1 = int(int64_t(steps) * (w.sp + 1) / w.ns);

    f32x4_t acc[RB][DB], accl[RB];
    float m[RB], nm[RB], th[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        accl[rb] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[rb][db] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        m[rb] = -INFINITY, nm[rb] = 0.0f, th[rb] = -INFINITY;
    }
    int vref = INT_MIN, vacc = INT_MIN;  // reference scale of the staged step, and of acc

    // ---- staging: lane i of every wave knows page i of 16 steps
    constexpr int kBlock = 64 / kPrefillStep;
    PageInfo info;
    const auto look_up = [&](int step) {
        const int j = kPrefillStep * step + lane;
        info = page_info<Q8>(p, w.b, w.h, span.page(j), j < span.pages && step + lane / kPrefillStep < s1);
    };
    uint4 kreg[LD], vreg[LD];
    float kf[kPrefillStep], kf_next[kPrefillStep];
    const int k_off = (lane / SRC) * p.k_tok + 16 * (lane % SRC), v_off = (lane / SRC) * p.v_tok + 16 * (lane % SRC);
    const auto issue = [&](int step) {
        const int at = kPrefillStep * ((step - s0) % kBlock) + wv, j = kPrefillStep * step + wv;
        const int kid = __builtin_amdgcn_readlane(info.kid, at), vid = __builtin_amdgcn_readlane(info.vid, at);
        const int first = j < span.pages ? span.page(j) * kPage : 1 << 30;
        const int valid = kid < 0 ? 0 : min(w.e.n - first, kPage);  // rows behind the cache's end read as zeros
        const char* const kb = p.k_pool + (kid < 0 ? 0 : kid) * p.k_block + int64_t(w.h) * p.k_head;
        const char* const vb = p.v_pool + (kid < 0 ? 0 : vid) * p.v_block + int64_t(w.h) * p.v_head;
        const auto rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(kb), 0, valid > 0 ? (valid - 1) * p.k_tok + D * ES : 0, kBufferFlags);
        const auto rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(vb), 0, valid > 0 ? (valid - 1) * p.v_tok + D * ES : 0, kBufferFlags);
#pragma unroll
        for (int e = 0; e < LD; ++e) kreg[e] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rk, k_off, e * (64 / SRC) * p.k_tok, 0));
#pragma unroll
        for (int e = 0; e < LD; ++e) vreg[e] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rv, v_off, e * (64 / SRC) * p.v_tok, 0));
    };
    const auto stage = [&](int step, lds_char* kl, lds_char* vl) {
        const int at = kPrefillStep * ((step - s0) % kBlock);
        float vs = 1.0f;
#pragma unroll
        for (int i = 0; i < kPrefillStep; ++i)
            kf_next[i] = score_factor<Q8>(p, __builtin_amdgcn_readlane(info.vid, at + i), __builtin_amdgcn_readlane(info.kb, at + i),
                                          __builtin_amdgcn_readlane(info.vb, at + i));
        if constexpr (Q8) {
            int most = INT_MIN;
#pragma unroll
            for (int i = 0; i < kPrefillStep; ++i) most = max(most, __builtin_amdgcn_readlane(info.vb, at + i) - 127);
            if (vref == INT_MIN || most > vref + kScaleLead) vref = most;
            vs = power_of_two(__builtin_amdgcn_readlane(info.vb, at + wv) - 127 - vref);
        }
#pragma unroll
        for (int e = 0; e < LD; ++e) {
            const int t = e * (64 / SRC) + lane / SRC, c = lane % SRC, row = (wv * kPage + t) * ROWB;
            if constexpr (Q8) {
                const auto put = [&](lds_char* l, int chunk, const uint4& x) {
                    *reinterpret_cast<lds_u32x4*>(l + row + 16 * place<D>(t, chunk)) = __builtin_bit_cast(u32x4_t, x);
                };
                put(kl, 2 * c, f8_octet<F16>(kreg[e].x, kreg[e].y, 1.0f, 1.0f));
                put(kl, 2 * c + 1, f8_octet<F16>(kreg[e].z, kreg[e].w, 1.0f, 1.0f));
                put(vl, 2 * c, f8_octet<true>(vreg[e].x, vreg[e].y, vs, vs));
                put(vl, 2 * c + 1, f8_octet<true>(vreg[e].z, vreg[e].w, vs, vs));
            } else {
                *reinterpret_cast<lds_u32x4*>(kl + row + 16 * place<D>(t, c)) = __builtin_bit_cast(u32x4_t, kreg[e]);
                *reinterpret_cast<lds_u32x4*>(vl + row + 16 * place<D>(t, c)) = __builtin_bit_cast(u32x4_t, vreg[e]);
            }
        }
    };

    const auto compute = [&](int step, const lds_char* kl, const lds_char* vl, int ref) {
        int first[kPrefillStep];
        bool some = false;
#pragma unroll
        for (int i = 0; i < kPrefillStep; ++i) {
            const int j = kPrefillStep * step + i;
            first[i] = j < span.pages ? span.page(j) * kPage : 1 << 30;
            some |= first[i] <= pos_b && (first[i] + kPage - 1 > pos_a - p.window || first[i] < p.sinks);
        }
        if (!some || !has_rows) return;  // wave-uniform
        f32x4_t s[RB][kPrefillStep];
#pragma unroll
        for (int i = 0; i < kPrefillStep; ++i) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) s[rb][i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const u32x4_t a = *reinterpret_cast<const lds_u32x4*>(kl + (i * kPage + n16) * ROWB + 16 * place<D>(n16, 4 * ks + g));
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) s[rb][i] = E::mma32(__builtin_bit_cast(uint4, a), qb[rb][ks], s[rb][i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kPrefillStep; ++i) {
            const int last = first[i] + kPage - 1;
            if (last > pos_a || (first[i] <= pos_b - p.window && last >= p.sinks)) {  // some row does not see all of it
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[rb][i][k] = see[rb](p, first[i] + 4 * g + k) ? s[rb][i][k] : -INFINITY;
            }
        }
        if constexpr (Q8) {
            if (vacc != ref) {  // wave-uniform
                if (vacc != INT_MIN) {
                    const float f = power_of_two(vacc - ref);
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                        for (int db = 0; db < DB; ++db) acc[rb][db] *= f;
                }
                vacc = ref;
            }
        }
        uint4 pb[RB][kPrefillStep / 2];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < kPrefillStep; ++i) {
                const float a = __builtin_elementwise_maximum(__builtin_elementwise_maximum(s[rb][i][0], s[rb][i][1]),
                                                              __builtin_elementwise_maximum(s[rb][i][2], s[rb][i][3]));
                mx = __builtin_elementwise_maximum(mx, a * kf[i]);
            }
            if (__any(mx > th[rb])) {
                mx = fmaxf(mx, __shfl_xor(mx, 16));
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const bool grow = mx > th[rb];
                const float mn = grow ? mx : m[rb], alpha = grow ? exp2_fast(m[rb] - mn) : 1.0f;
                m[rb] = mn;
                nm[rb] = grow ? -mn : nm[rb];
                th[rb] = grow ? mn + kLazy : th[rb];
                accl[rb] *= alpha;
#pragma unroll
                for (int db = 0; db < DB; ++db) acc[rb][db] *= alpha;
            }
            uint32_t e2[2 * kPrefillStep];
#pragma unroll
            for (int i = 0; i < kPrefillStep; ++i)
#pragma unroll
                for (int k = 0; k < 4; k += 2)
                    e2[2 * i + k / 2] = EV::pack_p(exp2_fast(__builtin_fmaf(s[rb][i][k], kf[i], nm[rb])),
                                                   exp2_fast(__builtin_fmaf(s[rb][i][k + 1], kf[i], nm[rb])));
#pragma unroll
            for (int i = 0; i < kPrefillStep / 2; ++i) pb[rb][i] = make_uint4(e2[4 * i], e2[4 * i + 1], e2[4 * i + 2], e2[4 * i + 3]);
        }
        const uint32_t one2 = EV::pack_p(1.0f, 1.0f);
        const uint4 ones = make_uint4(one2, one2, one2, one2);
#pragma unroll
        for (int i = 0; i < kPrefillStep / 2; ++i) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) accl[rb] = EV::mma32(ones, pb[rb][i], accl[rb]);
            const int t = 4 * g + (n16 >> 2);
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const lds_char* const at = vl + (32 * i + t) * ROWB + 16 * place<D>(t, 2 * db + ((n16 & 3) >> 1)) + 8 * (n16 & 1);
                const s16x4_t u[2] = {ds_read_tr16(at), ds_read_tr16(at + kPage * ROWB)};
                const uint4 a = __builtin_bit_cast(uint4, u);
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) acc[rb][db] = EV::mma32(a, pb[rb][i], acc[rb][db]);
            }
        }
    };

    if (s0 < s1) {
        look_up(s0);
        issue(s0);
        stage(s0, (lds_char*)lds_k0, (lds_char*)lds_v0);
    }
    const auto turn = [&](int t, lds_char* kl, lds_char* vl, lds_char* kn, lds_char* vn) {
#pragma unroll
        for (int i = 0; i < kPrefillStep; ++i) kf[i] = kf_next[i];
        const int ref = vref;
        __syncthreads();  // step t is staged; the other buffer is free
        const bool more = t + 1 < s1;
        if (more) {
            if ((t + 1 - s0) % kBlock == 0) look_up(t + 1);
            issue(t + 1);
        }
        compute(t, kl, vl, ref);
        if (more) stage(t + 1, kn, vn);
    };
    for (int t = s0; t < s1; t += 2) {
        turn(t, (lds_char*)lds_k0, (lds_char*)lds_v0, (lds_char*)lds_k1, (lds_char*)lds_v1);
        if (t + 1 < s1) turn(t + 1, (lds_char*)lds_k1, (lds_char*)lds_v1, (lds_char*)lds_k0, (lds_char*)lds_v0);
    }

    if (!has_rows) return;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int row = row0 + 16 * rb + n16;
        float l = accl[rb][0], sum = l;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += acc[rb][db][i];
        if (__any(row < rows && !(fabsf(sum) <= __FLT_MAX__))) {
            exact_keys<D, F16, Q8>(p, w.b, w.h, qrow[rb], see[rb], [&](int i) {
                const int j = kPrefillStep * s0 + i;
                return j < kPrefillStep * s1 && j < span.pages ? span.page(j) : -1;
            }, acc[rb], m[rb], l);
        } else if (Q8 && vacc != INT_MIN) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[rb][db][i] = ldexpf(acc[rb][db][i], vacc);
        }
        if (row >= rows) continue;
        if (w.ns > 1) {
            const int64_t at = int64_t(blockIdx.x) * ROWS + (row - w.tile * ROWS);
            float* const po = partial_rows(p) + at * D + 4 * g;
#pragma unroll
            for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4_t*>(po + 16 * db) = acc[rb][db];
            if (g == 0) *reinterpret_cast<float2*>(partial_rows(p) + int64_t(p.slots) * ROWS * D + 2 * at) = make_float2(m[rb], l);
            continue;
        }
        const float inv = 1.0f / l;
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            float o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = see[rb].any ? acc[rb][db][i] * inv : 0.0f;
            *reinterpret_cast<uint2*>(p.out + orow[rb] + 16 * db + 4 * g) = make_uint2(E::pack_p(o[0], o[1]), E::pack_p(o[2], o[3]));
        }
    }
}

template <bool F16, bool Q8, int RB>
int prefill_of(const BatchAttn& p, int D, hipStream_t stream) {
    const dim3 grid(unsigned(p.slots)), block(256);
    if (D == 64) hipLaunchKernelGGL((batch_prefill_kernel<64, F16, Q8, RB>), grid, block, 0, stream, p);
    else if (D == 128) hipLaunchKernelGGL((batch_prefill_kernel<128, F16, Q8, RB>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((batch_prefill_kernel<256, F16, Q8, RB>), grid, block, 0, stream, p);
    GENLLM_LAUNCH_CHECK("batch_prefill_kernel");
    return GENLLM_OK;
}
template <int RB>
int prefill_rows(const BatchAttn& p, int D, bool f16, hipStream_t s) {
    return f16 ? p.k_scales ? prefill_of<true, true, RB>(p, D, s) : prefill_of<true, false, RB>(p, D, s)
               : p.k_scales ? prefill_of<false, true, RB>(p, D, s) : prefill_of<false, false, RB>(p, D, s);
}

}  // namespace

int launch_batch_prefill(const BatchAttn& p, int tile_rows, int D, bool f16, hipStream_t stream) {
    return tile_rows == 64 ? prefill_rows<1>(p, D, f16, stream) : prefill_rows<2>(p, D, f16, stream);
}

}  // namespace genllm
