// paged_batch_prefill.hip -- attention of a padded batch over paged caches, for more than
// 16 rows per kv head: prompts, chunks on top of a cache, drafts of many heads.
//
// Rows are the (query, q head) pairs of a kv head, q heads fastest; a step is four pages, 64
// keys.  Two forms:
//   tiles of 128 rows, four waves of 32 (RB = 2 blocks of 16) that take all keys of a step:
//     an operand read from LDS feeds two MFMAs, as long as its read takes the four waves;
//   tiles of 64 rows, eight waves of 16 in two groups (KG = 2) with half of a step's keys
//     each, joined through LDS in the end: more waves for few rows (the rule is plan_of's).
// Waves stage the pages of the next step: 16-byte loads into registers while this step is
// computed, then to LDS as 16-bit rows, two buffers, one barrier a step.  K's 16-byte chunks
// are swizzled, V's rows padded.  8-bit codes are converted once here, for all waves: K's to
// q's type (without loss; the page's scale is in the factor of the scores), V's to fp16
// relative to a reference scale that follows the largest, so that P is rounded to fp16 (11
// bits) whatever q's type is.  From 16-bit pages P has the elements' type, as the MFMA takes it:
// over bf16 pages results are off by 2.1e-3 (relative, against 64 bits) where their own rounding
// alone leaves 1.7e-3.  In two parts, as for few rows, P V takes twice the MFMAs, where a wave's
// chain is the bound: 4096 tokens in windows of 512 35.1 -> 40.9 us, 2 x 512 queries on 8192 tokens 159 ->
// 203, over 8-bit pages 148 -> 197.  Per step:
//   S^T = K Q^T   v_mfma 16x16x32, K's operand read once for the RB row blocks
//   O^T += V^T P^T  with V^T by transposing LDS reads; the sum of a row's probabilities
//        by one more MFMA with ones, from the same rounded values
// Lane (row, g) has the scores of keys 4g..4g+3 of each page: the running maximum and the
// rescaling stay in the lane.
//
// Bound by a wave's chain where two waves share a SIMD: of a step's 4,400 cycles for both
// (D = 128, 8-bit) the matrix core is busy in 2,180, vector instructions and exponentials
// take about as many and overlap it in part.  2 x 512 queries on 8192 tokens, 32 and 8 heads
// of 128: 145 us, 920 TFLOP/s (a large library product reaches 1,184); 8192 tokens, 16 and 8
// heads, causal: 268 us.  2048 tokens, 16 and 8 heads: 40.7 us, where the kernel for one sequence over 16-bit
// pages (paged_prefill.hip) takes 30: this one issues 1.5 times its vector and twice its scalar instructions and
// LDS cycles (pages found and descriptors formed anew each step, conversion, conflicts of the
// staging writes).  At D = 128 registers go to scratch memory: 2 of the form with 64 rows over
// 8-bit pages, 12 over 16-bit ones, 4 of the form with 128 rows over 16-bit ones.  Also tried: staging between the MFMAs of P V (no gain), loads two
// steps ahead (none), Q and the output through LDS as whole rows (2 % slower).
#include <type_traits>

#include "paged_batch.hpp"

namespace genllm {

namespace {

// The two waves of a SIMD: one whose MFMA waits for the matrix core keeps the other's vector
// instructions from being issued, unless those come first (8192 tokens, 16 and 8 heads of 128:
// 309 us without priorities, 295 with both at 3, 275 so; 2 x 512 queries on 8192 158, 154, 150).
constexpr int kSoftmaxPrio = 2, kStagePrio = 3;
constexpr int kKeys = kPrefillStep * kPage;

typedef __attribute__((address_space(3))) u32x4_t lds_u32x4;

// K in LDS: 16-byte chunk c of token r (of 16) at place c ^ f(r) of its row, so that the
// reads of an operand (16 rows, one chunk) cover all banks once.
template <int D>
__device__ __forceinline__ int k_place(int r, int c) {
    if constexpr (D == 64) return c ^ (((r >> 2) & 1) | ((r >> 1) & 1) << 1 | (r >> 3) << 2);
    return (c & ~15) | ((c & 15) ^ ((((r & 7) ^ ((r >> 1) & 4)) << 1) | (r >> 3)));
}
// V in LDS: rows apart by two chunks more than they have, those from the eighth on of a
// page by eight more: the halves of a transposing read (rows 0-3 and 8-11, or 4-7 and 12-15,
// two neighbouring chunks) cover all banks once, and the chunks of a row lie at fixed
// distances: one address for all of them.
template <int D>
constexpr int kVRow = 2 * D + 32;
template <int D>
constexpr int kVPage = kPage * kVRow<D> + 128;
template <int D>
__device__ __forceinline__ int v_row(int r) { return r * kVRow<D> + (r >> 3) * 128; }

// KG groups of four waves share the keys of a step: 1 with 32 rows a wave (RB = 2), 2 with 16.
template <int D, bool F16, bool Q8, int RB, int KG>
__global__ __launch_bounds__(256 * KG, KG == 2 ? (D == 256 ? 2 : 4) : D == 256 ? 1 : 2) void batch_prefill_kernel(BatchAttn p) {
    using E = Elem<F16>;
    using EV = Elem<F16 || Q8>;
    constexpr int ES = Q8 ? 1 : 2, KS = D / 32, DB = D / 16;
    constexpr int ROWS = 64 * RB, NP = kPrefillStep / KG;  // pages of a step that are a wave's
    constexpr int ROWB = 2 * D;          // bytes of a token's row in LDS
    constexpr int SRC = D * ES / 16;     // 16-byte chunks of a token's row in memory
    constexpr int LD = SRC / 4;          // 16-byte loads of a lane for a page
    constexpr int TILE = kKeys * ROWB;
    __shared__ __attribute__((aligned(16))) char lds_k0[TILE], lds_k1[TILE], lds_v0[kPrefillStep * kVPage<D>], lds_v1[kPrefillStep * kVPage<D>];

    prefetch_kernargs<sizeof(BatchAttn)>();
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, g = lane >> 4;
    Work w;
    if (!find_work<ROWS, kPrefillStep>(p, int(blockIdx.x), w)) return;
    put_header(p, w);
    const int rows = w.e.ql * p.G, row0 = w.tile * ROWS + 16 * RB * (wv & 3);  // of the entry; the wave's first
    const int kg = KG == 1 ? 0 : wv >> 2, p0 = NP * kg;  // its group; the first of its pages in a step

    const Divisor by_g(p.G);
    uint4 qb[RB][KS];
    int query[RB];
    // addresses and sights of rows are formed where they are used
    const auto row_at = [&](int rb, int64_t batch, int64_t tok, int64_t head) {
        int row = min(row0 + 16 * rb + n16, rows - 1);
        __asm__ volatile("" : "+v"(row));
        return w.b * batch + query[rb] * tok + (w.h * p.G + row - query[rb] * p.G) * head;
    };
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        query[rb] = by_g(min(row0 + 16 * rb + n16, rows - 1));
        const uint16_t* const qrow = p.q + row_at(rb, p.q_batch, p.q_tok, p.q_head);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qb[rb][ks] = *reinterpret_cast<const uint4*>(qrow + 32 * ks + 8 * g);
    }
    // positions of the wave's first and last row
    const auto pos_of = [&](int row) { return p.causal ? w.e.n - w.e.ql + by_g(min(row, rows - 1)) : w.e.n - 1; };
    const int pos_a = __builtin_amdgcn_readfirstlane(pos_of(row0)), pos_b = __builtin_amdgcn_readfirstlane(pos_of(row0 + 16 * RB - 1));

    const TileKeys keys = tile_keys<ROWS>(p, w.e, w.tile);
    const Span span = span_of(p, keys.first, keys.end);
    const int steps = (span.pages + kPrefillStep - 1) / kPrefillStep;
    const int s0 = int(int64_t(steps) * w.sp / w.ns), s1 = int(int64_t(steps) * (w.sp + 1) / w.ns);

    f32x4_t acc[RB][DB], accl[RB];
    constexpr float kBelow = kHead<F16 || Q8>;
    float m[RB], nm[RB], th[RB];  // kBelow under a row's maximum, its negative (0 while there is none), where it grows
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        accl[rb] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[rb][db] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        m[rb] = -INFINITY, nm[rb] = 0.0f, th[rb] = -INFINITY;
    }
    int vref = INT_MIN, vacc = INT_MIN;  // reference scale of the staged step, and of acc
    ScaleRange range;

    // ---- staging: lane i of every wave knows page i of 16 steps
    constexpr int kBlock = 64 / kPrefillStep;
    PageInfo info;
    // where its rows are that this wave stages (64 bits; K's, or V's in the second of two
    // groups), and how many: formed by the lanes, taken by `issue`
    int info_k[2], info_v[KG == 1 ? 2 : 1], info_n;
    const auto look_up = [&](int step) {
        const int j = kPrefillStep * step + lane;
        info = page_info<Q8>(p, w.b, w.h, span.page(j), j < span.pages && step + lane / kPrefillStep < s1);
        const char* const k = p.k_pool + max(info.kid, 0) * p.k_block + int64_t(w.h) * p.k_head;
        const char* const v = p.v_pool + max(info.vid, 0) * p.v_block + int64_t(w.h) * p.v_head;
        const uintptr_t one = uintptr_t(KG == 1 || kg == 0 ? k : v);
        info_k[0] = int(one), info_k[1] = int(one >> 32);
        if constexpr (KG == 1) info_v[0] = int(uintptr_t(v)), info_v[1] = int(uintptr_t(v) >> 32);
        info_n = info.kid < 0 ? 0 : min(w.e.n - span.page(j) * kPage, kPage);  // rows behind the cache's end read as zeros
    };
    float info_kf = 0.0f;  // of info, once its scales are needed
    uint4 kreg[LD], vreg[KG == 1 ? LD : 1];  // two groups: one stages K (both in kreg), the other V
    const int pg = wv & 3;
    float kf[NP], kf_next[NP];
    // the next step's loads: `aim` finds the rows, `load` brings one of kLoads 16-byte parts
    struct Rows { __amdgpu_buffer_rsrc_t at; int tok, off; } from[KG == 1 ? 2 : 1];
    constexpr int kLoads = KG == 1 ? 2 * LD : LD;
    // many loads at once hold the wave up (16 of 16 bytes to a lane, 1200 cycles of a step's
    // 5900 at D = 256): they are issued between the MFMAs of the scores (a window of 512 on 4096
    // tokens 36.1 -> 35.1 us); four or eight are not (8 at D = 128: 2 x 512 on 8192 160 and 158 us)
    constexpr bool kSpread = kLoads >= 16;
    const auto aim = [&](int step) {
        const int at = kPrefillStep * ((step - s0) % kBlock) + pg;
        const int n = step < s1 ? __builtin_amdgcn_readlane(info_n, at) : 0;
        const auto rows_of = [&](const int (&place)[2], int tok) {
            const uint64_t base = uint32_t(__builtin_amdgcn_readlane(place[0], at)) | uint64_t(uint32_t(__builtin_amdgcn_readlane(place[1], at))) << 32;
            return Rows{__builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(base), 0, n > 0 ? (n - 1) * tok + D * ES : 0, kBufferFlags), tok,
                        (lane / SRC) * tok + 16 * (lane % SRC)};
        };
        from[0] = rows_of(info_k, KG == 1 || kg == 0 ? p.k_tok : p.v_tok);
        if constexpr (KG == 1) from[1] = rows_of(info_v, p.v_tok);
    };
    const auto load = [&](int l) {
        const Rows& f = from[KG == 1 ? l / LD : 0];
        (KG == 2 || l < LD ? kreg : vreg)[l % LD] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(f.at, f.off, l % LD * (64 / SRC) * f.tok, 0));
    };
    const auto stage = [&](int step, lds_char* kl, lds_char* vl) {
        const int at = kPrefillStep * ((step - s0) % kBlock);
        float vs = 1.0f;
        if (at == 0) {
            info_kf = score_factor<Q8>(p, info.vid, info.kb, info.vb);
            if constexpr (Q8) range.add(info);
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) kf_next[i] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(info_kf), at + p0 + i));
        if constexpr (Q8) {
            int most = INT_MIN;
#pragma unroll
            for (int i = 0; i < kPrefillStep; ++i) most = max(most, __builtin_amdgcn_readlane(info.vb, at + i) - 127);
            if (vref == INT_MIN || most > vref + kScaleLead) vref = most;
            vs = power_of_two(__builtin_amdgcn_readlane(info.vb, at + pg) - 127 - vref);
        }
        const auto put = [](lds_char* at, const uint4& x) { *reinterpret_cast<lds_u32x4*>(at) = __builtin_bit_cast(u32x4_t, x); };
        const auto put_k = [&](const uint4* reg) {
#pragma unroll
            for (int e = 0; e < LD; ++e) {
                const int t = e * (64 / SRC) + lane / SRC, c = lane % SRC;
                lds_char* const to = kl + (pg * kPage + t) * ROWB;
                if constexpr (Q8) {
                    // chunks 32 bytes apart over the lanes: a step's writes (32 KB at D = 128) take 256 cycles
                    // of bank conflicts; the two in turn from row to row take as many
                    put(to + 16 * k_place<D>(t, 2 * c), f8_octet<F16>(reg[e].x, reg[e].y, 1.0f, 1.0f));
                    put(to + 16 * k_place<D>(t, 2 * c + 1), f8_octet<F16>(reg[e].z, reg[e].w, 1.0f, 1.0f));
                } else {
                    put(to + 16 * k_place<D>(t, c), reg[e]);
                }
            }
        };
        const auto put_v = [&](const uint4* reg) {
#pragma unroll
            for (int e = 0; e < LD; ++e) {
                const int t = e * (64 / SRC) + lane / SRC, c = lane % SRC;
                lds_char* const to = vl + pg * kVPage<D> + v_row<D>(t);
                if constexpr (Q8) {
                    put(to + 32 * c, f8_octet<true>(reg[e].x, reg[e].y, vs, vs));
                    put(to + 32 * c + 16, f8_octet<true>(reg[e].z, reg[e].w, vs, vs));
                } else {
                    put(to + 16 * c, reg[e]);
                }
            }
        };
        if (KG == 1 || kg == 0) put_k(kreg);
        if constexpr (KG == 1) put_v(vreg);
        else if (kg == 1) put_v(kreg);
    };

    // whether the wave's rows see all of its pages of a step
    const auto sees_all = [&](int step) {
        const int j = kPrefillStep * step + p0, first = span.page(j) * kPage;
        if (j + NP > span.pages) return false;
        const int last = span.page(j + NP - 1) * kPage + kPage - 1;
        return last <= pos_a && (first > pos_b - p.window || last < p.sinks);
    };
    const uint32_t one2 = EV::pack_p(1.0f, 1.0f);
    const uint4 ones = make_uint4(one2, one2, one2, one2);
    const auto compute = [&](int step, const lds_char* kl, const lds_char* vl, int ref) {
        f32x4_t s[RB][NP];
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) s[rb][i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        // Two pages in turn: the MFMAs of a sum wait for each other.  kAheadK operands on
        // their way from LDS while one is used: a read takes as long as six MFMAs or more, and
        // two waves to a SIMD do not hide that (2 x 512 queries on 8192 keys 170 -> 157 us).
        constexpr int NK = NP * KS, kAheadK = KG == 1 && NK >= 4 ? 4 : 2;
        u32x4_t ka[kAheadK];
        const auto k_operand = [&](int x) {  // x: page pair, k-step, page of the pair
            const int i = 2 * (x / (2 * KS)) + (x & 1), ks = x / 2 % KS;
            return *reinterpret_cast<const lds_u32x4*>(kl + ((p0 + i) * kPage + n16) * ROWB + 16 * k_place<D>(n16, 4 * ks + g));
        };
#pragma unroll
        for (int x = 0; x < kAheadK; ++x) ka[x] = k_operand(x);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < NK; ++x) {
            const int i = 2 * (x / (2 * KS)) + (x & 1), ks = x / 2 % KS;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) s[rb][i] = E::mma32(__builtin_bit_cast(uint4, ka[x % kAheadK]), qb[rb][ks], s[rb][i]);
            if (x + kAheadK < NK) ka[x % kAheadK] = k_operand(x + kAheadK);
#pragma unroll
            for (int l = (x * kLoads + NK - 1) / NK; kSpread && l < ((x + 1) * kLoads + NK - 1) / NK; ++l) load(l);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(kSoftmaxPrio);
        if (!sees_all(step))  // wave-uniform
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int j = kPrefillStep * step + p0 + i, first = j < span.pages ? span.page(j) * kPage : 1 << 30, last = first + kPage - 1;
                if (last <= pos_a && (first > pos_b - p.window || last < p.sinks)) continue;  // every row sees all of it
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    const Sight see = sight_of(p, w.e, query[rb]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[rb][i][k] = see(p, first + 4 * g + k) ? s[rb][i][k] : -INFINITY;
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
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const float a = __builtin_elementwise_maximum(__builtin_elementwise_maximum(s[rb][i][0], s[rb][i][1]),
                                                              __builtin_elementwise_maximum(s[rb][i][2], s[rb][i][3]));
                mx = __builtin_elementwise_maximum(mx, a * kf[i]);
            }
            if (__any(mx > th[rb])) {
                mx = fmaxf(mx, __shfl_xor(mx, 16));
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const bool grow = mx > th[rb];
                const float mn = grow ? mx - kBelow : m[rb], alpha = grow ? exp2_fast(m[rb] - mn) : 1.0f;
                m[rb] = mn;
                nm[rb] = grow ? -mn : nm[rb];
                th[rb] = grow ? mn + (kBelow + kLazy) : th[rb];
                accl[rb] *= alpha;
#pragma unroll
                for (int db = 0; db < DB; ++db) acc[rb][db] *= alpha;
            }
        }
        // V's first operands come while the probabilities are formed
        constexpr int NV = NP / 2 * DB, kAheadV = KG == 1 ? 4 : 2;
        const int t = 4 * g + (n16 >> 2);
        const lds_char* const vt = vl + p0 * kVPage<D> + v_row<D>(t) + 8 * (n16 & 3);
        s16x4_t va[kAheadV][2];
        const auto v_operand = [&](int x, s16x4_t (&to)[2]) {
            const int i = x / DB, db = x % DB;
            to[0] = ds_read_tr16(vt + 2 * i * kVPage<D> + 32 * db), to[1] = ds_read_tr16(vt + (2 * i + 1) * kVPage<D> + 32 * db);
        };
#pragma unroll
        for (int x = 0; x < kAheadV; ++x) v_operand(x, va[x]);
        __builtin_amdgcn_sched_barrier(0);
        uint4 pb[RB][NP / 2];
#pragma unroll
        for (int i = 0; i < NP / 2; ++i)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                uint32_t e[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f32x4_t& x = s[rb][2 * i + (k >> 1)];
                    const float f = kf[2 * i + (k >> 1)];
                    e[k] = EV::pack_p(exp2_fast(__builtin_fmaf(x[2 * (k & 1)], f, nm[rb])), exp2_fast(__builtin_fmaf(x[2 * (k & 1) + 1], f, nm[rb])));
                }
                pb[rb][i] = make_uint4(e[0], e[1], e[2], e[3]);
                accl[rb] = EV::mma32(ones, pb[rb][i], accl[rb]);
            }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int x = 0; x < NV; ++x) {
            const uint4 a = __builtin_bit_cast(uint4, va[x % kAheadV]);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) acc[rb][x % DB] = EV::mma32(a, pb[rb][x / DB], acc[rb][x % DB]);
            if (x + kAheadV < NV) v_operand(x + kAheadV, va[x % kAheadV]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    if (s0 < s1) {
        look_up(s0);
        aim(s0);
#pragma unroll
        for (int l = 0; l < kLoads; ++l) load(l);
        stage(s0, (lds_char*)lds_k0, (lds_char*)lds_v0);
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) landed(qb[rb][ks]);
    const auto turn = [&](int t, lds_char* kl, lds_char* vl, lds_char* kn, lds_char* vn) {
#pragma unroll
        for (int i = 0; i < NP; ++i) kf[i] = kf_next[i];
        const int ref = vref;
        __syncthreads();  // step t is staged; the other buffer is free
        const bool more = t + 1 < s1;
        if (more && (t + 1 - s0) % kBlock == 0) look_up(t + 1);
        aim(t + 1);
#pragma unroll
        for (int l = 0; !kSpread && l < kLoads; ++l) load(l);
        compute(t, kl, vl, ref);
        __builtin_amdgcn_s_setprio(kStagePrio);
        if (more) stage(t + 1, kn, vn);
        __builtin_amdgcn_s_setprio(0);
    };
    for (int t = s0; t < s1; t += 2) {
        turn(t, (lds_char*)lds_k0, (lds_char*)lds_v0, (lds_char*)lds_k1, (lds_char*)lds_v1);
        if (t + 1 < s1) turn(t + 1, (lds_char*)lds_k1, (lds_char*)lds_v1, (lds_char*)lds_k0, (lds_char*)lds_v0);
    }

    const auto page_of = [&](int i) {
        const int j = kPrefillStep * (s0 + i / NP) + p0 + i % NP;
        return j < kPrefillStep * s1 && j < span.pages ? span.page(j) : -1;
    };
    const bool left = Q8 && range.left<D>(p, w.b, w.h, vref, page_of);
    float ls[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int row = row0 + 16 * rb + n16;
        float sum = accl[rb][0], &l = ls[rb];
        l = sum;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += fabsf(acc[rb][db][i]);
        if (__any(row < rows && !(sum <= kMostSum)) || left) {
            exact_keys<D, F16, Q8>(p, w.b, w.h, p.q + row_at(rb, p.q_batch, p.q_tok, p.q_head), sight_of(p, w.e, query[rb]), page_of, acc[rb], m[rb], l);
        } else if (Q8 && vacc != INT_MIN) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[rb][db][i] = ldexpf(acc[rb][db][i], vacc);
        }
    }
    if constexpr (KG == 2) {
        // the second group's state through LDS to the first's: m = max, l and O weighed by 2^(m_i - m)
        constexpr int HAND = DB * 4 * 64 * 4;
        static_assert(RB == 1 && 2 * HAND <= TILE, "two waves' O^T in a buffer of K");
        __shared__ float lds_ml[4][2][64];
        auto const x = (__attribute__((address_space(3))) float*)((lds_char*)(wv & 2 ? lds_k1 : lds_k0) + (wv & 1) * HAND) + lane;
        __syncthreads();  // the buffers are free
        if (kg == 1) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[(db * 4 + i) * 64] = acc[0][db][i];
            lds_ml[wv & 3][0][lane] = m[0];
            lds_ml[wv & 3][1][lane] = ls[0];
        }
        __syncthreads();
        if (kg == 1) return;
        const float m1 = lds_ml[wv][0][lane], l1 = lds_ml[wv][1][lane], mt = __builtin_elementwise_maximum(m[0], m1);
        const float a0 = m[0] == -INFINITY ? 0.0f : exp2_fast(m[0] - mt), a1 = m1 == -INFINITY ? 0.0f : exp2_fast(m1 - mt);
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[0][db][i] = acc[0][db][i] * a0 + x[(db * 4 + i) * 64] * a1;
        ls[0] = ls[0] * a0 + l1 * a1;
        m[0] = mt;
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int row = row0 + 16 * rb + n16;
        const float l = ls[rb];
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
        const bool any = sight_of(p, w.e, query[rb]).any;
        uint16_t* const orow = p.out + row_at(rb, p.o_batch, p.o_tok, p.o_head);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            float o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = any ? acc[rb][db][i] * inv : 0.0f;
            *reinterpret_cast<uint2*>(orow + 16 * db + 4 * g) = make_uint2(E::pack_p(o[0], o[1]), E::pack_p(o[2], o[3]));
        }
    }
}

template <bool F16, bool Q8, int RB, int KG>
int prefill_of(const BatchAttn& p, int D, hipStream_t stream) {
    const dim3 grid(unsigned(p.slots)), block(256 * KG);
    if (D == 64) hipLaunchKernelGGL((batch_prefill_kernel<64, F16, Q8, RB, KG>), grid, block, 0, stream, p);
    else if (D == 128) hipLaunchKernelGGL((batch_prefill_kernel<128, F16, Q8, RB, KG>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((batch_prefill_kernel<256, F16, Q8, RB, KG>), grid, block, 0, stream, p);
    GENLLM_LAUNCH_CHECK("batch_prefill_kernel");
    return GENLLM_OK;
}
template <int RB, int KG>
int prefill_rows(const BatchAttn& p, int D, bool f16, hipStream_t s) {
    return f16 ? p.k_scales ? prefill_of<true, true, RB, KG>(p, D, s) : prefill_of<true, false, RB, KG>(p, D, s)
               : p.k_scales ? prefill_of<false, true, RB, KG>(p, D, s) : prefill_of<false, false, RB, KG>(p, D, s);
}

}  // namespace

int launch_batch_prefill(const BatchAttn& p, int tile_rows, int D, bool f16, hipStream_t stream) {
    return tile_rows == 64 ? prefill_rows<1, 2>(p, D, f16, stream) : prefill_rows<2, 1>(p, D, f16, stream);
}

}  // namespace genllm
