// paged_batch.hip -- attention of a padded batch over paged caches, for few rows: the
// split kernel and the merge; and the entry point.
//
//   out[b, i, h] = sum_t softmax_t(scale q.k_t) v_t      over the keys t that the query
//   at p = n_cached[b] - q_lens[b] + i sees: t <= p, and t > p - window or t < sinks
//
// Rows are the (query, q head) pairs of a kv head, at most 16 here: the columns of the
// MFMA tiles, so that K and V are read once for all of them.  A wave takes two pages (32
// keys) a step:
//   S^T = K Q^T   v_mfma 16x16x32: K straight from memory, 16 bytes to a lane.  From 8-bit
//        pages they are 16 dims of a token (the dims of a k-step are in the order that
//        makes them so; Q follows), converted two at a time without loss; the page's scale
//        is part of the factor that takes the scores to log2 units.
//   O^T += V^T P^T   16x16x32 over both pages: lane (row, g) has the probabilities of
//        tokens 4g..4g+3 of either page, V^T comes from LDS by transposing reads.
// From 8-bit pages V's codes are fp16 values and P is rounded to fp16 (11 bits), whatever
// q's type is: the scale of a page is taken relative to a reference of the wave, which
// follows the largest as the running maximum does.  From bf16 pages P is split into two
// bf16 parts (16 bits).  fp16 in two parts as well would leave bf16 results as far from 64-bit ones
// as they are, by their own rounding (relative 1.7e-3), fp16 ones 2.1e-4 in place of 2.4e-4,
// and takes time: 64 sequences of up to 4096 tokens 55.0 -> 57.6 us, six drafts of 4 queries
// 10.4 -> 12.0, one token after 300 7.7 -> 8.5.  The sum of a row's
// probabilities comes from one more MFMA with ones, so from the same rounded values.
//
// Sequences of a batch are unlike in length, so workgroups are given equal numbers of
// steps, not equal shares of a sequence: each finds its part from the lengths on the device
// (find_work).
//
// Long contexts are bound by memory: one token each of 64 sequences of up to 4096 tokens (8 kv heads
// of 128, 8-bit pages) 55 us a call, 5.0 TB/s, as a large copy; one of 131072 tokens 51 us, 5.3 TB/s.
// Short ones are bound by launches and by loads after each other (lengths, ids, rows): 300
// tokens 7.7 us, 8192 in a split and a merge launch 11.2 (among other calls of its own; 12.5 to 13 over
// three sets of inputs in turn).  Eight waves to a workgroup in place
// of four made no difference there (600 tokens 9.2 us both ways).  At D = 256 over fp16 pages two
// registers go to scratch memory.
#include <algorithm>
#include <climits>
#include <cmath>
#include <string>

#include "paged_batch.hpp"
#include "rows.hpp"
#include "sequences.hpp"

namespace genllm {

namespace {

constexpr int kRows = kDecodeRows;
constexpr int kStep = kDecodeStep;
constexpr int kWaves = 4;
constexpr int kNonTemporal = 2;

typedef int i32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ i32x2_t ds_read_tr8(const lds_char* p) {
    return __builtin_amdgcn_ds_read_tr8_b64_v2i32(reinterpret_cast<__attribute__((address_space(3))) i32x2_t*>(const_cast<lds_char*>(p)));
}

// The 16-byte chunk of row t of page pp that lies at chunk position c of its LDS row is
// c ^ swizzle: the transposing reads of a half wave (rows 0-3 and 8-11, or 4-7 and 12-15,
// of both pages in 8 bits, of one in 16) then cover all banks once.
template <int RB, bool Q8>
__device__ __forceinline__ int v_swizzle(int t, int pp) {
    if constexpr (Q8) {
        constexpr int b = RB == 16 ? 4 : RB == 8 ? 3 : 2;  // log2(RB)
        return (t & 3) >> (4 - b) | pp << (b - 2) | (t >> 3) << (b - 1);
    } else {
        return RB == 8 ? 2 * (((t & 3) >> 1) | (t >> 3) << 1) : 2 * ((t & 3) | (t >> 3) << 2);
    }
}

// The loads of a step in flight, and what its pages are.
template <int D, bool Q8>
struct Step {
    static constexpr int kLoads = D * (Q8 ? 1 : 2) / 64;  // 16-byte loads of a page and kind
    uint4 k[kStep][kLoads], v[kStep][kLoads];
    int first[kStep];  // the pages' first tokens
    int vid[kStep];
    int at;  // the lane that knows the first page
};

// The next step's loads in flight beside this one's, where that leaves the registers for
// the workgroups above.
template <int D, bool Q8>
constexpr bool kAheadOf = D * (Q8 ? 1 : 2) <= 128;

template <int D, bool F16, bool Q8>
__global__ __launch_bounds__(kWaves * 64, resident(D)) void batch_decode_kernel(BatchAttn p) {
    using E = Elem<F16>;                 // q, out
    using EV = Elem<F16 || Q8>;          // P and V as the MFMA takes them
    constexpr int ES = Q8 ? 1 : 2;
    constexpr int KS = D / 32, DB = D / 16;
    constexpr int ROWB = D * ES, RB = ROWB / 16;  // bytes and 16-byte chunks of a token's row
    constexpr int LD = Step<D, Q8>::kLoads;
    constexpr bool kTwoParts = !F16 && !Q8;
    constexpr int VLDS = kStep * kPage * ROWB;
    constexpr int HAND = DB * 4 * 64 * 4;  // bytes of a wave's O^T
    constexpr int LDS = kWaves * VLDS > 2 * HAND ? kWaves * VLDS : 2 * HAND;
    __shared__ __attribute__((aligned(16))) char lds[LDS];
    __shared__ float lds_ml[2][2][64];

    prefetch_kernargs<sizeof(BatchAttn)>();
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, g = lane >> 4;
    Work w;
    if (!find_work<kRows, kStep>(p, int(blockIdx.x), w)) return;
    put_header(p, w);
    const int rows = w.e.ql * p.G;
    // the row's query; its addresses are formed where they are used: held through the
    // loop they cost the registers of a workgroup per CU
    const int query = min(n16, rows - 1) / p.G;
    const auto row_at = [&](int64_t batch, int64_t tok, int64_t head) {
        int r = min(n16, rows - 1);
        __asm__ volatile("" : "+v"(r));
        return w.b * batch + query * tok + (w.h * p.G + r - query * p.G) * head;
    };

    // Q^T operands: k-step 2 j + i of 8-bit keys is dims 64 j + 16 g + 8 i, of 16-bit ones 32 ks + 8 g
    uint4 qb[KS];
    const uint16_t* const qrow = p.q + row_at(p.q_batch, p.q_tok, p.q_head);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int d = Q8 ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1) : 32 * ks + 8 * g;
        qb[ks] = *reinterpret_cast<const uint4*>(qrow + d);
        if (n16 >= rows) qb[ks] = make_uint4(0, 0, 0, 0);
    }

    const TileKeys keys = tile_keys<kRows>(p, w.e, 0);
    const Span span = span_of(p, keys.first, keys.end);
    const int steps = (span.pages + kStep - 1) / kStep;
    const int s0 = int(int64_t(steps) * w.sp / w.ns), s1 = int(int64_t(steps) * (w.sp + 1) / w.ns);
    const int mine = s1 - s0 - wv > 0 ? (s1 - s0 - wv + kWaves - 1) / kWaves : 0;  // this wave's steps
    // keys from clear_from on and below clear_to are seen by every row
    const int first_pos = keys.first, last_pos = w.e.n - 1;
    const int clear_from = last_pos - p.window + 1;

    f32x4_t acc[DB], accl = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr float kBelow = kHead<F16 || Q8>;
    float m = -INFINITY, nm = 0.0f, th = -INFINITY;  // kBelow under the row's maximum, its negative (0 while there is none), where it grows
    int vref = INT_MIN;
    ScaleRange range;
    lds_char* const vt = (lds_char*)lds + wv * VLDS;

    const int k_off = n16 * p.k_tok + 16 * g;
    const int v_off = (lane / RB) * p.v_tok + 16 * (lane % RB);
    PageInfo info;
    const auto look_up = [&](int block) {  // lane i: page i % 2 of the wave's step block + i / 2
        const int j = kStep * (s0 + wv + kWaves * (block + (lane >> 1))) + (lane & 1);
        const bool there = block + (lane >> 1) < mine && j < span.pages;
        info = page_info<Q8>(p, w.b, w.h, span.page(j), there);
    };
    const auto load = [&](int i, int at, Step<D, Q8>& s) {  // step i of the wave; its pages are in lanes 2 at, 2 at + 1
        s.at = 2 * at;
#pragma unroll
        for (int pp = 0; pp < kStep; ++pp) {
            const int j = kStep * (s0 + wv + kWaves * i) + pp, from = 2 * at + pp;
            s.first[pp] = j < span.pages ? span.page(j) * kPage : 1 << 30;
            const int kid = __builtin_amdgcn_readlane(info.kid, from), vid = __builtin_amdgcn_readlane(info.vid, from);
            s.vid[pp] = vid;
            const int valid = kid < 0 ? 0 : min(w.e.n - s.first[pp], kPage);  // rows behind the cache's end read as zeros
            const char* const kb = p.k_pool + (kid < 0 ? 0 : kid) * p.k_block + int64_t(w.h) * p.k_head;
            const char* const vb = p.v_pool + (kid < 0 ? 0 : vid) * p.v_block + int64_t(w.h) * p.v_head;
            const auto rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(kb), 0, valid > 0 ? (valid - 1) * p.k_tok + ROWB : 0, kBufferFlags);
            const auto rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(vb), 0, valid > 0 ? (valid - 1) * p.v_tok + ROWB : 0, kBufferFlags);
#pragma unroll
            for (int e = 0; e < LD; ++e)
                s.k[pp][e] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rk, k_off + 64 * e, 0, kNonTemporal));
#pragma unroll
            for (int e = 0; e < LD; ++e)
                s.v[pp][e] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rv, v_off, e * (64 / RB) * p.v_tok, kNonTemporal));
        }
    };
    const auto compute = [&](const Step<D, Q8>& s) {
        // read here, not with the loads: the scales come after the ids, as K and V do
        float kf[kStep];
        int ve[kStep];
#pragma unroll
        for (int pp = 0; pp < kStep; ++pp) {
            const int kb = __builtin_amdgcn_readlane(info.kb, s.at + pp), vb = __builtin_amdgcn_readlane(info.vb, s.at + pp);
            kf[pp] = score_factor<Q8>(p, s.vid[pp], kb, vb);
            ve[pp] = vb - 127;
        }
        // V's rows to LDS, at [page][token][chunk ^ swizzle]
#pragma unroll
        for (int pp = 0; pp < kStep; ++pp)
#pragma unroll
            for (int e = 0; e < LD; ++e) {
                const int t = e * (64 / RB) + lane / RB, c = (lane % RB) ^ v_swizzle<RB, Q8>(t, pp);
                *reinterpret_cast<__attribute__((address_space(3))) u32x4_t*>(vt + (pp * kPage + t) * ROWB + 16 * c) =
                    __builtin_bit_cast(u32x4_t, s.v[pp][e]);
            }
        f32x4_t x[kStep];
#pragma unroll
        for (int pp = 0; pp < kStep; ++pp) {
            x[pp] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int e = 0; e < LD; ++e) {
                const uint4 u = s.k[pp][e];
                if constexpr (Q8) {
                    x[pp] = E::mma32(f8_octet<F16>(u.x, u.y, 1.0f, 1.0f), qb[2 * e], x[pp]);
                    x[pp] = E::mma32(f8_octet<F16>(u.z, u.w, 1.0f, 1.0f), qb[2 * e + 1], x[pp]);
                } else {
                    x[pp] = E::mma32(u, qb[e], x[pp]);
                }
            }
        }
#pragma unroll
        for (int pp = 0; pp < kStep; ++pp) {
            const int last = s.first[pp] + kPage - 1;
            if (last > first_pos || (s.first[pp] < clear_from && last >= p.sinks)) {  // some row does not see all of it
                const Sight see = sight_of(p, w.e, query);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[pp][i] = see(p, s.first[pp] + 4 * g + i) ? x[pp][i] : -INFINITY;
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int pp = 0; pp < kStep; ++pp) {
            const float a = __builtin_elementwise_maximum(__builtin_elementwise_maximum(x[pp][0], x[pp][1]),
                                                          __builtin_elementwise_maximum(x[pp][2], x[pp][3]));
            mx = __builtin_elementwise_maximum(mx, a * kf[pp]);
        }
        if (__any(mx > th)) {
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const bool grow = mx > th;
            const float mn = grow ? mx - kBelow : m, alpha = grow ? exp2_fast(m - mn) : 1.0f;
            m = mn;
            nm = grow ? -mn : nm;
            th = grow ? mn + (kBelow + kLazy) : th;
            accl *= alpha;
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] *= alpha;
        }
        float vs[kStep] = {1.0f, 1.0f};
        if constexpr (Q8) {
            const int most = max(ve[0], ve[1]);
            if (most > (vref == INT_MIN ? vref : vref + kScaleLead)) {  // wave-uniform
                const float f = vref == INT_MIN ? 0.0f : power_of_two(vref - most);
#pragma unroll
                for (int db = 0; db < DB; ++db) acc[db] *= f;
                vref = most;
            }
            vs[0] = power_of_two(ve[0] - vref), vs[1] = power_of_two(ve[1] - vref);
        }
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = exp2_fast(__builtin_fmaf(x[i >> 2][i & 3], kf[i >> 2], nm));
        const uint4 pb = make_uint4(EV::pack_p(e[0], e[1]), EV::pack_p(e[2], e[3]), EV::pack_p(e[4], e[5]), EV::pack_p(e[6], e[7]));
        uint4 pl;  // what the first part leaves
        if constexpr (kTwoParts) {
            pl = make_uint4(EV::pack_p(e[0] - EV::lo(pb.x), e[1] - EV::hi(pb.x)), EV::pack_p(e[2] - EV::lo(pb.y), e[3] - EV::hi(pb.y)),
                            EV::pack_p(e[4] - EV::lo(pb.z), e[5] - EV::hi(pb.z)), EV::pack_p(e[6] - EV::lo(pb.w), e[7] - EV::hi(pb.w)));
        }
        const uint32_t one2 = EV::pack_p(1.0f, 1.0f);
        const uint4 ones = make_uint4(one2, one2, one2, one2);
        accl = EV::mma32(ones, pb, accl);
        if constexpr (kTwoParts) accl = EV::mma32(ones, pl, accl);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            uint4 a;
            if constexpr (Q8) {
                const int r = n16 >> 1, pp = r >> 2, t = 4 * g + (r & 3), c = db ^ v_swizzle<RB, Q8>(t, pp);
                const i32x2_t u = ds_read_tr8(vt + (pp * kPage + t) * ROWB + 16 * c + 8 * (n16 & 1));
                a = f8_octet<true>(uint32_t(u.x), uint32_t(u.y), vs[0], vs[1]);
            } else {
                const int t = 4 * g + (n16 >> 2), c = (2 * db + ((n16 & 3) >> 1)) ^ v_swizzle<RB, Q8>(t, 0);
                const s16x4_t u[2] = {ds_read_tr16(vt + t * ROWB + 16 * c + 8 * (n16 & 1)),
                                      ds_read_tr16(vt + (kPage + t) * ROWB + 16 * c + 8 * (n16 & 1))};
                a = __builtin_bit_cast(uint4, u);
            }
            acc[db] = EV::mma32(a, pb, acc[db]);
            if constexpr (kTwoParts) acc[db] = EV::mma32(a, pl, acc[db]);
        }
    };

    for (int block = 0; block < mine; block += 32) {
        look_up(block);
        const int end = min(mine - block, 32);
        Step<D, Q8> s;
        if constexpr (kAheadOf<D, Q8>) {
            // not unrolled by two, which would save the copies: that took the registers of the
            // third workgroup (64 sequences of 4096 tokens 57.0 -> 60.5 us)
            load(block, 0, s);
            for (int i = 0; i + 1 < end; ++i) {
                Step<D, Q8> next;
                load(block + i + 1, i + 1, next);
                compute(s);
                s = next;
            }
            compute(s);
        } else {
            for (int i = 0; i < end; ++i) {
                load(block + i, i, s);
                compute(s);
            }
        }
        if constexpr (Q8) range.add(info);
    }

    float l = accl[0];
    {
        float sum = l;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += fabsf(acc[db][i]);
        const auto page_of = [&](int i) {
            const int j = kStep * (s0 + wv + kWaves * (i >> 1)) + (i & 1);
            return (i >> 1) < mine && j < span.pages ? span.page(j) : -1;
        };
        if (__any(n16 < rows && !(sum <= kMostSum)) || (Q8 && range.left<D>(p, w.b, w.h, vref, page_of))) {
            exact_keys<D, F16, Q8>(p, w.b, w.h, p.q + row_at(p.q_batch, p.q_tok, p.q_head), sight_of(p, w.e, query), page_of, acc, m, l);
        } else if (Q8 && vref != INT_MIN) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[db][i] = ldexpf(acc[db][i], vref);
        }
    }

    // The waves of the workgroup, two into two, then one into one: m = max, l and O
    // weighed by 2^(m_i - m) (a wave without keys has m = -inf, weight 0).
    const auto slot = [&](int i) { return (__attribute__((address_space(3))) float*)((lds_char*)lds + i * HAND) + lane; };
#pragma unroll
    for (int half = kWaves / 2; half >= 1; half /= 2) {
        __syncthreads();  // the LDS is free
        if (wv >= half && wv < 2 * half) {
            const auto x = slot(wv - half);
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[(db * 4 + i) * 64] = acc[db][i];
            lds_ml[wv - half][0][lane] = m;
            lds_ml[wv - half][1][lane] = l;
        }
        __syncthreads();
        if (wv < half) {
            const auto x = slot(wv);
            const float m1 = lds_ml[wv][0][lane], l1 = lds_ml[wv][1][lane], mt = __builtin_elementwise_maximum(m, m1);
            const float a0 = m == -INFINITY ? 0.0f : exp2_fast(m - mt), a1 = m1 == -INFINITY ? 0.0f : exp2_fast(m1 - mt);
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[db][i] = acc[db][i] * a0 + x[(db * 4 + i) * 64] * a1;
            l = l * a0 + l1 * a1;
            m = mt;
        }
    }
    if (wv != 0 || n16 >= rows) return;
    if (w.ns > 1) {
        const int64_t at = int64_t(blockIdx.x) * kRows + n16;
        float* const po = partial_rows(p) + at * D + 4 * g;
#pragma unroll
        for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4_t*>(po + 16 * db) = acc[db];
        if (g == 0) *reinterpret_cast<float2*>(partial_rows(p) + int64_t(p.slots) * kRows * D + 2 * at) = make_float2(m, l);
        return;
    }
    const bool any = sight_of(p, w.e, query).any;
    const float inv = 1.0f / l;
    uint16_t* const orow = p.out + row_at(p.o_batch, p.o_tok, p.o_head);
#pragma unroll
    for (int db = 0; db < DB; ++db) {
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = any ? acc[db][i] * inv : 0.0f;
        *reinterpret_cast<uint2*>(orow + 16 * db + 4 * g) = make_uint2(E::pack_p(o[0], o[1]), E::pack_p(o[2], o[3]));
    }
}


// Merge of the splits: M = max m_s, l = sum l_s 2^(m_s - M), o = sum o_s 2^(m_s - M) / l.
// A lane has 4 dims of a row; SG groups of D / 4 lanes share a row's splits (SG = 1: a row
// per group).  Entries with one split were written by their workgroup.
// A row's splits are shared by four waves where there are many of them on average.
// kMergeU splits at once (whole calls with 8 of them, 4, 2: 2 x 512 queries on 8192 tokens 151.1 us,
// 149.7, 149.0; one token after 131072 50.6, 50.7, 51.6).
constexpr int kMergeU = 4, kMergeWide = 16;
template <int D, bool F16, int ROWS, int SG, int THREADS>
__global__ __launch_bounds__(THREADS) void batch_merge_kernel(BatchAttn p, int row_blocks) {
    using E = Elem<F16>;
    constexpr int LR = D / 4, GROUPS = THREADS / LR, RPB = GROUPS / SG;
    static_assert(GROUPS % SG == 0 && RPB >= 1, "whole rows");
    __shared__ float lds_o[SG > 1 ? GROUPS : 1][D], lds_ml[GROUPS][2];
    unsigned rest = blockIdx.x;
    const int rb = int(rest % unsigned(row_blocks));
    rest /= unsigned(row_blocks);
    const int h = int(rest % unsigned(p.Hkv)), unit = int(rest / unsigned(p.Hkv));
    const int b = unit / p.tiles_max, tile = unit - b * p.tiles_max;
    const Header of = reinterpret_cast<const Header*>(p.partial)[unit];
    const Entry e = entry_of(p, b);
    const int group = int(threadIdx.x) / LR, d = 4 * (int(threadIdx.x) % LR);
    const int in_tile = rb * RPB + group / SG, sg = group % SG;
    const int row = tile * ROWS + in_tile;
    if (tile * ROWS >= e.ql * p.G || of.ns < 2) return;  // no rows and no header, or one split
    const bool there = in_tile < ROWS && row < e.ql * p.G;
    if (SG > 1 && !there) return;  // RPB is 1 then: the whole workgroup
    float M = -INFINITY, L = 0.0f;
    f32x4_t o = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const float* const po = partial_rows(p);
    const float2* const ml = reinterpret_cast<const float2*>(po + int64_t(p.slots) * ROWS * D);
    for (int s0 = sg; there && s0 < of.ns; s0 += SG * kMergeU) {
        f32x4_t x[kMergeU];
        float2 y[kMergeU];
#pragma unroll
        for (int u = 0; u < kMergeU; ++u) {
            const int s = s0 + SG * u;
            const int64_t at = (int64_t(of.base) + int64_t(s) * p.Hkv + h) * ROWS + in_tile;
            x[u] = s < of.ns ? *reinterpret_cast<const f32x4_t*>(po + at * D + d) : f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            y[u] = s < of.ns ? ml[at] : make_float2(-INFINITY, 0.0f);
        }
        float mn = M;
#pragma unroll
        for (int u = 0; u < kMergeU; ++u) mn = __builtin_elementwise_maximum(mn, y[u].x);
        const float a = M == -INFINITY ? 0.0f : exp2_fast(M - mn);
        L *= a;
        o *= a;
#pragma unroll
        for (int u = 0; u < kMergeU; ++u) {
            const float f = y[u].x == -INFINITY ? 0.0f : exp2_fast(y[u].x - mn);
            L += y[u].y * f;
            o += x[u] * f;
        }
        M = mn;
    }
    if constexpr (SG > 1) {
        *reinterpret_cast<f32x4_t*>(&lds_o[group][d]) = o;
        if (d == 0) lds_ml[group][0] = M, lds_ml[group][1] = L;
        __syncthreads();
        if (group > 0) return;
        float all = M;
#pragma unroll
        for (int i = 1; i < SG; ++i) all = __builtin_elementwise_maximum(all, lds_ml[i][0]);
        const float a = M == -INFINITY ? 0.0f : exp2_fast(M - all);
        L *= a;
        o *= a;
#pragma unroll
        for (int i = 1; i < SG; ++i) {
            const float f = lds_ml[i][0] == -INFINITY ? 0.0f : exp2_fast(lds_ml[i][0] - all);
            L += lds_ml[i][1] * f;
            o += *reinterpret_cast<const f32x4_t*>(&lds_o[i][d]) * f;
        }
    }
    if (!there) return;
    const int query = row / p.G, head = h * p.G + row % p.G;
    const bool any = sight_of(p, e, query).any;
    const float inv = 1.0f / L;
    o *= inv;
    uint16_t* const to = p.out + b * p.o_batch + query * p.o_tok + head * p.o_head + d;
    *reinterpret_cast<uint2*>(to) = any ? make_uint2(E::pack_p(o[0], o[1]), E::pack_p(o[2], o[3])) : make_uint2(0, 0);
}

template <bool F16, bool Q8>
int decode_of(const BatchAttn& p, int D, hipStream_t stream) {
    const dim3 grid(unsigned(p.slots)), block(kWaves * 64);
    if (D == 64) hipLaunchKernelGGL((batch_decode_kernel<64, F16, Q8>), grid, block, 0, stream, p);
    else if (D == 128) hipLaunchKernelGGL((batch_decode_kernel<128, F16, Q8>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((batch_decode_kernel<256, F16, Q8>), grid, block, 0, stream, p);
    GENLLM_LAUNCH_CHECK("batch_decode_kernel");
    return GENLLM_OK;
}

template <int D, bool F16>
int merge_of(const BatchAttn& p, const BatchPlan& plan, hipStream_t stream) {
    const int rows = int(std::min<int64_t>(plan.rows, int64_t(p.S) * p.G));  // of a tile that may be there
    const auto go = [&](auto kernel, int threads, int per_block) {
        const int blocks = (rows + per_block - 1) / per_block;
        hipLaunchKernelGGL(kernel, dim3(unsigned(plan.tiles * blocks)), dim3(threads), 0, stream, p, blocks);
    };
    constexpr int G64 = 64 / (D / 4), G256 = 256 / (D / 4);
    if (plan.decode && plan.tiles * kMergeWide <= plan.target)
        go(batch_merge_kernel<D, F16, 16, G256, 256>, 256, 1);
    else if (plan.decode)
        go(batch_merge_kernel<D, F16, 16, G64, 64>, 64, 1);
    else if (plan.rows == 64)
        go(batch_merge_kernel<D, F16, 64, 1, 256>, 256, G256);
    else
        go(batch_merge_kernel<D, F16, 128, 1, 256>, 256, G256);
    GENLLM_LAUNCH_CHECK("batch_merge_kernel");
    return GENLLM_OK;
}

}  // namespace

int launch_batch_decode(const BatchAttn& p, int D, bool f16, hipStream_t stream) {
    return f16 ? p.k_scales ? decode_of<true, true>(p, D, stream) : decode_of<true, false>(p, D, stream)
               : p.k_scales ? decode_of<false, true>(p, D, stream) : decode_of<false, false>(p, D, stream);
}

}  // namespace genllm

using namespace genllm;

extern "C" size_t genllm_paged_attention_batch_workspace_bytes(int32_t batch, int32_t seq_len, int32_t n_q_heads, int32_t n_kv_heads,
                                                               int32_t head_dim, int32_t max_pages) {
    const BatchSizes z{batch, seq_len, n_q_heads, n_kv_heads, head_dim, max_pages};
    if (z.refused() || z.empty() || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return 0;
    const BatchPlan plan = plan_of(z);
    return plan.slots > kMostWorkgroups ? 0 : workspace_of(plan, batch, head_dim);
}

extern "C" int genllm_paged_attention_batch(
    const void* q, int64_t q_batch_stride, int64_t q_tok_stride, int64_t q_head_stride, void* out, int64_t o_batch_stride,
    int64_t o_tok_stride, int64_t o_head_stride, const void* k_pool, int64_t kp_block_stride, int64_t kp_tok_stride,
    int64_t kp_head_stride, const void* v_pool, int64_t vp_block_stride, int64_t vp_tok_stride, int64_t vp_head_stride,
    const uint8_t* k_scales, const uint8_t* v_scales, int32_t n_blocks, const int32_t* k_ids, int64_t k_ids_stride,
    const int32_t* v_ids, int64_t v_ids_stride, int32_t max_pages, const int32_t* n_cached, const int32_t* q_lens, int32_t batch,
    int32_t seq_len, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t dtype, float scale, int32_t causal,
    int32_t window, int32_t sinks, void* workspace, size_t workspace_bytes, void* stream) {
    const auto refuse = [](int code, const std::string& why) { return fail(code, "paged_attention_batch: " + why); };
    const BatchSizes z{batch, seq_len, n_q_heads, n_kv_heads, head_dim, max_pages};
    if (const char* why = z.refused()) return refuse(GENLLM_ERR_INVALID, why);
    if (n_blocks < 0) return refuse(GENLLM_ERR_INVALID, "negative size");
    if (n_blocks == 0 && !z.empty()) return refuse(GENLLM_ERR_INVALID, "a pool without blocks");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return refuse(GENLLM_ERR_UNSUPPORTED, "head_dim 64, 128 or 256");
    if (dtype != GENLLM_DTYPE_BF16 && dtype != GENLLM_DTYPE_F16) return refuse(GENLLM_ERR_UNSUPPORTED, "bf16 or fp16 elements");
    if (!(scale >= 0.0f) || !std::isfinite(scale * kLog2e)) return refuse(GENLLM_ERR_INVALID, "the scale must be finite and not negative");
    if (window < 0 || sinks < 0) return refuse(GENLLM_ERR_INVALID, "negative window or sinks");
    if (window > 0 && !causal) return refuse(GENLLM_ERR_INVALID, "a window goes with causal attention");
    if ((k_scales != nullptr) != (v_scales != nullptr)) return refuse(GENLLM_ERR_INVALID, "k_scales and v_scales go together");
    if (z.empty()) return GENLLM_OK;
    if (!q || !out || !k_pool || !v_pool || (max_pages > 0 && (!k_ids || !v_ids)) || !n_cached) return refuse(GENLLM_ERR_INVALID, "null pointer");
    const bool q8 = k_scales != nullptr;
    const int64_t es = q8 ? 1 : 2, row = head_dim * es;
    const auto one = [](int64_t stride, int64_t n) { return n > 1 ? stride : 0; };  // the stride of a dim of one never matters
    q_batch_stride = one(q_batch_stride, batch), o_batch_stride = one(o_batch_stride, batch);
    q_tok_stride = one(q_tok_stride, seq_len), o_tok_stride = one(o_tok_stride, seq_len);
    q_head_stride = one(q_head_stride, n_q_heads), o_head_stride = one(o_head_stride, n_q_heads);
    kp_block_stride = es * one(kp_block_stride, n_blocks), vp_block_stride = es * one(vp_block_stride, n_blocks);
    kp_head_stride = es * one(kp_head_stride, n_kv_heads), vp_head_stride = es * one(vp_head_stride, n_kv_heads);
    kp_tok_stride *= es, vp_tok_stride *= es;
    if (!aligned_to(q, 16) || !aligned_to(out, 16) || !aligned_to(k_pool, 16) || !aligned_to(v_pool, 16) ||
        ((q_batch_stride | q_tok_stride | q_head_stride | o_batch_stride | o_tok_stride | o_head_stride) & 7) ||
        ((kp_block_stride | kp_tok_stride | kp_head_stride | vp_block_stride | vp_tok_stride | vp_head_stride) & 15))
        return refuse(GENLLM_ERR_INVALID, "rows must be 16-byte aligned");
    if (!aligned_to(k_ids, 4) || !aligned_to(v_ids, 4) || !aligned_to(n_cached, 4) || !aligned_to(q_lens, 4))
        return refuse(GENLLM_ERR_INVALID, "a pointer is not aligned to its type");
    // a page's rows are read through 32-bit offsets, and those behind the cache's end by the size of what is read
    const auto page_rows = [&](int64_t tok, int64_t head) {
        return tok >= row && head >= 0 && tok < (1 << 26) && head < (int64_t(1) << 31) / n_kv_heads;
    };
    if (!page_rows(kp_tok_stride, kp_head_stride) || !page_rows(vp_tok_stride, vp_head_stride))
        return refuse(GENLLM_ERR_INVALID, "a pool's token rows must follow each other within less than 2^26 bytes, a block's heads within 2^31");

    const BatchPlan plan = plan_of(z);
    if (plan.slots > kMostWorkgroups) return refuse(GENLLM_ERR_INVALID, "more rows than one launch takes");
    const size_t need = workspace_of(plan, batch, head_dim);
    if (need && (!workspace || workspace_bytes < need || !aligned_to(workspace, 16)))
        return refuse(GENLLM_ERR_INVALID, "a 16-byte aligned workspace of " + std::to_string(need) + " bytes is needed");

    BatchAttn p;
    p.n_cached = n_cached, p.q_lens = q_lens;
    p.q = static_cast<const uint16_t*>(q), p.q_batch = q_batch_stride, p.q_tok = q_tok_stride, p.q_head = q_head_stride;
    p.out = static_cast<uint16_t*>(out), p.o_batch = o_batch_stride, p.o_tok = o_tok_stride, p.o_head = o_head_stride;
    p.k_pool = static_cast<const char*>(k_pool), p.v_pool = static_cast<const char*>(v_pool);
    p.k_block = kp_block_stride, p.v_block = vp_block_stride;
    p.k_tok = int32_t(kp_tok_stride), p.k_head = int32_t(kp_head_stride), p.v_tok = int32_t(vp_tok_stride), p.v_head = int32_t(vp_head_stride);
    p.k_scales = k_scales, p.v_scales = v_scales;
    p.k_ids = k_ids, p.v_ids = v_ids, p.k_ids_row = one(k_ids_stride, batch), p.v_ids_row = one(v_ids_stride, batch);
    p.B = batch, p.S = seq_len, p.Hq = n_q_heads, p.Hkv = n_kv_heads, p.G = n_q_heads / n_kv_heads;
    p.blocks = n_blocks, p.capacity = max_pages * kPage;
    p.window = window > 0 ? std::min(window, kNoWindow) : kNoWindow, p.sinks = sinks, p.causal = causal != 0;
    p.c = std::max(scale * kLog2e, __FLT_MIN__);
    p.tiles_max = int32_t(plan.tiles_max), p.target = plan.target, p.least = plan.least, p.can_split = plan.can_split, p.paired = plan.paired && causal, p.slots = int32_t(plan.slots);
    p.partial = need ? static_cast<float*>(workspace) : nullptr;

    const auto rows_of = [&](const void* at, int64_t b, int64_t t, int64_t h) {
        Rows r = Rows::whole(at, int64_t(head_dim) * 2);
        r.n[0] = batch, r.n[1] = seq_len, r.n[2] = n_q_heads, r.stride[0] = 2 * b, r.stride[1] = 2 * t, r.stride[2] = 2 * h;
        return r;
    };
    const auto pool_of = [&](const void* at, int64_t b, int64_t t, int64_t h) {
        Rows r = Rows::whole(at, row);
        r.n[0] = n_blocks, r.n[1] = kPage, r.n[2] = n_kv_heads, r.stride[0] = b, r.stride[1] = t, r.stride[2] = h;
        return r;
    };
    const auto table = [&](const int32_t* at, int64_t stride) {
        Rows r = Rows::whole(at, int64_t(max_pages) * 4);
        r.n[0] = batch, r.stride[0] = 4 * stride;
        return r;
    };
    const NamedRows written[] = {{"out", rows_of(out, o_batch_stride, o_tok_stride, o_head_stride)},
                                 {"the workspace", Rows::whole(p.partial, int64_t(need))}};
    const NamedRows read[] = {{"q", rows_of(q, q_batch_stride, q_tok_stride, q_head_stride)},
                              {"k_pool", pool_of(k_pool, p.k_block, p.k_tok, p.k_head)},
                              {"v_pool", pool_of(v_pool, p.v_block, p.v_tok, p.v_head)},
                              {"k_scales", Rows::whole(k_scales, int64_t(n_blocks) * n_kv_heads)},
                              {"v_scales", Rows::whole(v_scales, int64_t(n_blocks) * n_kv_heads)},
                              {"k_ids", table(k_ids, p.k_ids_row)},
                              {"v_ids", table(v_ids, p.v_ids_row)},
                              {"n_cached", Rows::whole(n_cached, int64_t(batch) * 4)},
                              {"q_lens", Rows::whole(q_lens, int64_t(batch) * 4)}};
    // out may be q: a workgroup writes only rows that it alone has read, or the merge does
    const auto allowed = [&](const Rows& w, const Rows& r) { return r.p == static_cast<const char*>(q) && w.same_as(r); };
    const char *a, *b;
    if (find_overlap(written, read, allowed, a, b)) return refuse(GENLLM_ERR_INVALID, std::string(a) + " overlaps " + b);
    if (rows_shared_within(written[0].rows)) return refuse(GENLLM_ERR_INVALID, "rows of out share memory");

    const hipStream_t s = as_stream(stream);
    const bool f16 = dtype == GENLLM_DTYPE_F16;
    if (const int rc = plan.decode ? launch_batch_decode(p, head_dim, f16, s) : launch_batch_prefill(p, plan.rows, head_dim, f16, s)) return rc;
    if (!plan.can_split) return GENLLM_OK;
    if (f16) return head_dim == 64 ? merge_of<64, true>(p, plan, s) : head_dim == 128 ? merge_of<128, true>(p, plan, s) : merge_of<256, true>(p, plan, s);
    return head_dim == 64 ? merge_of<64, false>(p, plan, s) : head_dim == 128 ? merge_of<128, false>(p, plan, s) : merge_of<256, false>(p, plan, s);
}
