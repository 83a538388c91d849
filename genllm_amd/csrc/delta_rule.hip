// delta_rule.hip -- the gated delta rule, the memory of a hybrid model's
// linear layers.  Per value head h (key head h / (Hv / Hk)) a matrix S [Dk][Dv]
// in fp32 takes one token after another:
//
//   S <- alpha S          alpha = exp(g)
//   u  = beta (v - S^T k)
//   S <- S + k u^T
//   o  = scale S^T q
//
// q and k are the given ones or, with l2_eps >= 0, x / sqrt(sum x^2 + l2_eps);
// g and beta are given in fp32, or g = -exp(a_log) softplus(a + dt_bias) and
// beta = sigmoid(b) from elements.  1/sqrt(...) stays a factor beside the raw
// elements of a row, so that products with them have one exact operand.
//
// delta_recurrent_kernel runs the rule as written, the state in registers.
//
// Longer calls run in chunks of C = 64 tokens.  With G the running sum of g in a
// chunk, S0 the state before it and U the chunk's rows u:
//
//   (1 + L) U = diag(beta) (V - diag(e^G) K S0)      L_ij = beta_i e^(G_i - G_j) k_i.k_j, j < i
//   O  = scale (diag(e^G) Q S0 + P U)                P_ij = e^(G_i - G_j) q_i.k_j, j <= i
//   S1 = e^(G_last) S0 + K^T diag(e^(G_last - G)) U
//
// delta_chunk_prepare_kernel forms T = (1 + L)^-1 diag(beta), P and the factors
// of every chunk and head at once; delta_chunk_scan_kernel takes 16 columns of
// a head's state from chunk to chunk through the matrix cores.  The state and
// everything that enters it keep 24 bits there: an fp32 value is the exact sum
// of three bf16 parts (24 = 3 x 8 bits), q and k are one part (fp16: two, 11 bits),
// and the products of parts below 2^-24 are left out.  out is formed the same way
// and rounded once, so that it has the bits of the rule token by token.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "rows.hpp"
#include "sequences.hpp"

namespace genllm {

namespace {

struct Rows3 {  // an element of [batch][token][head][dim], strides in elements, dim dense
    const uint16_t* p = nullptr;
    int64_t batch = 0, tok = 0, head = 0;
};

struct DeltaParams {
    Rows3 q, k, v;
    uint16_t* out = nullptr;
    int64_t o_batch = 0, o_tok = 0, o_head = 0;
    const void* a = nullptr;  // [batch][token][Hv]: fp32 log decays, or elements when a_log is there
    const void* b = nullptr;
    int64_t a_batch = 0, a_tok = 0, b_batch = 0, b_tok = 0;
    const float* a_log = nullptr;
    const float* dt_bias = nullptr;
    float* state = nullptr;  // [n_states][Hv][Dk][Dv]
    Sequences seq;
    int32_t B = 0, Hk = 0, Hv = 0, G = 0, Dk = 0, Dv = 0;
    float scale = 0.0f, l2_eps = -1.0f;
};

// log decay and beta of one token and head, from what was loaded for them:
// elements, or fp32 values as they are
struct GateLoad {
    uint32_t a, b;
};
__device__ __forceinline__ GateLoad load_gates(const DeltaParams& p, int b, int64_t t, int h) {
    const int64_t ia = b * p.a_batch + t * p.a_tok + h, ib = b * p.b_batch + t * p.b_tok + h;
    if (p.a_log) return {static_cast<const uint16_t*>(p.a)[ia], static_cast<const uint16_t*>(p.b)[ib]};
    return {static_cast<const uint32_t*>(p.a)[ia], static_cast<const uint32_t*>(p.b)[ib]};
}
// rate = -exp(a_log[h]), bias = dt_bias[h], for elements
template <bool F16>
__device__ __forceinline__ void gates(const DeltaParams& p, const GateLoad& x, float rate, float bias, float& g, float& beta) {
    if (!p.a_log) {
        g = __uint_as_float(x.a);
        beta = __uint_as_float(x.b);
        return;
    }
    const float y = Elem<F16>::lo(x.a) + bias;
    // fmaxf drops a NaN: the sum keeps it through fabsf(y)
    g = rate * (fmaxf(y, 0.0f) + log1pf(expf(-fabsf(y))));
    beta = 1.0f / (1.0f + expf(-Elem<F16>::lo(x.b)));
}
__device__ __forceinline__ void gate_rates(const DeltaParams& p, int h, float& rate, float& bias) {
    rate = bias = 0.0f;
    if (p.a_log) rate = -expf(p.a_log[h]), bias = p.dt_bias[h];
}

// N consecutive elements (N = 4, 8 or 16), aligned to 2 N bytes up to 16
template <int N>
__device__ __forceinline__ void load_words(const uint16_t* p, uint32_t (&w)[N / 2]) {
    if constexpr (N == 4) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x, w[1] = u.y;
    } else {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) {
            const uint4 u = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
        }
    }
}
template <bool F16, int N>
__device__ __forceinline__ void unpack(const uint32_t (&w)[N / 2], float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) f[2 * i] = Elem<F16>::lo(w[i]), f[2 * i + 1] = Elem<F16>::hi(w[i]);
}

// 1 / sqrt(sum + eps), or 1 without a normalisation; the hardware's reciprocal
// root is off by one step of fp32 at most
__device__ __forceinline__ float l2_factor(float sum, float eps) {
    return eps < 0.0f ? 1.0f : __builtin_amdgcn_rsqf(sum + eps);
}

// The sum over the lanes with the same lane % CQ, CQ = 4 or 8: within rows of 16
// lanes by rotations, across them by exchanging rows and halves of the wave.
template <int CQ>
__device__ __forceinline__ float sum_of_groups(float x) {
    if constexpr (CQ == 4) x += dpp<0x124>(x);  // row_ror:4
    x += dpp<0x128>(x);                         // row_ror:8
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Tokens t0 .. t1 - 1 through 4 CQ columns of a head's state in one wave's
// registers: lane (rg, cq) = (lane / CQ, lane % CQ) holds rows rg NR .. + NR - 1
// of columns col .. + 3.  S^T k and S^T q of the state before the token are summed
// in one pass over the registers and one reduction over the row groups; then
//   u = beta (v - alpha S^T k),  o = scale (alpha S^T q + (k.q) u),
// and the state is updated.  At most 64 tokens: lane l forms the gates of token t0 +
// l for all.  A token's rows are loaded while the one before it runs.
template <int DK, int CQ, bool F16>
__device__ __forceinline__ void recur(const DeltaParams& p, f32x4_t (&s)[DK * CQ / 64], int b, int h, int col, int t0, int t1) {
    constexpr int NR = DK * CQ / 64;
    const int rg = int(threadIdx.x & 63) / CQ, hk = h / p.G;
    const uint16_t* const q = p.q.p + b * p.q.batch + hk * p.q.head + rg * NR;
    const uint16_t* const k = p.k.p + b * p.k.batch + hk * p.k.head + rg * NR;
    const uint16_t* const v = p.v.p + b * p.v.batch + h * p.v.head + col;
    uint16_t* const out = p.out + b * p.o_batch + h * p.o_head + col;
    struct Token {
        uint32_t k[NR / 2], q[NR / 2], v[2];
    };
    const auto load = [&](Token& x, int t) {
        load_words<NR>(k + t * p.k.tok, x.k);
        load_words<NR>(q + t * p.q.tok, x.q);
        load_words<4>(v + t * p.v.tok, x.v);
    };
    Token next;
    load(next, t0);
    float alphas, betas;
    {
        const int t = min(t0 + int(threadIdx.x & 63), t1 - 1);
        const GateLoad gate = load_gates(p, b, t, h);
        float rate, bias, g;
        gate_rates(p, h, rate, bias);
        gates<F16>(p, gate, rate, bias, g, betas);
        alphas = exp2_fast(kLog2e * g);
    }
    for (int t = t0; t < t1; ++t) {
        float kf[NR], qf[NR], vf[4];
        unpack<F16, NR>(next.k, kf);
        unpack<F16, NR>(next.q, qf);
        unpack<F16, 4>(next.v, vf);
        if (t + 1 < t1) load(next, t + 1);
        const float alpha = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(alphas), t - t0));
        const float beta = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(betas), t - t0));
        float r[11] = {};  // k.k, q.q, k.q, S^T k, S^T q
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            r[0] = __builtin_fmaf(kf[i], kf[i], r[0]);
            r[1] = __builtin_fmaf(qf[i], qf[i], r[1]);
            r[2] = __builtin_fmaf(kf[i], qf[i], r[2]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                r[3 + c] = __builtin_fmaf(s[i][c], kf[i], r[3 + c]);
                r[7 + c] = __builtin_fmaf(s[i][c], qf[i], r[7 + c]);
            }
        }
#pragma unroll
        for (int j = 0; j < 11; ++j) r[j] = sum_of_groups<CQ>(r[j]);
        const float rk = l2_factor(r[0], p.l2_eps), rq = p.scale * l2_factor(r[1], p.l2_eps);
        const float kq = r[2] * rk;
        float u[4], o[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            u[c] = beta * (vf[c] - alpha * (rk * r[3 + c]));
            o[c] = rq * (alpha * r[7 + c] + kq * u[c]);
        }
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[i][c] = __builtin_fmaf(rk * kf[i], u[c], alpha * s[i][c]);
        if (rg == 0)
            *reinterpret_cast<uint2*>(out + t * p.o_tok) =
                make_uint2(Elem<F16>::pack_p(o[0], o[1]), Elem<F16>::pack_p(o[2], o[3]));
    }
}

// NaN in four columns of an entry's rows, one row per lane group of CQ lanes
template <int CQ, bool F16>
__device__ __forceinline__ void nan_rows(const DeltaParams& p, int b, int h, int col, int t0, int t1) {
    const uint32_t nan2 = Elem<F16>::pack_p(__builtin_nanf(""), __builtin_nanf(""));
    uint16_t* const out = p.out + b * p.o_batch + h * p.o_head + col;
    for (int t = t0 + int(threadIdx.x & 63) / CQ; t < t1; t += 64 / CQ)
        *reinterpret_cast<uint2*>(out + t * p.o_tok) = make_uint2(nan2, nan2);
}

// One wave per 4 CQ columns of a head's state, token after token.  Bound by the
// state, read and written once: 64 sequences with a token each, 32 heads of 128 x 128,
// 54.5 us, 4.9 TB/s.  One sequence: 4.5 us, three loads after each other (the id, the
// state and the token's rows, the reduction) and the launch.
template <int DK, int CQ, bool F16>
__global__ __launch_bounds__(256) void delta_recurrent_kernel(DeltaParams p, int64_t units) {
    constexpr int NR = DK * CQ / 64;
    prefetch_kernargs<sizeof(DeltaParams) + sizeof(int64_t)>();
    const int64_t unit = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (unit >= units) return;
    const int lane = threadIdx.x & 63, rg = lane / CQ;
    const int slices = p.Dv / (4 * CQ);
    const int64_t bh = unit / slices;
    const int col = int(unit - bh * slices) * 4 * CQ + 4 * (lane % CQ);
    const int b = int(bh / p.Hv), h = int(bh - int64_t(b) * p.Hv);
    const int slot = entry_state(p.seq, b), len = entry_len(p.seq, b);
    if (slot == kEntryEmpty || len == 0) return;
    if (slot == kEntryBad) {
        nan_rows<CQ, F16>(p, b, h, col, 0, len);
        return;
    }
    float* const st = p.state + ((int64_t(slot) * p.Hv + h) * DK + rg * NR) * p.Dv + col;
    f32x4_t s[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) s[i] = *reinterpret_cast<const f32x4_t*>(st + int64_t(i) * p.Dv);
    recur<DK, CQ, F16>(p, s, b, h, col, 0, len);
#pragma unroll
    for (int i = 0; i < NR; ++i) *reinterpret_cast<f32x4_t*>(st + int64_t(i) * p.Dv) = s[i];
}

// ------------------------------------------------------------------ chunks
constexpr int kChunk = 64;
constexpr int kScanCols = 16;  // columns of the state per chain of the scan

// What the scan needs of one chunk and value head, in the order its lanes read
// it: operand fragments of 64 lanes x 16 bytes.  Of the 64 x 64 triangles only
// the six fragments (row tile, 32 columns) on and below the diagonal are kept:
// row tiles 0 and 1 have one, 2 and 3 two.
constexpr int kFrag = 64 * 8;                    // elements of a fragment
constexpr int kTriFrags = 6;
constexpr int kTPart = kTriFrags * kFrag;        // elements of one part of T or P
constexpr int kUnitT = 0, kUnitP = 3 * kTPart;   // T and P in three parts
constexpr int kUnitVec = 6 * kTPart;             // floats: see kVec*
constexpr int kVecC = 0, kVecD = 64, kVecE = 128, kVecLast = 192, kVecBad = 196, kVecFloats = 208;
// kVecBad: a flag per wave of the preparation, read by the wave of the scan with that number
constexpr int kUnitElems = kUnitVec + 2 * kVecFloats;
__device__ __forceinline__ constexpr int tri_frag(int tile, int ks) { return tile < 2 ? tile : 2 * tile - 2 + ks; }

// Row rho of 16-row tile t, for tokens and for the state's rows.  A product
// leaves rows 4 j + i, i < 4, of a tile in lane group j; as the right operand of the
// next product the group holds 8 consecutive ones of 32.  With this order of
// the rows its rows of two tiles are those eight: no lane needs another's.
__device__ __forceinline__ constexpr int tile_row(int t, int rho) {
    return 32 * (t >> 1) + 8 * (rho >> 2) + 4 * (t & 1) + (rho & 3);
}

// Below these sizes U stays in fp32: 8 lanes hold a row of T, so that |U| < 8 kMaxT kMaxY =
// 2^93, and |e^(G_last - G) U| < 2^123 with the keys' factors in it.  A chunk with more runs
// token by token: an infinite u of one token, times the zeros of P, would make the outputs
// of earlier ones NaN.
constexpr float kMaxT = 0x1p20f;  // the sum of |T| over 8 columns
constexpr float kMaxY = 0x1p70f;  // the sum of |Y| over 4 rows
constexpr float kMaxD = 0x1p30f;  // e^(G_last - G) with the key's factor

struct ChunkPlan {
    uint16_t* units = nullptr;  // [batch][chunk][Hv][kUnitElems]
    int32_t first = 0, count = 0;      // chunks of this launch
    int32_t b_first = 0, b_count = 0;  // batch entries of this launch
};

// the top 16 bits of an fp32 value are a bf16 value; two of them in one word
__device__ __forceinline__ uint32_t top2(float lo, float hi) {
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
// what a part leaves of (lo, hi), exactly: x - 1 part.lo - 0 part.hi.  (A part that
// is infinite makes both NaN: nothing finite is lost, as such a chunk runs token
// by token.)
__device__ __forceinline__ void residual2(uint32_t part, float& lo, float& hi) {
    const bf16x2_t_ x = __builtin_bit_cast(bf16x2_t_, part);
    // (-1, 0) and (0, -1) from registers: as an inline constant the instruction
    // takes -1.0 for the fp32 pattern, the other pair
    uint32_t first = 0x0000BF80u, second = 0xBF800000u;
    __asm__("" : "+s"(first), "+s"(second));
    lo = __builtin_amdgcn_fdot2_f32_bf16(x, __builtin_bit_cast(bf16x2_t_, first), lo, false);
    hi = __builtin_amdgcn_fdot2_f32_bf16(x, __builtin_bit_cast(bf16x2_t_, second), hi, false);
}

// (lo, hi) in three bf16 parts each, exactly: 8 + 8 + 8 bits
__device__ __forceinline__ void split3(float lo, float hi, uint32_t& a, uint32_t& b, uint32_t& c) {
    a = top2(lo, hi);
    residual2(a, lo, hi);
    b = top2(lo, hi);
    residual2(b, lo, hi);
    c = top2(lo, hi);
}
// in two parts, the second rounded: 2^-17
__device__ __forceinline__ void split2(float lo, float hi, uint32_t& a, uint32_t& b) {
    a = top2(lo, hi);
    residual2(a, lo, hi);
    b = Elem<false>::pack_p(lo, hi);
}
// eight fp16 elements in two bf16 parts each, exactly (11 bits)
__device__ __forceinline__ void split_f16(const uint4& x, uint4& a, uint4& b) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t p[4], r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) split2(Elem<true>::lo(w[i]), Elem<true>::hi(w[i]), p[i], r[i]);
    a = make_uint4(p[0], p[1], p[2], p[3]);
    b = make_uint4(r[0], r[1], r[2], r[3]);
}
__device__ __forceinline__ f32x4_t mma(const uint4& a, const uint4& b, const f32x4_t& c) { return Elem<false>::mma32(a, b, c); }

// acc += A B for 16 x 16 fp32 matrices, A given as row (lane % 16), columns 4 (lane
// / 16) .. + 3, B and acc as the products leave them (rows 4 (lane / 16) + i, column
// lane % 16): step i contracts the columns 4 j + i of A with those rows of B
__device__ __forceinline__ f32x4_t mm16(const f32x4_t& a, const f32x4_t& b, f32x4_t acc) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
    return acc;
}

// The value head of workgroup i of Hv.  Workgroups go round the eight XCDs, and i, i +
// 8, .. share an L2: an XCD takes Hv / 8 heads in a row, where the key heads allow it,
// so that K and Q of a key head are read from memory once for its value heads (16 / 32
// heads of 128, 2048 tokens, both kernels 70.2 -> 69.0 us; the preparation's reads 36 -> 19 MB).
__device__ __forceinline__ int head_of(const DeltaParams& p, int i) {
    return p.Hk & 7 ? i : (i & 7) * (p.Hv >> 3) + (i >> 3);
}

// LDS written before it is seen after it; loads from memory stay in flight (a
// __syncthreads would wait for them too)
__device__ __forceinline__ void lds_barrier() {
    __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
}

// 16 bytes per lane from memory into LDS at `to` + 16 lane, `to` uniform
__device__ __forceinline__ void load_lds(const void* from, void* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)from,
                                     (__attribute__((address_space(3))) uint32_t*)to, 16, 0, 0);
}

__device__ __forceinline__ uint2 read_transposed(const uint2* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)p));
}
// Place of row r, elements 8 g .. + 7 of a 16 x 32 block: rows of four units, so that
// four lanes of a load cover 64 bytes (16 rows at once took four times the cache
// accesses), rotated so that neither 16 rows of one g nor 4 rows of all g meet in
// an LDS bank.
__device__ __forceinline__ constexpr int row_unit(int r, int g) { return 4 * r + (g ^ (r >> 2)); }

// Inclusive sum over the lanes of a wave in 64 bits: within rows of 16 lanes by
// DPP shifts, then the last lane of a row to the next row, and of lane 31 to the
// upper half.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, int(uint32_t(u)), CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, int(uint32_t(u >> 32)), CTRL, ROWS, 0xF, false);
    return x + __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_running_sum(double x) {
    x = dpp_add<0x111, 0xF>(x);  // row_shr:1
    x = dpp_add<0x112, 0xF>(x);
    x = dpp_add<0x114, 0xF>(x);
    x = dpp_add<0x118, 0xF>(x);
    x = dpp_add<0x142, 0xA>(x);  // row_bcast:15 into rows 1 and 3
    return dpp_add<0x143, 0xC>(x);  // row_bcast:31 into rows 2 and 3
}

// Four waves per chunk and value head.  Products of rows with rows are formed
// with the roles that leave four neighbours of a row in a lane (rows of the other
// factor in the order tile_row for P), so that P leaves the registers as
// fragments and L enters LDS in 16-byte writes.  (1 + L)^-1 by halves: the four
// diagonal 16 x 16 blocks by substitution, a lane per column; then T10 = -T11
// (L10 T00) for 16- and for 32-wide blocks, as fp32 matrix products.
// 17.8 us for 2048 tokens of 16 / 32 heads of 128 (39 MB of units written, 19 MB read, 3.2
// TB/s): 1024 workgroups, all on the GPU at once, four to a CU, each bound by its own
// chain (loads, norms, L, the substitution's 120 dependent steps, four products after
// each other): 64 workgroups alone take 8.4 us, 2048 take 34.
template <int DK, bool F16>
__global__ __launch_bounds__(256, 4) void delta_chunk_prepare_kernel(DeltaParams p, ChunkPlan c) {
    constexpr int KS = DK / 32, LD = 68, LK = DK + 8;
    prefetch_kernargs<sizeof(DeltaParams) + sizeof(ChunkPlan)>();
    __shared__ __attribute__((aligned(16))) float s_l[64 * LD];  // L, then the products M in its upper blocks
    __shared__ __attribute__((aligned(16))) float s_t[64 * LD];  // the inverse
    uint16_t* const s_k = reinterpret_cast<uint16_t*>(s_t);      // K until then
    static_assert(sizeof(uint16_t) * 64 * LK <= sizeof(s_t), "s_k lies in s_t");
    __shared__ __attribute__((aligned(16))) double s_g[64];  // running sums of log2 of the decays
    __shared__ __attribute__((aligned(16))) float s_beta[64], s_rk[64], s_rq[64];
    __shared__ int s_bad;
    const int h = head_of(p, int(blockIdx.x % uint32_t(p.Hv))), rest = int(blockIdx.x / uint32_t(p.Hv));
    const int n = rest % c.count, b_at = rest / c.count, b = c.b_first + b_at;
    const int t0 = (c.first + n) * kChunk;
    const int slot = entry_state(p.seq, b), len = entry_len(p.seq, b);
    if (slot < 0 || t0 >= len) return;
    const int left = len - t0;  // tokens of this chunk and behind it
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g4 = lane >> 4;
    const int hk = h / p.G;
    uint16_t* const unit = c.units + ((int64_t(b_at) * c.count + n) * p.Hv + h) * kUnitElems;
    float* const vec = reinterpret_cast<float*>(unit + kUnitVec);

    // K's rows of tile w, four lanes to 64 bytes of a row, into LDS; Q's rows in
    // the order of P's fragments, as operands; rows behind the end are zeros
    uint4 kin[KS], qf[KS];
    {
        const int row = 16 * w + (lane >> 2), q_row = tile_row(w, r);
        const uint16_t* const kp = p.k.p + b * p.k.batch + hk * p.k.head + (t0 + row) * p.k.tok + 8 * (lane & 3);
        const uint16_t* const qp = p.q.p + b * p.q.batch + hk * p.q.head + (t0 + q_row) * p.q.tok + 8 * g4;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            kin[ks] = qf[ks] = make_uint4(0, 0, 0, 0);
            if (row < left) kin[ks] = *reinterpret_cast<const uint4*>(kp + 32 * ks);
            if (q_row < left) qf[ks] = *reinterpret_cast<const uint4*>(qp + 32 * ks);
        }
    }
    if (threadIdx.x == 0) s_bad = 0;
    float g = 0.0f, beta = 0.0f;
    if (w == 0 && lane < left) {
        float rate, bias;
        gate_rates(p, h, rate, bias);
        gates<F16>(p, load_gates(p, b, t0 + lane, h), rate, bias, g, beta);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) *reinterpret_cast<uint4*>(s_k + (16 * w + (lane >> 2)) * LK + 32 * ks + 8 * (lane & 3)) = kin[ks];
    __syncthreads();
    // What is not finite, or a factor that may overflow, would reach earlier tokens
    // through the zeros of T and P: the scan runs such a chunk token by token.  64 log
    // decays of at most 1 leave e^G below 2^93.
    bool odd = false;
    if (w == 0) {
        // the running sum in 64 bits: differences of far sums enter the exponents;
        // exp(-2000) is 0 in either precision
        odd = !(g <= 1.0f) || !(fabsf(beta) < INFINITY);
        s_g[lane] = wave_running_sum(double(g < -2000.0f ? -2000.0f : g) * 1.4426950408889634);
        s_beta[lane] = beta;
    }
    const auto k_rows = [&](int row, int ks) { return *reinterpret_cast<const uint4*>(s_k + row * LK + 32 * ks + 8 * g4); };
    const f32x4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
    {  // the rows' norms: diagonals of K K^T and Q Q^T
        f32x4_t kk = zero, qq = zero;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const uint4 x = k_rows(16 * w + r, ks);
            kk = Elem<F16>::mma32(x, x, kk);
            qq = Elem<F16>::mma32(qf[ks], qf[ks], qq);
        }
        if (r >> 2 == g4) {
            const int i = r & 3, k_row = 16 * w + r, q_row = tile_row(w, r);
            const float k2 = i == 0 ? kk[0] : i == 1 ? kk[1] : i == 2 ? kk[2] : kk[3];
            const float q2 = i == 0 ? qq[0] : i == 1 ? qq[1] : i == 2 ? qq[2] : qq[3];
            const float rk = k_row < left ? l2_factor(k2, p.l2_eps) : 0.0f;
            s_rk[k_row] = rk;
            s_rq[q_row] = q_row < left ? p.scale * l2_factor(q2, p.l2_eps) : 0.0f;
            odd |= !(fabsf(rk) < INFINITY) || !(fabsf(k2) < INFINITY);
        }
    }
    if (odd) s_bad = 1;
    __syncthreads();

    // e^(G_row - G_col) with the columns' norms, four columns
    const auto fade = [&](double g_row, int row, int col, float (&f)[4]) {
        const double2 g01 = *reinterpret_cast<const double2*>(s_g + col), g23 = *reinterpret_cast<const double2*>(s_g + col + 2);
        const f32x4_t rk = *reinterpret_cast<const f32x4_t*>(s_rk + col);
        const double gc[4] = {g01.x, g01.y, g23.x, g23.y};
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = row >= col + i ? exp2_fast(float(g_row - gc[i])) * rk[i] : 0.0f;
    };
    {  // P: rows tile_row(w, r), the fragments of tile w
        const int row = tile_row(w, r);
        const double g_row = s_g[row];
        const float rq = s_rq[row];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if (ks > w >> 1) continue;
            uint32_t a[4], d[4], e[4];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                f32x4_t x = zero;
#pragma unroll
                for (int q = 0; q < KS; ++q) x = Elem<F16>::mma32(k_rows(tile_row(2 * ks + half, r), q), qf[q], x);
                float f[4];
                fade(g_row, row, 32 * ks + 8 * g4 + 4 * half, f);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    split3(rq * f[2 * i] * x[2 * i], rq * f[2 * i + 1] * x[2 * i + 1], a[2 * half + i], d[2 * half + i],
                           e[2 * half + i]);
            }
            uint16_t* const to = unit + kUnitP + tri_frag(w, ks) * kFrag + 8 * lane;
            *reinterpret_cast<uint4*>(to) = make_uint4(a[0], a[1], a[2], a[3]);
            *reinterpret_cast<uint4*>(to + kTPart) = make_uint4(d[0], d[1], d[2], d[3]);
            *reinterpret_cast<uint4*>(to + 2 * kTPart) = make_uint4(e[0], e[1], e[2], e[3]);
        }
    }
    {  // L: rows of tile 3 - w, the longest for the wave with the fewest of P
        const int ti = 3 - w, row = 16 * ti + r;
        const double g_row = s_g[row];
        const float f_row = s_beta[row] * s_rk[row];
        uint4 kf[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kf[ks] = k_rows(row, ks);
        for (int tj = 0; tj <= ti; ++tj) {
            f32x4_t x = zero;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) x = Elem<F16>::mma32(k_rows(16 * tj + r, ks), kf[ks], x);
            const int col = 16 * tj + 4 * g4;
            float f[4];
            fade(g_row, row, col, f);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = row > col + i ? f_row * f[i] * x[i] : 0.0f;
            *reinterpret_cast<f32x4_t*>(s_l + row * LD + col) = x;
        }
    }
    bool over = false;
    if (w == 3) {
        const double last = s_g[63], at = s_g[lane];
        const float d = s_rk[lane] * exp2_fast(float(last - at));
        over = !(d < kMaxD);
        vec[kVecC + lane] = s_rk[lane] * exp2_fast(float(at));
        vec[kVecD + lane] = d;
        vec[kVecE + lane] = s_rq[lane] * exp2_fast(float(at));
        if (lane == 0) vec[kVecLast] = exp2_fast(float(last));
    }
    __syncthreads();  // K has been read, L is there
    // the inverse of diagonal block w: column r in every lane group, by substitution
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float* const row = s_l + (16 * w + i) * LD + 16 * w;
        float a = i == r ? 1.0f : 0.0f;
#pragma unroll
        for (int m = 0; m < i; ++m) a = __builtin_fmaf(-row[m], x[m], a);
        x[i] = a;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (i / 4 == g4) s_t[(16 * w + i) * LD + 16 * w + r] = x[i];
    __syncthreads();
    const auto row_of = [&](const float* m, int i, int j) {  // block (i, j) as the left operand
        return *reinterpret_cast<const f32x4_t*>(m + (16 * i + r) * LD + 16 * j + 4 * g4);
    };
    const auto col_of = [&](const float* m, int i, int j) {  // block (i, j) as the right operand
        f32x4_t v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = m[(16 * i + 4 * g4 + e) * LD + 16 * j + r];
        return v;
    };
    const auto put = [&](float* m, int i, int j, const f32x4_t& v, float sign) {
#pragma unroll
        for (int e = 0; e < 4; ++e) m[(16 * i + 4 * g4 + e) * LD + 16 * j + r] = sign * v[e];
    };
    if ((w & 1) == 0) {  // blocks (1, 0) and (3, 2)
        const f32x4_t m = mm16(row_of(s_l, w + 1, w), col_of(s_t, w, w), zero);
        put(s_t, w + 1, w, mm16(row_of(s_t, w + 1, w + 1), m, zero), -1.0f);
    }
    __syncthreads();
    const int bi = 2 + (w >> 1), bj = w & 1;  // the lower left half: M = L T, then -T M
    {
        f32x4_t m = zero;
        for (int e = bj; e < 2; ++e) m = mm16(row_of(s_l, bi, e), col_of(s_t, e, bj), m);
        put(s_l, bj, bi, m, 1.0f);  // an upper block of L
    }
    __syncthreads();
    {
        f32x4_t m = zero;
        for (int e = 2; e <= bi; ++e) m = mm16(row_of(s_t, bi, e), col_of(s_l, bj, e), m);
        put(s_t, bi, bj, m, -1.0f);
    }
    __syncthreads();
    float sum = 0.0f;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        if (ks > w >> 1) continue;
        const int row = tile_row(w, r), col = 32 * ks + 8 * g4;
        const f32x4_t* const src = reinterpret_cast<const f32x4_t*>(s_t + row * LD + col);
        const f32x4_t* const bt = reinterpret_cast<const f32x4_t*>(s_beta + col);
        f32x4_t t[2] = {src[0] * bt[0], src[1] * bt[1]};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (col + i > row) t[i >> 2][i & 3] = 0.0f;  // what was never written
            sum += fabsf(t[i >> 2][i & 3]);
        }
        uint32_t a[4], d[4], e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split3(t[i >> 1][2 * (i & 1)], t[i >> 1][2 * (i & 1) + 1], a[i], d[i], e[i]);
        uint16_t* const to = unit + kUnitT + tri_frag(w, ks) * kFrag + 8 * lane;
        *reinterpret_cast<uint4*>(to) = make_uint4(a[0], a[1], a[2], a[3]);
        *reinterpret_cast<uint4*>(to + kTPart) = make_uint4(d[0], d[1], d[2], d[3]);
        *reinterpret_cast<uint4*>(to + 2 * kTPart) = make_uint4(e[0], e[1], e[2], e[3]);
    }
    // keys far above 1 without a normalisation: T grows with every token, and may overflow where the rule itself does not
    over = __ballot(over || !(sum < kMaxT)) != 0;
    if (lane == 0) vec[kVecBad + w] = over || s_bad ? 1.0f : 0.0f;
}

// A right operand of MT tiles' rows in lane order: 8 (MT = 2, a step of 32) or 4
// values (MT = 1, a step of 16) per lane.
template <int MT>
struct Operand {
    uint32_t w[2 * MT];
};
template <int MT>
__device__ __forceinline__ f32x4_t mma_step(const Operand<MT>& a, const Operand<MT>& b, const f32x4_t& c) {
    if constexpr (MT == 2)
        return Elem<false>::mma32(make_uint4(a.w[0], a.w[1], a.w[2], a.w[3]), make_uint4(b.w[0], b.w[1], b.w[2], b.w[3]), c);
    else
        return Elem<false>::mma16(make_uint2(a.w[0], a.w[1]), make_uint2(b.w[0], b.w[1]), c);
}
// fp16 elements in two bf16 parts
template <int MT>
__device__ __forceinline__ void split_f16(const Operand<MT>& x, Operand<MT>& a, Operand<MT>& b) {
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) split2(Elem<true>::lo(x.w[i]), Elem<true>::hi(x.w[i]), a.w[i], b.w[i]);
}

// The kernel's first argument, read again where it is used: a rare path then
// keeps none of it in registers through the loop around it.
__device__ __forceinline__ DeltaParams kernel_params() {
    typedef const __attribute__((address_space(4))) void kernarg;
    kernarg* a = (kernarg*)__builtin_amdgcn_kernarg_segment_ptr();
    __asm__ volatile("" : "+s"(a));
    DeltaParams p;
    __builtin_memcpy(&p, (const void*)a, sizeof(p));
    return p;
}

// 16 columns of one head's state from chunk to chunk (a chain), in twelve waves.  Waves 0
// to 3 keep the state: wave w its rows of the tiles MT w .. in fp32, as the
// products leave them, which is also how the next product takes them.  Per chunk:
//   (1) wave w: its rows' share of K S0 for all tokens; (2) wave w: the sum of the
//   shares and Y = V - diag(e^G) K S0 for token tile w; (3) wave w: tile w of U = T Y;
//   (4) wave w: its rows of the new state, S <- e^(G_last) S + K^T diag(e^(G_last - G)) U.
// Waves 4 to 7 have the state and U from LDS and form out, tile w - 4: Q S0
// during (2) and (3) (the third part of S0 there: in (2) it takes 1 % longer), P U during
// (4).  Waves 8 to 11 load what waves 0 to 3 need straight into LDS, two chunks ahead: the
// chain (1) to (4) is bound by the instructions that one wave can issue, and 53 KB a
// chunk keep the memory pipe busy.  Rows behind the end come as copies of the last row;
// T has zeros in their place.
// 2048 tokens of 16 / 32 heads of 128, a workgroup per CU, 32 chunks: 53 us in calls after
// each other, 58 to 61 in a few with idle time before.  The chain alone, with nothing loaded
// or stored, takes 47 of the 53: three exchanges through LDS and a product's latency
// between each two, 1.5 us a chunk.
// NC = 2: two chains of neighbouring columns beside each other, waves 0 to 3 and 4 to 7,
// with K, Q and T in common.  They hide each other's latency where there are more
// chains than CUs; the waves of out and of the loads, 8 to 11 and 12 to 15, serve both.
// T and Q have one buffer then, and are taken into registers before (1).
template <int NC>
constexpr int kScanThreads = 256 * NC + 512;
template <int DK, int NC, bool F16>
__global__ __launch_bounds__(kScanThreads<NC>) void delta_chunk_scan_kernel(DeltaParams p, ChunkPlan c) {
    constexpr int KS = DK / 32, MT = DK / 64;  // MT: 16-row tiles of the state per wave
    constexpr int LW = 20;
    constexpr int TQ = NC == 1 ? 2 : 1;        // buffers of T and Q
    constexpr bool kAhead = F16 || NC == 2;    // Q is in registers before (1)
    using Op = Operand<MT>;
    struct Stage {
        uint4 k[4 * KS * 64];                      // [token tile][step][row_unit]
        uint16_t v[kChunk * kScanCols * NC];
        float vec[kVecFloats];
    };
    struct Exchange {                              // of one chain
        f32x4_t x[4 * 3 * 64];                     // shares of K S0 for other waves [token tile][wave][lane]
        uint4 s[3 * KS * 64];                      // the state in three parts [part][step][lane]
        uint4 y[3 * 2 * 64];                       // Y in three parts [part][step][lane], a tile's half of each
        uint4 d[3 * 2 * 64];                       // diag(e^(G_last - G)) U in three parts
        uint4 u[3 * 2 * 64];                       // U
    };
    __shared__ __attribute__((aligned(16))) Stage s_in[2];
    __shared__ uint4 s_q[TQ][4 * KS * 64];
    __shared__ uint4 s_t[TQ][3 * kTriFrags * 64];  // [part][fragment][lane]
    __shared__ __attribute__((aligned(16))) Exchange s_ex[NC];
    __shared__ int s_bad;  // the last chunk that has to run token by token, from 1
    prefetch_kernargs<sizeof(DeltaParams) + sizeof(ChunkPlan)>();
    const int heads = c.b_count * p.Hv;
    const int bh = int(blockIdx.x) % heads, col0 = int(blockIdx.x) / heads * (kScanCols * NC);
    const int b_at = bh / p.Hv, b = c.b_first + b_at, h = head_of(p, bh - b_at * p.Hv), hk = h / p.G;
    const int slot = entry_state(p.seq, b), len = entry_len(p.seq, b);
    const int begin = c.first * kChunk;
    if (slot == kEntryEmpty || begin >= len) return;
    const int end = min(len, begin + c.count * kChunk);
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g4 = lane >> 4;
    if (slot == kEntryBad) {
        if (w < NC) nan_rows<4, F16>(p, b, h, col0 + kScanCols * w + 4 * (lane & 3), begin, end);
        return;
    }
    const int tile = w & 3;
    const int chunks = (end - begin + kChunk - 1) / kChunk;
    const int tok0 = tile_row(tile, 4 * g4);  // the lane's four tokens of tile `tile`
    const f32x4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const int half = 2 * ((tile >> 1) * 64 + lane) + (tile & 1);  // the lane's half of an operand, in uint2
    constexpr int kPart = 2 * 2 * 64;                             // uint2 per part of y, d and u

    const int unit_at = row_unit(r, g4);  // the lane's operand in K and Q
    const int64_t unit_step = int64_t(p.Hv) * kUnitElems;
    const uint16_t* const units = c.units + (int64_t(b_at) * c.count * p.Hv + h) * kUnitElems + 8 * lane;

    if (w >= 4 * NC + 4) {  // the loads: a quarter of each chunk's
        // lane l of a load takes unit l of its fragment: four lanes cover 64 bytes of a row
        const int krow = tile_row(tile, lane >> 2), chunk = (lane & 3) ^ (lane >> 4);
        const int vrow = NC == 1 ? 32 * (tile & 1) + (lane >> 1) : 16 * tile + (lane >> 2), vcol = 8 * (lane & (2 * NC - 1));
        const uint16_t* unit = units;
        const uint16_t* k = p.k.p + b * p.k.batch + hk * p.k.head + begin * p.k.tok + 8 * chunk;
        const uint16_t* q = p.q.p + b * p.q.batch + hk * p.q.head + begin * p.q.tok + 8 * chunk;
        const uint16_t* v = p.v.p + b * p.v.batch + h * p.v.head + begin * p.v.tok + col0 + vcol;
        int64_t k_at = krow * p.k.tok, q_at = krow * p.q.tok, v_at = vrow * p.v.tok;
        const auto stage_t = [&](int n) {
            if (n >= chunks) return;
#pragma unroll
            for (int i = 0; i < 5; ++i)
                if (4 * i + tile < 3 * kTriFrags) load_lds(unit + kUnitT + (4 * i + tile) * kFrag, s_t[n & (TQ - 1)] + (4 * i + tile) * 64);
            unit += unit_step;
        };
        const auto stage = [&](int n) {
            if (n >= chunks) return;
            Stage& to = s_in[n & 1];
            const int last = end - 1 - begin - n * kChunk;
            if (last < kChunk - 1) k_at = min(krow, last) * p.k.tok, v_at = min(vrow, last) * p.v.tok;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) load_lds(k + k_at + 32 * ks, to.k + (tile * KS + ks) * 64);
            if constexpr (NC == 1) stage_t(n);
            if (tile < 2 * NC) load_lds(v + v_at, to.v + tile * 32 * kScanCols);
            if (tile == 2 && lane < kVecFloats / 4) load_lds(units + n * unit_step + kUnitVec, to.vec);
            k += kChunk * p.k.tok, v += kChunk * p.v.tok;
        };
        // Q, which the waves of out take after (1), or have taken before it: half a chunk later, so that the
        // loads spread over it (2048 tokens, both kernels, 72.0 -> 69.0 us)
        const auto stage_q = [&](int n) {
            if (n >= chunks) return;
            const int last = end - 1 - begin - n * kChunk;
            if (last < kChunk - 1) q_at = min(krow, last) * p.q.tok;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) load_lds(q + q_at + 32 * ks, s_q[n & (TQ - 1)] + (tile * KS + ks) * 64);
            q += kChunk * p.q.tok;
        };
        stage(0);
        if constexpr (NC == 2) stage_t(0);
        stage_q(0);
        __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
        lds_barrier();  // chunk 0 is there
        stage(1);
        for (int n = 0; n < chunks; ++n) {
            lds_barrier();  // (1)
            stage_q(n + 1);  // where chunk n - 1's was, or n's, which has been read
            if constexpr (NC == 2) stage_t(n + 1);  // chunk n's has been read
            lds_barrier();   // (2)
            __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);  // chunk n + 1 is there, for all after (3)
            const int slow_word = s_bad;
            const bool slow = __builtin_amdgcn_readfirstlane(slow_word) == n + 1;
            lds_barrier();  // (3)
            if (slow) {
                lds_barrier();
                lds_barrier();
                lds_barrier();
            }
            stage(n + 2);  // in chunk n's place: its last reads came before (3)
        }
        return;
    }

    if (w >= 4 * NC) {  // rows of out
        uint16_t* out = p.out + b * p.o_batch + h * p.o_head + (begin + tok0) * p.o_tok + col0 + r;
        const uint16_t* unit = units + kUnitP;
        const int tri0 = tri_frag(tile, 0) * kFrag, tri1 = tri_frag(tile, tile >> 1) * kFrag;
        uint4 tri[2][3];
        f32x4_t e;
        const auto load_tri = [&](int n) {
            if (n >= chunks) return;
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                tri[0][i] = *reinterpret_cast<const uint4*>(unit + i * kTPart + tri0);
                tri[1][i] = *reinterpret_cast<const uint4*>(unit + i * kTPart + tri1);
            }
            unit += unit_step;
        };
        // fp16: Q is read and split during (4) of the chunk before (2048 tokens of 32 heads of
        // 128, both kernels, 92.1 -> 86.9 us); bf16, with nothing to split, after (1) (69.0 against 70.6)
        uint4 q0[KS], q1[KS];
        const auto load_q = [&](int at) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                q0[ks] = s_q[at & (TQ - 1)][(tile * KS + ks) * 64 + unit_at];
                if constexpr (F16) split_f16(q0[ks], q0[ks], q1[ks]);
            }
        };
        load_tri(0);
        lds_barrier();  // chunk 0 is there
        if constexpr (kAhead) load_q(0);
        for (int n = 0; n < chunks; ++n) {
            lds_barrier();  // (1)
            e = *reinterpret_cast<const f32x4_t*>(s_in[n & 1].vec + kVecE + tok0);
            f32x4_t a0[NC], a1[NC];
            if constexpr (!kAhead) load_q(n);
#pragma unroll
            for (int g = 0; g < NC; ++g) {
                const Exchange& ex = s_ex[g];
                a0[g] = a1[g] = zero;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const uint4 s0 = ex.s[ks * 64 + lane], s1 = ex.s[(KS + ks) * 64 + lane];
                    a0[g] = mma(q0[ks], s0, a0[g]);
                    a1[g] = mma(q0[ks], s1, a1[g]);
                    if constexpr (F16) a1[g] = mma(q1[ks], s0, a1[g]), a1[g] = mma(q1[ks], s1, a1[g]);
                }
            }
            lds_barrier();  // (2)
            const int slow_word = s_bad;
            const bool slow = __builtin_amdgcn_readfirstlane(slow_word) == n + 1;
#pragma unroll
            for (int g = 0; g < NC; ++g) {  // the third part: these waves have nothing else to do here
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) a1[g] = mma(q0[ks], s_ex[g].s[(2 * KS + ks) * 64 + lane], a1[g]);
                a0[g] = (a0[g] + a1[g]) * e;
                a1[g] = zero;
            }
            lds_barrier();  // (3)
            if (slow) {
                lds_barrier();
                lds_barrier();
                lds_barrier();
            } else {
                const int left = end - begin - n * kChunk - tok0;
#pragma unroll
                for (int g = 0; g < NC; ++g) {
                    const Exchange& ex = s_ex[g];
                    f32x4_t a2 = zero;
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks) {
                        if (ks > tile >> 1) continue;
                        const uint4 u0 = ex.u[ks * 64 + lane], u1 = ex.u[(2 + ks) * 64 + lane], u2 = ex.u[(4 + ks) * 64 + lane];
                        a0[g] = mma(tri[ks][0], u0, a0[g]);
                        a1[g] = mma(tri[ks][0], u1, a1[g]);
                        a2 = mma(tri[ks][0], u2, a2);
                        a1[g] = mma(tri[ks][1], u0, a1[g]);
                        a2 = mma(tri[ks][1], u1, a2);
                        a2 = mma(tri[ks][2], u0, a2);
                    }
                    a0[g] += a1[g] + a2;
                    uint16_t* to = out + kScanCols * g;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (i < left) *to = uint16_t(Elem<F16>::pack_p(a0[g][i], 0.0f));
                        to += p.o_tok;
                    }
                }
            }
            load_tri(n + 1);
            if constexpr (kAhead) load_q(n + 1);
            out += kChunk * p.o_tok;
        }
        return;
    }

    const int chain = NC == 1 ? 0 : w >> 2, cw = NC == 1 ? w : w & 3;  // the wave's chain, and its number there
    Exchange& ex = s_ex[chain];
    const int col = col0 + kScanCols * chain;
    float* const s_w = reinterpret_cast<float*>(ex.x);  // the state of a chunk that runs token by token
    static_assert(DK * LW * sizeof(float) <= sizeof(ex.x), "s_w lies in x");
    __builtin_amdgcn_s_setprio(3);  // the chain goes first where waves meet on a SIMD
    const int row0 = tile_row(MT * cw, 4 * g4);  // the lane's first row of the state; tile m: + 4 m
    float* const st = p.state + ((int64_t(slot) * p.Hv + h) * DK + row0) * p.Dv + col + r;
    f32x4_t s[MT];
    const auto put3 = [&](uint2* to, float x0, float x1, float x2, float x3) {
        uint32_t a[2], d[2], e[2];
        split3(x0, x1, a[0], d[0], e[0]);
        split3(x2, x3, a[1], d[1], e[1]);
        to[0] = make_uint2(a[0], a[1]);
        to[kPart] = make_uint2(d[0], d[1]);
        to[2 * kPart] = make_uint2(e[0], e[1]);
    };
    // K: the tokens of all tiles, the wave's own first, and the lane's rows of the state
    const auto load_k = [&](const Stage& in, Op (&fk)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = (cw + i) & 3;
            if constexpr (MT == 2) {
                const uint4 x = in.k[(j * KS + cw) * 64 + unit_at];
                fk[i].w[0] = x.x, fk[i].w[1] = x.y, fk[i].w[2] = x.z, fk[i].w[3] = x.w;
            } else {
                const uint2 x = reinterpret_cast<const uint2*>(in.k)[2 * ((j * KS + (cw >> 1)) * 64 + unit_at) + (cw & 1)];
                fk[i].w[0] = x.x, fk[i].w[1] = x.y;
            }
        }
    };
    // K^T: the lane's row of state tile m, eight tokens, from two transposing
    // reads: 16 lanes give 4 rows of 16 elements, lane i takes column i of them
    const auto k_t = [&](const Stage& in, int m, int ks) {
        const int state_tile = MT * cw + m;
        const uint2* const at = reinterpret_cast<const uint2*>(in.k) +
                                2 * ((2 * ks * KS + (state_tile >> 1)) * 64 + row_unit(4 * g4 + (r >> 2), r & 3)) + (state_tile & 1);
        const uint2 lo = read_transposed(at), hi = read_transposed(at + 2 * KS * 64);
        return make_uint4(lo.x, lo.y, hi.x, hi.y);
    };
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[m][i] = st[int64_t(4 * m + i) * p.Dv];
    if (threadIdx.x == 0) s_bad = 0;
    lds_barrier();
    for (int n = 0; n < chunks; ++n) {
        const Stage& in = s_in[n & 1];
        Op fk[4];
        load_k(in, fk);
        const uint4* const t = s_t[n & (TQ - 1)];
        uint4 ft[2][3];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            ft[0][i] = t[(i * kTriFrags + tri_frag(tile, 0)) * 64 + lane];
            ft[1][i] = t[(i * kTriFrags + tri_frag(tile, tile >> 1)) * 64 + lane];
        }
        const f32x4_t e = *reinterpret_cast<const f32x4_t*>(in.vec + kVecC + tok0);
        const f32x4_t d = *reinterpret_cast<const f32x4_t*>(in.vec + kVecD + tok0);
        const float last = in.vec[kVecLast], bad = in.vec[kVecBad + tile];
        const uint2 v = read_transposed(reinterpret_cast<const uint2*>(in.v) + 4 * (NC * (tok0 + (r >> 2)) + chain) + (r & 3));
        f32x4_t x[4];
        {  // (1)
            Op s0, s1, s2;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                split3(s[m][0], s[m][1], s0.w[2 * m], s1.w[2 * m], s2.w[2 * m]);
                split3(s[m][2], s[m][3], s0.w[2 * m + 1], s1.w[2 * m + 1], s2.w[2 * m + 1]);
            }
            if constexpr (MT == 2) {
                ex.s[cw * 64 + lane] = make_uint4(s0.w[0], s0.w[1], s0.w[2], s0.w[3]);
                ex.s[(KS + cw) * 64 + lane] = make_uint4(s1.w[0], s1.w[1], s1.w[2], s1.w[3]);
                ex.s[(2 * KS + cw) * 64 + lane] = make_uint4(s2.w[0], s2.w[1], s2.w[2], s2.w[3]);
            } else {
                uint2* const to = reinterpret_cast<uint2*>(ex.s) + 2 * ((cw >> 1) * 64 + lane) + (cw & 1);
                to[0] = make_uint2(s0.w[0], s0.w[1]);
                to[2 * KS * 64] = make_uint2(s1.w[0], s1.w[1]);
                to[4 * KS * 64] = make_uint2(s2.w[0], s2.w[1]);
            }
            Op k0[4], k1[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                k0[j] = fk[j];
                if constexpr (F16) split_f16(fk[j], k0[j], k1[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = mma_step(k0[j], s2, zero);
            if constexpr (F16)
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = mma_step(k1[j], s1, x[j]);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = mma_step(k0[j], s1, x[j]);
            if constexpr (F16)
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = mma_step(k1[j], s0, x[j]);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = mma_step(k0[j], s0, x[j]);
#pragma unroll
            for (int j = 1; j < 4; ++j) ex.x[(((cw + j) & 3) * 3 + j - 1) * 64 + lane] = x[j];
        }
        lds_barrier();  // (1)
        uint4 fkt[2 * MT];
        {  // (2)
            const f32x4_t x1 = ex.x[3 * tile * 64 + lane], x2 = ex.x[(3 * tile + 1) * 64 + lane], x3 = ex.x[(3 * tile + 2) * 64 + lane];
            const f32x4_t z = (x[0] + x1) + (x2 + x3);
            const float vf[4] = {Elem<F16>::lo(v.x), Elem<F16>::hi(v.x), Elem<F16>::lo(v.y), Elem<F16>::hi(v.y)};
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = vf[i] - e[i] * z[i];
            put3(reinterpret_cast<uint2*>(ex.y) + half, y[0], y[1], y[2], y[3]);
            if (!((fabsf(y[0]) + fabsf(y[1])) + (fabsf(y[2]) + fabsf(y[3])) < kMaxY) || bad != 0.0f) s_bad = n + 1;
        }
        lds_barrier();  // (2)
        const int slow_word = s_bad;
        {  // (3)
            uint4 y[2][3];  // NC = 2: the second step for all tiles, as a branch here leaves one of its parts in scratch memory
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    if (NC == 2 || ks <= tile >> 1) y[ks][i] = ex.y[(2 * i + ks) * 64 + lane];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) fkt[2 * m + ks] = k_t(in, m, ks);
            f32x4_t a0 = zero, a1 = zero, a2 = zero;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                if (ks > tile >> 1) continue;
                a2 = mma(ft[ks][0], y[ks][2], a2);
                a1 = mma(ft[ks][0], y[ks][1], a1);
                a0 = mma(ft[ks][0], y[ks][0], a0);
                a2 = mma(ft[ks][1], y[ks][1], a2);
                a1 = mma(ft[ks][1], y[ks][0], a1);
                a2 = mma(ft[ks][2], y[ks][0], a2);
            }
            const f32x4_t u = a0 + (a1 + a2);
            put3(reinterpret_cast<uint2*>(ex.d) + half, d[0] * u[0], d[1] * u[1], d[2] * u[2], d[3] * u[3]);
            put3(reinterpret_cast<uint2*>(ex.u) + half, u[0], u[1], u[2], u[3]);
        }
        const bool slow = __builtin_amdgcn_readfirstlane(slow_word) == n + 1;
        lds_barrier();  // (3)
        if (slow) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) s_w[(row0 + 4 * m + i) * LW + r] = s[m][i];
            lds_barrier();
            if (cw == 0) {
                constexpr int NR = DK / 16;
                const int t0 = begin + n * kChunk;
                f32x4_t sr[NR];
#pragma unroll
                for (int i = 0; i < NR; ++i) sr[i] = *reinterpret_cast<const f32x4_t*>(s_w + (lane / 4 * NR + i) * LW + 4 * (lane & 3));
                recur<DK, 4, F16>(kernel_params(), sr, b, h, col + 4 * (lane & 3), t0, min(end, t0 + kChunk));
#pragma unroll
                for (int i = 0; i < NR; ++i) *reinterpret_cast<f32x4_t*>(s_w + (lane / 4 * NR + i) * LW + 4 * (lane & 3)) = sr[i];
            }
            lds_barrier();
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[m][i] = s_w[(row0 + 4 * m + i) * LW + r];
            lds_barrier();  // before (1) writes over it
            continue;
        }
        // (4)
        uint4 dp[2][3];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < 3; ++i) dp[ks][i] = ex.d[(2 * i + ks) * 64 + lane];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            f32x4_t a0 = s[m] * last, a1 = zero, a2 = zero;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                uint4 k0 = fkt[2 * m + ks], k1;
                if constexpr (F16) split_f16(fkt[2 * m + ks], k0, k1);
                a2 = mma(k0, dp[ks][2], a2);
                a1 = mma(k0, dp[ks][1], a1);
                a0 = mma(k0, dp[ks][0], a0);
                if constexpr (F16) a2 = mma(k1, dp[ks][1], a2), a1 = mma(k1, dp[ks][0], a1);
            }
            s[m] = a0 + (a1 + a2);
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) st[int64_t(4 * m + i) * p.Dv] = s[m][i];
}

// What one pair of launches takes: entries of the batch and chunks of each, with
// units of about 96 MB, which the caches hold between the two kernels (8192 tokens:
// 48 and 64 MB 314, 80 to 128 MB 297, 256 MB 327 us; 32768 tokens: 64 MB 1215, 96 MB 1173,
// 115 MB 1163, 128 MB 1196, 256 MB 1355 us).  Whole entries where they fit, a multiple of
// what fills the GPU: a launch's start costs a workgroup about two chunks' time.  More
// chains than CUs go two to a workgroup (both kernels, us, one chain per workgroup against this: 2048
// tokens of 32 heads of 128, 3 sequences 229 / 199, 8 sequences 602 / 483, fp16 714 / 581;
// 40 heads 127 / 107, 64 heads 149 / 119; as many chains as CUs, 32 heads, 69 / 100).
constexpr size_t kUnitBytes = kUnitElems * 2;
// CUs of the whole card, not of the current device: a call's plan has to be the one that
// its workspace was sized for, wherever that was asked.
constexpr int64_t kCus = 256;
struct LaunchPlan {
    int64_t entries, chunks;
};
LaunchPlan launch_plan(int64_t B, int64_t S, int64_t Hv, int64_t Dv) {
    const int64_t all = (S + kChunk - 1) / kChunk;
    const int64_t units = std::max<int64_t>(int64_t((size_t(96) << 20) / kUnitBytes) / Hv, 1);  // chunks of all heads
    const int64_t chains = Hv * (Dv / kScanCols), round = B * chains > kCus ? 2 * kCus : kCus;
    const int64_t fill = (round + chains - 1) / chains;  // entries
    const auto even = [](int64_t n, int64_t most) {  // n in equal parts of at most `most`
        const int64_t parts = (n + most - 1) / most;
        return (n + parts - 1) / parts;
    };
    const int64_t entries = even(B, std::max(units / all / fill, int64_t(1)) * fill);
    return {entries, even(all, std::max<int64_t>(units / entries, 1))};
}

// Whether the rule runs in chunks.  Token by token a call takes about 0.7 us a
// token while its waves (16 columns each) find SIMDs of their own, the two chunk
// kernels 12.7 us for any prompt of up to 64 tokens: 16 / 32 heads of 128, 12 tokens
// 11.6 against 12.7 us, 16 tokens 14.5 against 13.3.  More waves share the chunk
// kernels' CUs and fill the SIMDs better: 2 sequences, 16 tokens 14.9 against 16.1, 20
// tokens 17.6 against 16.0; 8 sequences, 24 tokens 33.9 against 35.7, 28 tokens 36.8
// against 36.1; 64 sequences, 28 tokens 223 against 250, 32 tokens 249 against 250, 40
// tokens 300 against 265.  (Between the lines: 4 sequences, 24 tokens 24.4 against 22.6, 28
// tokens 27.7 against 22.7.)  64-wide heads, 4 / 8, are faster token by token up to 12 to 16
// tokens, and up to 28 to 32 for 64 sequences: 9.6 / 12.5 and 11.8 / 12.2; 28.4 / 29.9 and 31.9 / 30.4.
constexpr int64_t kManyWaves = 1024;  // one per SIMD
int64_t column_waves(int64_t B, int64_t Hv, int64_t Dv) { return B * Hv * (Dv / 16); }
bool in_chunks(int64_t B, int64_t S, int64_t Hv, int64_t Dv) {
    const int64_t waves = column_waves(B, Hv, Dv);
    return S > (waves >= kManyWaves ? 28 : 2 * waves >= kManyWaves ? 16 : 12);
}

template <bool F16>
int launch_chunks(const DeltaParams& p, void* ws, hipStream_t stream) {
    const LaunchPlan plan = launch_plan(p.B, p.seq.S, p.Hv, p.Dv);
    const int64_t all = (int64_t(p.seq.S) + kChunk - 1) / kChunk;
    ChunkPlan c;
    c.units = static_cast<uint16_t*>(ws);
    auto* prepare = p.Dk == 128 ? delta_chunk_prepare_kernel<128, F16> : delta_chunk_prepare_kernel<64, F16>;
    auto* one = p.Dk == 128 ? delta_chunk_scan_kernel<128, 1, F16> : delta_chunk_scan_kernel<64, 1, F16>;
    auto* two = p.Dk == 128 ? delta_chunk_scan_kernel<128, 2, F16> : delta_chunk_scan_kernel<64, 2, F16>;
    for (int64_t b_first = 0; b_first < p.B; b_first += plan.entries)
        for (int64_t first = 0; first < all; first += plan.chunks) {
            c.b_first = int32_t(b_first), c.b_count = int32_t(std::min(plan.entries, p.B - b_first));
            c.first = int32_t(first), c.count = int32_t(std::min(plan.chunks, all - first));
            const int64_t heads = int64_t(c.b_count) * p.Hv;
            hipLaunchKernelGGL(prepare, dim3(unsigned(heads * c.count)), dim3(256), 0, stream, p, c);
            GENLLM_LAUNCH_CHECK("delta_chunk_prepare_kernel");
            const int64_t chains = heads * (p.Dv / kScanCols);
            if (chains > kCus)
                hipLaunchKernelGGL(two, dim3(unsigned(chains / 2)), dim3(kScanThreads<2>), 0, stream, p, c);
            else
                hipLaunchKernelGGL(one, dim3(unsigned(chains)), dim3(kScanThreads<1>), 0, stream, p, c);
            GENLLM_LAUNCH_CHECK("delta_chunk_scan_kernel");
        }
    return GENLLM_OK;
}

// 32 columns per wave where that leaves every SIMD one, else 16: the wider wave
// reads and sums a token's q and k once for twice the columns (16 / 32 heads of
// 128, 8 tokens: 8 sequences 16.6 against 18.5 us, 64 sequences 91 against 97; one
// sequence 12.2 against 9.5).
template <int CQ, bool F16>
int launch_recurrent(const DeltaParams& p, hipStream_t stream) {
    const int64_t units = int64_t(p.B) * p.Hv * (p.Dv / (4 * CQ));
    auto* kern = p.Dk == 128 ? delta_recurrent_kernel<128, CQ, F16> : delta_recurrent_kernel<64, CQ, F16>;
    hipLaunchKernelGGL(kern, dim3(unsigned((units + 3) / 4)), dim3(256), 0, stream, p, units);
    GENLLM_LAUNCH_CHECK("delta_recurrent_kernel");
    return GENLLM_OK;
}

bool dim_served(int32_t d) { return d == 64 || d == 128; }
bool heads_served(int64_t B, int64_t Hv) { return B * Hv <= (int64_t(1) << 19); }  // a grid has at most 2^32 threads
bool tokens_served(int64_t S) { return S <= (int64_t(1) << 30); }

bool strides_ok(const Rows3& r) { return aligned_to(r.p, 16) && ((r.batch | r.tok | r.head) & 7) == 0; }

// "NAME overlaps NAME" where a call would write what it or another workgroup reads.
// out may be v itself: a workgroup has read an element before it writes over it.
std::string overlap_of(const DeltaParams& p, const void* ws, size_t ws_bytes) {
    const auto rows = [&](const void* at, int64_t batch, int64_t tok, int64_t head, int64_t heads, int64_t bytes, int64_t elem) {
        Rows r = Rows::whole(at, bytes * elem);
        const int64_t n[3] = {p.B, p.seq.S, heads}, stride[3] = {batch * elem, tok * elem, head * elem};
        std::copy(n, n + 3, r.n), std::copy(stride, stride + 3, r.stride);
        return r;
    };
    const Rows v = rows(p.v.p, p.v.batch, p.v.tok, p.v.head, p.Hv, p.Dv, 2);
    const int64_t gate = p.a_log ? 2 : 4, states = p.seq.ids ? p.seq.n_states : p.B;
    const NamedRows written[] = {{"out", rows(p.out, p.o_batch, p.o_tok, p.o_head, p.Hv, p.Dv, 2)},
                               {"the state", Rows::whole(p.state, states * p.Hv * p.Dk * p.Dv * 4)},
                               {"the workspace", Rows::whole(ws, int64_t(ws_bytes))}};
    const NamedRows read[] = {{"q", rows(p.q.p, p.q.batch, p.q.tok, p.q.head, p.Hk, p.Dk, 2)},
                            {"k", rows(p.k.p, p.k.batch, p.k.tok, p.k.head, p.Hk, p.Dk, 2)},
                            {"v", v},
                            {"a", rows(p.a, p.a_batch, p.a_tok, 0, 1, p.Hv, gate)},
                            {"b", rows(p.b, p.b_batch, p.b_tok, 0, 1, p.Hv, gate)},
                            {"a_log", Rows::whole(p.a_log, p.Hv * 4)},
                            {"dt_bias", Rows::whole(p.dt_bias, p.Hv * 4)},
                            {"state_ids", Rows::whole(p.seq.ids, p.B * 4)},
                            {"seq_lens", Rows::whole(p.seq.lens, p.B * 4)}};
    const char *a, *b;
    const auto out_is_v = [&](const Rows& w, const Rows& r) { return w.same_as(v) && r.same_as(v); };
    if (find_overlap(written, read, out_is_v, a, b)) return std::string(a) + " overlaps " + b;
    return rows_shared_within(written[0].rows) ? "rows of out share memory" : std::string();
}

}  // namespace

}  // namespace genllm

using namespace genllm;

extern "C" size_t genllm_gated_delta_workspace_bytes(int32_t batch, int32_t seq_len, int32_t n_k_heads, int32_t n_v_heads,
                                                     int32_t k_dim, int32_t v_dim) {
    if (batch <= 0 || seq_len <= 0 || n_k_heads <= 0 || n_v_heads <= 0 || !dim_served(k_dim) || !dim_served(v_dim) ||
        !heads_served(batch, n_v_heads) || !tokens_served(seq_len) || !in_chunks(batch, seq_len, n_v_heads, v_dim))
        return 0;
    const LaunchPlan plan = launch_plan(batch, seq_len, n_v_heads, v_dim);
    return size_t(plan.entries) * size_t(plan.chunks) * size_t(n_v_heads) * kUnitBytes;
}

extern "C" int genllm_gated_delta_rule(const void* q, int64_t q_batch_stride, int64_t q_tok_stride, int64_t q_head_stride,
                                       const void* k, int64_t k_batch_stride, int64_t k_tok_stride, int64_t k_head_stride,
                                       const void* v, int64_t v_batch_stride, int64_t v_tok_stride, int64_t v_head_stride,
                                       const void* a, int64_t a_batch_stride, int64_t a_tok_stride, const void* b,
                                       int64_t b_batch_stride, int64_t b_tok_stride, const float* a_log,
                                       const float* dt_bias, float* state, int32_t n_states, const int32_t* state_ids,
                                       const int32_t* seq_lens, void* out, int64_t o_batch_stride, int64_t o_tok_stride,
                                       int64_t o_head_stride, int32_t batch, int32_t seq_len, int32_t n_k_heads,
                                       int32_t n_v_heads, int32_t k_dim, int32_t v_dim, int32_t dtype, float scale,
                                       float l2_eps, void* workspace, size_t workspace_bytes, void* stream) {
    if (batch < 0 || seq_len < 0 || n_k_heads <= 0 || n_v_heads <= 0 || n_states < 0)
        return fail(GENLLM_ERR_INVALID, "gated_delta_rule: negative or zero size");
    if (n_v_heads % n_k_heads)
        return fail(GENLLM_ERR_INVALID, "gated_delta_rule: n_v_heads must be a multiple of n_k_heads");
    if (!dim_served(k_dim) || !dim_served(v_dim))
        return fail(GENLLM_ERR_UNSUPPORTED, "gated_delta_rule: k_dim and v_dim of 64 or 128 are served");
    if (dtype != GENLLM_DTYPE_BF16 && dtype != GENLLM_DTYPE_F16)
        return fail(GENLLM_ERR_UNSUPPORTED, "gated_delta_rule: bf16 or fp16 elements");
    if (!std::isfinite(scale) || std::isnan(l2_eps) || l2_eps == INFINITY)
        return fail(GENLLM_ERR_INVALID, "gated_delta_rule: scale and l2_eps must be finite");
    if (batch == 0 || seq_len == 0) return GENLLM_OK;
    if (!q || !k || !v || !a || !b || !state || !out) return fail(GENLLM_ERR_INVALID, "gated_delta_rule: null pointer");
    if (!a_log != !dt_bias)
        return fail(GENLLM_ERR_INVALID, "gated_delta_rule: a_log and dt_bias go together");
    if (!state_ids && n_states < batch)
        return fail(GENLLM_ERR_INVALID, "gated_delta_rule: fewer states than batch entries");
    // the stride of a dim of one never matters
    if (batch == 1) q_batch_stride = k_batch_stride = v_batch_stride = a_batch_stride = b_batch_stride = o_batch_stride = 0;
    if (seq_len == 1) q_tok_stride = k_tok_stride = v_tok_stride = a_tok_stride = b_tok_stride = o_tok_stride = 0;
    if (n_k_heads == 1) q_head_stride = k_head_stride = 0;
    if (n_v_heads == 1) v_head_stride = o_head_stride = 0;
    if ((batch > 1 && !o_batch_stride) || (seq_len > 1 && !o_tok_stride) || (n_v_heads > 1 && !o_head_stride))
        return fail(GENLLM_ERR_INVALID, "gated_delta_rule: rows of out share memory");
    DeltaParams p;
    p.q = {static_cast<const uint16_t*>(q), q_batch_stride, q_tok_stride, q_head_stride};
    p.k = {static_cast<const uint16_t*>(k), k_batch_stride, k_tok_stride, k_head_stride};
    p.v = {static_cast<const uint16_t*>(v), v_batch_stride, v_tok_stride, v_head_stride};
    p.out = static_cast<uint16_t*>(out);
    p.o_batch = o_batch_stride, p.o_tok = o_tok_stride, p.o_head = o_head_stride;
    if (!strides_ok(p.q) || !strides_ok(p.k) || !strides_ok(p.v) ||
        !strides_ok({p.out, o_batch_stride, o_tok_stride, o_head_stride}) || !aligned_to(state, 16))
        return fail(GENLLM_ERR_INVALID, "gated_delta_rule: q, k, v, out rows and the state must be 16-byte aligned");
    const bool f16 = dtype == GENLLM_DTYPE_F16;
    const uintptr_t gate_align = a_log ? 2 : 4;
    if (!aligned_to(a, gate_align) || !aligned_to(b, gate_align) || !aligned_to(a_log, 4) || !aligned_to(dt_bias, 4) ||
        !aligned_to(state_ids, 4) || !aligned_to(seq_lens, 4))
        return fail(GENLLM_ERR_INVALID, "gated_delta_rule: a pointer is not aligned to its type");
    if (!tokens_served(seq_len)) return fail(GENLLM_ERR_INVALID, "gated_delta_rule: seq_len must be at most 2^30");
    if (!heads_served(batch, n_v_heads))
        return fail(GENLLM_ERR_INVALID, "gated_delta_rule: batch * n_v_heads must be at most 2^19");
    p.a = a, p.b = b, p.a_batch = a_batch_stride, p.a_tok = a_tok_stride, p.b_batch = b_batch_stride, p.b_tok = b_tok_stride;
    p.a_log = a_log, p.dt_bias = dt_bias, p.state = state;
    p.seq.ids = state_ids, p.seq.lens = seq_lens, p.seq.n_states = n_states, p.seq.S = seq_len;
    p.B = batch, p.Hk = n_k_heads, p.Hv = n_v_heads, p.G = n_v_heads / n_k_heads, p.Dk = k_dim, p.Dv = v_dim;
    p.scale = scale, p.l2_eps = l2_eps < 0.0f ? -1.0f : l2_eps;
    const bool chunks = in_chunks(batch, seq_len, n_v_heads, v_dim);
    size_t need = 0;
    if (chunks) {
        need = genllm_gated_delta_workspace_bytes(batch, seq_len, n_k_heads, n_v_heads, k_dim, v_dim);
        if (!workspace || workspace_bytes < need || !aligned_to(workspace, 16))
            return fail(GENLLM_ERR_INVALID, "gated_delta_rule: a workspace of " + std::to_string(need) +
                                                " bytes, 16-byte aligned, is needed (have " +
                                                std::to_string(workspace_bytes) + ")");
    }
    if (const std::string why = overlap_of(p, chunks ? workspace : nullptr, need); !why.empty())
        return fail(GENLLM_ERR_INVALID, "gated_delta_rule: " + why);
    if (chunks)
        return f16 ? launch_chunks<true>(p, workspace, as_stream(stream)) : launch_chunks<false>(p, workspace, as_stream(stream));
    const hipStream_t s = as_stream(stream);
    if (column_waves(batch, n_v_heads, v_dim) >= 2 * kManyWaves)
        return f16 ? launch_recurrent<8, true>(p, s) : launch_recurrent<8, false>(p, s);
    return f16 ? launch_recurrent<4, true>(p, s) : launch_recurrent<4, false>(p, s);
}
