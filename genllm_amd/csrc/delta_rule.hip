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
#include <climits>
#include <cmath>

#include "common.hpp"
#include "kernels.hpp"
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

// log decay and beta of one token and head
template <bool F16>
__device__ __forceinline__ void gates(const DeltaParams& p, int b, int64_t t, int h, float& g, float& beta) {
    const int64_t ia = b * p.a_batch + t * p.a_tok + h, ib = b * p.b_batch + t * p.b_tok + h;
    if (!p.a_log) {
        g = static_cast<const float*>(p.a)[ia];
        beta = static_cast<const float*>(p.b)[ib];
        return;
    }
    const float x = Elem<F16>::lo(static_cast<const uint16_t*>(p.a)[ia]) + p.dt_bias[h];
    const float softplus = fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x)));
    // fmaxf drops a NaN: the sum keeps it through fabsf(x)
    g = -expf(p.a_log[h]) * softplus;
    beta = 1.0f / (1.0f + expf(-Elem<F16>::lo(static_cast<const uint16_t*>(p.b)[ib])));
}

template <bool F16>
__device__ __forceinline__ void unpack_pair(uint32_t w, float& lo, float& hi) {
    lo = Elem<F16>::lo(w);
    hi = Elem<F16>::hi(w);
}

// N consecutive elements (N = 4, 8 or 16), aligned to 2 N bytes up to 16
template <bool F16, int N>
__device__ __forceinline__ void load_elems(const uint16_t* p, float (&f)[N]) {
    uint32_t w[N / 2];
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
#pragma unroll
    for (int i = 0; i < N / 2; ++i) unpack_pair<F16>(w[i], f[2 * i], f[2 * i + 1]);
}

// 1 / sqrt(sum + eps), or 1 without a normalisation
__device__ __forceinline__ float l2_factor(float sum, float eps) {
    return eps < 0.0f ? 1.0f : 1.0f / __builtin_sqrtf(sum + eps);
}

// One wave per 4 CQ columns of a head's state, whole tokens in its registers:
// lane (rg, cq) = (lane / CQ, lane % CQ) holds rows rg NR .. + NR - 1 of columns
// 4 cq .. + 3.  S^T k and S^T q of the state before the token are summed in one
// pass over the registers and one reduction over the row groups; then
//   u = beta (v - alpha S^T k),  o = scale (alpha S^T q + (k.q) u),
// and the state is updated.
template <int DK, int CQ, bool F16>
__global__ __launch_bounds__(256) void delta_recurrent_kernel(DeltaParams p, int64_t units) {
    constexpr int RG = 64 / CQ, NR = DK / RG;
    const int64_t unit = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (unit >= units) return;
    const int lane = threadIdx.x & 63, cq = lane % CQ, rg = lane / CQ;
    const int slices = p.Dv / (4 * CQ);
    const int64_t bh = unit / slices;
    const int col = int(unit - bh * slices) * 4 * CQ + 4 * cq;
    const int b = int(bh / p.Hv), h = int(bh - int64_t(b) * p.Hv);
    const int slot = entry_state(p.seq, b), len = entry_len(p.seq, b);
    if (slot == kEntryEmpty || len == 0) return;
    uint16_t* const out = p.out + b * p.o_batch + h * p.o_head + col;
    if (slot == kEntryBad) {
        const uint32_t nan2 = Elem<F16>::pack_p(__builtin_nanf(""), __builtin_nanf(""));
        for (int t = rg; t < len; t += RG) *reinterpret_cast<uint2*>(out + t * p.o_tok) = make_uint2(nan2, nan2);
        return;
    }
    float* const st = p.state + ((int64_t(slot) * p.Hv + h) * DK + rg * NR) * p.Dv + col;
    f32x4_t s[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) s[i] = *reinterpret_cast<const f32x4_t*>(st + int64_t(i) * p.Dv);
    const int hk = h / p.G;
    const uint16_t* const q = p.q.p + b * p.q.batch + hk * p.q.head + rg * NR;
    const uint16_t* const k = p.k.p + b * p.k.batch + hk * p.k.head + rg * NR;
    const uint16_t* const v = p.v.p + b * p.v.batch + h * p.v.head + col;
    for (int t = 0; t < len; ++t) {
        float kf[NR], qf[NR], vf[4], g, beta;
        load_elems<F16>(k + t * p.k.tok, kf);
        load_elems<F16>(q + t * p.q.tok, qf);
        load_elems<F16>(v + t * p.v.tok, vf);
        gates<F16>(p, b, t, h, g, beta);
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
        for (int m = CQ; m < 64; m <<= 1)
#pragma unroll
            for (int j = 0; j < 11; ++j) r[j] += __shfl_xor(r[j], m);
        const float rk = l2_factor(r[0], p.l2_eps), rq = p.scale * l2_factor(r[1], p.l2_eps);
        const float alpha = expf(g), kq = r[2] * rk;
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
#pragma unroll
    for (int i = 0; i < NR; ++i) *reinterpret_cast<f32x4_t*>(st + int64_t(i) * p.Dv) = s[i];
}

template <bool F16>
int launch_recurrent(const DeltaParams& p, hipStream_t stream) {
    constexpr int CQ = 4;
    const int64_t units = int64_t(p.B) * p.Hv * (p.Dv / (4 * CQ));
    auto* kern = p.Dk == 128 ? delta_recurrent_kernel<128, CQ, F16> : delta_recurrent_kernel<64, CQ, F16>;
    hipLaunchKernelGGL(kern, dim3(unsigned((units + 3) / 4)), dim3(256), 0, stream, p, units);
    GENLLM_LAUNCH_CHECK("delta_recurrent_kernel");
    return GENLLM_OK;
}

bool strides_ok(const Rows3& r) { return aligned_to(r.p, 16) && ((r.batch | r.tok | r.head) & 7) == 0; }

}  // namespace

}  // namespace genllm

using namespace genllm;

extern "C" size_t genllm_gated_delta_workspace_bytes(int32_t batch, int32_t seq_len, int32_t n_k_heads, int32_t n_v_heads,
                                                     int32_t k_dim, int32_t v_dim) {
    return 0;
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
    if ((k_dim != 64 && k_dim != 128) || (v_dim != 64 && v_dim != 128))
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
    if (int64_t(batch) * n_v_heads > (int64_t(1) << 26))
        return fail(GENLLM_ERR_INVALID, "gated_delta_rule: batch * n_v_heads must be at most 2^26");
    p.a = a, p.b = b, p.a_batch = a_batch_stride, p.a_tok = a_tok_stride, p.b_batch = b_batch_stride, p.b_tok = b_tok_stride;
    p.a_log = a_log, p.dt_bias = dt_bias, p.state = state;
    p.seq.ids = state_ids, p.seq.lens = seq_lens, p.seq.n_states = n_states, p.seq.S = seq_len;
    p.B = batch, p.Hk = n_k_heads, p.Hv = n_v_heads, p.G = n_v_heads / n_k_heads, p.Dk = k_dim, p.Dv = v_dim;
    p.scale = scale, p.l2_eps = l2_eps < 0.0f ? -1.0f : l2_eps;
    return f16 ? launch_recurrent<true>(p, as_stream(stream)) : launch_recurrent<false>(p, as_stream(stream));
}
