// rope_axes.hip -- per-head RMSNorm of q and k with the rotation by positions on
// several axes (time, height, width) in the same pass:
//
//   y = x / sqrt(mean x^2 + eps) * gamma            (gamma given; else y = x)
//   (y[i], y[i + R/2]) rotated by row pos[axis(i)][token] of the cos/sin tables,
//   i < R/2; the dims from R on pass through
//
// in fp32, rounded once.  Pair i belongs to the axis of its section: one section
// after another, or interleaved (pair i to axis i mod n while that axis has
// pairs left, else to axis 0).
#include <climits>
#include <cmath>

#include "common.hpp"
#include "kernels.hpp"
#include "sequences.hpp"

namespace genllm {

namespace {

constexpr int kMaxAxes = 4;

struct AxesRows {  // q or k: [S][H][D], strides in elements
    const uint16_t* x = nullptr;
    int64_t x_tok = 0, x_head = 0;
    uint16_t* out = nullptr;
    int64_t o_tok = 0, o_head = 0;
    const float* gamma = nullptr;
};

struct AxesParams {
    AxesRows q, k;
    int32_t Hq = 0, Hk = 0, S = 0, rope_dim = 0, max_seq = 0, n_axes = 0;
    float eps = 0.0f;
    const float* cos_tab = nullptr;
    const float* sin_tab = nullptr;
    const int32_t* pos = nullptr;  // [n_axes][pos_stride]
    int64_t pos_stride = 0;
    uint16_t axis_bits[16] = {};  // two bits per pair, eight pairs per entry
};

template <bool F16>
__device__ __forceinline__ void unpack8(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = Elem<F16>::lo(w[i]), f[2 * i + 1] = Elem<F16>::hi(w[i]);
}

template <bool F16>
__device__ __forceinline__ uint4 pack8(const float* f) {
    return make_uint4(Elem<F16>::pack_p(f[0], f[1]), Elem<F16>::pack_p(f[2], f[3]), Elem<F16>::pack_p(f[4], f[5]),
                      Elem<F16>::pack_p(f[6], f[7]));
}

// D/16 lanes per row of D elements.  The first rope_dim/16 lanes hold eight pairs
// each (two runs of eight elements, R/2 apart), the others sixteen elements that
// pass through.
template <int D, bool F16>
__global__ __launch_bounds__(256) void norm_rope_axes_kernel(AxesParams p, int64_t rows) {
    constexpr int L = D / 16;
    const int64_t idx = int64_t(blockIdx.x) * 256 + threadIdx.x;
    const int slot = int(idx % L);
    const int64_t row = idx / L;
    if (row >= rows) return;  // whole rows: the lanes of one row leave together
    const int H = p.Hq + p.Hk;
    const int64_t t = row / H;
    int h = int(row - t * H);
    const bool is_k = h >= p.Hq;
    if (is_k) h -= p.Hq;
    const AxesRows& r = is_k ? p.k : p.q;
    const int half = p.rope_dim / 2, rot = p.rope_dim / 16;
    const bool turns = slot < rot;
    const int e0 = turns ? 8 * slot : p.rope_dim + 16 * (slot - rot), e1 = turns ? e0 + half : e0 + 8;
    const uint16_t* const x = r.x + t * r.x_tok + h * r.x_head;
    float y[16];
    unpack8<F16>(*reinterpret_cast<const uint4*>(x + e0), y);
    unpack8<F16>(*reinterpret_cast<const uint4*>(x + e1), y + 8);
    if (r.gamma) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = __builtin_fmaf(y[i], y[i], ss);
#pragma unroll
        for (int m = 1; m < L; m <<= 1) ss += __shfl_xor(ss, m);
        const float f = 1.0f / __builtin_sqrtf(ss * (1.0f / D) + p.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            y[i] = y[i] * f * r.gamma[e0 + i];
            y[8 + i] = y[8 + i] * f * r.gamma[e1 + i];
        }
    }
    if (turns) {
        const uint32_t bits = p.axis_bits[slot];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int axis = int(bits >> (2 * i)) & 3;
            const int32_t at = p.pos[axis * p.pos_stride + t];
            float c = __builtin_nanf(""), s = c;  // a position outside the tables
            if (uint32_t(at) < uint32_t(p.max_seq)) {
                c = p.cos_tab[int64_t(at) * p.rope_dim + e0 + i];
                s = p.sin_tab[int64_t(at) * p.rope_dim + e0 + i];
            }
            const float y0 = y[i], y1 = y[8 + i];
            y[i] = __builtin_fmaf(y0, c, -(y1 * s));
            y[8 + i] = __builtin_fmaf(y0, s, y1 * c);
        }
    }
    uint16_t* const o = r.out + t * r.o_tok + h * r.o_head;
    *reinterpret_cast<uint4*>(o + e0) = pack8<F16>(y);
    *reinterpret_cast<uint4*>(o + e1) = pack8<F16>(y + 8);
}

template <bool F16>
int launch_axes(const AxesParams& p, int D, hipStream_t stream) {
    const int64_t rows = int64_t(p.S) * (p.Hq + p.Hk), blocks = (rows * (D / 16) + 255) / 256;
    if (blocks > INT_MAX / 256) return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: more rows than one launch takes");
    auto* k = D == 64 ? norm_rope_axes_kernel<64, F16>
                      : D == 128 ? norm_rope_axes_kernel<128, F16> : norm_rope_axes_kernel<256, F16>;
    hipLaunchKernelGGL(k, dim3(unsigned(blocks)), dim3(256), 0, stream, p, rows);
    GENLLM_LAUNCH_CHECK("norm_rope_axes_kernel");
    return GENLLM_OK;
}

bool rows_ok(const AxesRows& r) {
    return aligned_to(r.x, 16) && aligned_to(r.out, 16) && aligned_to(r.gamma, 4) &&
           ((r.x_tok | r.x_head | r.o_tok | r.o_head) & 7) == 0;
}

}  // namespace

}  // namespace genllm

using namespace genllm;

extern "C" int genllm_qk_norm_rope_axes(const void* q, int64_t q_tok_stride, int64_t q_head_stride, void* q_out,
                                        int64_t qo_tok_stride, int64_t qo_head_stride, const float* gamma_q,
                                        int32_t n_q_heads, const void* k, int64_t k_tok_stride, int64_t k_head_stride,
                                        void* k_out, int64_t ko_tok_stride, int64_t ko_head_stride, const float* gamma_k,
                                        int32_t n_k_heads, float eps, const float* cos_tab, const float* sin_tab,
                                        int32_t max_seq, int32_t rope_dim, const int32_t* positions, int64_t pos_stride,
                                        int32_t n_axes, const int32_t* sections, int32_t interleaved, int32_t seq_len,
                                        int32_t head_dim, int32_t dtype, void* stream) {
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return fail(GENLLM_ERR_UNSUPPORTED, "qk_norm_rope_axes: head_dim 64, 128 or 256 are served");
    if (dtype != GENLLM_DTYPE_BF16 && dtype != GENLLM_DTYPE_F16)
        return fail(GENLLM_ERR_UNSUPPORTED, "qk_norm_rope_axes: bf16 or fp16 elements");
    if (seq_len < 0 || n_q_heads < 0 || n_k_heads < 0 || max_seq < 0)
        return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: negative size");
    if (rope_dim <= 0 || rope_dim > head_dim || rope_dim % 16)
        return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: rope_dim must be a multiple of 16, at most head_dim");
    if (n_axes < 1 || n_axes > kMaxAxes || !sections)
        return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: 1 to 4 axes with a section each");
    if (!std::isfinite(eps) || eps < 0.0f) return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: eps must be finite and >= 0");
    const int half = rope_dim / 2;
    int64_t total = 0;
    for (int i = 0; i < n_axes; ++i) {
        if (sections[i] < 0) return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: negative section");
        total += sections[i];
    }
    if (total != half) return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: the sections must sum to rope_dim / 2");
    AxesParams p;
    int count[kMaxAxes] = {};
    for (int i = 0, axis = 0, first = 0; i < half; ++i) {
        if (interleaved) {
            axis = i / n_axes < sections[i % n_axes] ? i % n_axes : 0;
        } else {
            while (i >= first + sections[axis]) first += sections[axis++];
        }
        ++count[axis];
        p.axis_bits[i / 8] = uint16_t(p.axis_bits[i / 8] | axis << (2 * (i % 8)));
    }
    for (int i = 0; i < n_axes; ++i)
        if (count[i] != sections[i])
            return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: these sections cannot be interleaved");
    if (seq_len == 0 || n_q_heads + int64_t(n_k_heads) == 0) return GENLLM_OK;
    if (!cos_tab || !sin_tab || !positions || (n_q_heads && (!q || !q_out)) || (n_k_heads && (!k || !k_out)))
        return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: null pointer");
    // the stride of a dim of one never matters
    if (seq_len == 1) q_tok_stride = qo_tok_stride = k_tok_stride = ko_tok_stride = 0;
    if (n_q_heads == 1) q_head_stride = qo_head_stride = 0;
    if (n_k_heads == 1) k_head_stride = ko_head_stride = 0;
    if ((seq_len > 1 && ((n_q_heads && !qo_tok_stride) || (n_k_heads && !ko_tok_stride))) ||
        (n_q_heads > 1 && !qo_head_stride) || (n_k_heads > 1 && !ko_head_stride))
        return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: rows of an output share memory");
    p.q = {static_cast<const uint16_t*>(q), q_tok_stride, q_head_stride, static_cast<uint16_t*>(q_out), qo_tok_stride,
           qo_head_stride, gamma_q};
    p.k = {static_cast<const uint16_t*>(k), k_tok_stride, k_head_stride, static_cast<uint16_t*>(k_out), ko_tok_stride,
           ko_head_stride, gamma_k};
    if ((n_q_heads && !rows_ok(p.q)) || (n_k_heads && !rows_ok(p.k)))
        return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: q, k and their outputs must be rows of 16-byte alignment");
    if (!aligned_to(cos_tab, 4) || !aligned_to(sin_tab, 4) || !aligned_to(positions, 4))
        return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: a pointer is not aligned to its type");
    p.Hq = n_q_heads, p.Hk = n_k_heads, p.S = seq_len, p.rope_dim = rope_dim, p.max_seq = max_seq, p.n_axes = n_axes;
    p.eps = eps, p.cos_tab = cos_tab, p.sin_tab = sin_tab, p.pos = positions, p.pos_stride = pos_stride;
    return dtype == GENLLM_DTYPE_F16 ? launch_axes<true>(p, head_dim, as_stream(stream))
                                     : launch_axes<false>(p, head_dim, as_stream(stream));
}
