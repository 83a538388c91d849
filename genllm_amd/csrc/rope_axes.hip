// rope_axes.hip -- per-head RMSNorm of q and k with the rotation by positions on
// several axes (time, height, width) in the same pass:
//
//   y = x / sqrt(mean x^2 + eps) * gamma            (gamma given; else y = x)
//   (y[i], y[i + R/2]) rotated by row pos[axis(i)][token] of the cos/sin tables,
//   i < R/2; the dims from R on pass through
//
// in fp32, rounded once.  Every element is read and written once, which bounds long
// calls (32 / 8 heads of 128, with cold caches: 2048 tokens 13.8 us, 3.0 TB/s; 32768
// tokens 134 us, 5.0 TB/s); a short one is the launch and two loads after each other,
// position then table (64 tokens 3.1 us).  Pair i belongs to the axis of its section: one section
// after another, or interleaved (pair i to axis i mod n while that axis has
// pairs left, else to axis 0).
#include <algorithm>
#include <climits>
#include <cmath>
#include <string>

#include "common.hpp"
#include "kernels.hpp"
#include "rows.hpp"
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
    int32_t Hq = 0, Hk = 0, S = 0, rope_dim = 0, max_seq = 0;
    int32_t tokens = 1, heads = 1;  // of a workgroup
    float eps = 0.0f;
    const float* cos_tab = nullptr;
    const float* sin_tab = nullptr;
    const int32_t* pos = nullptr;  // [n_axes][pos_stride]
    int64_t pos_stride = 0;
    uint32_t axis_bits[8] = {};  // two bits per pair, sixteen pairs per word
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
// pass through.  A workgroup has 256 NI / (D/16) rows of neighbouring tokens, or a
// part of one token's heads: it gathers those tokens' cos and sin once, into LDS,
// while its rows are on their way (a gather of 16 values per thread and row
// instead: 11.4 against 7.5 us for 2048 tokens of 10 heads of 256).
template <int D, int NI, bool F16>
__global__ __launch_bounds__(256) void norm_rope_axes_kernel(AxesParams p) {
    constexpr int L = D / 16;
    extern __shared__ __attribute__((aligned(16))) float s_tab[];  // [token][cos of the pairs, sin of them]
    prefetch_kernargs<sizeof(AxesParams)>();
    const int H = p.Hq + p.Hk, half = p.rope_dim / 2, rot = p.rope_dim / 16;
    const int slot = int(threadIdx.x) % L;
    const int t0 = int(blockIdx.x) * p.tokens;
    const int tokens = min(p.tokens, p.S - t0);
    const int h0 = int(blockIdx.y) * p.heads, heads = min(p.heads, H - h0);
    const int rows = tokens * heads;
    const bool turns = slot < rot;
    const int e0 = turns ? 8 * slot : p.rope_dim + 16 * (slot - rot), e1 = turns ? e0 + half : e0 + 8;
    uint4 lo[NI], hi[NI];
    uint16_t* to[NI];
    int tok[NI];
    bool is_k[NI], mine[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int row = (int(threadIdx.x) + 256 * i) / L;
        mine[i] = row < rows;
        tok[i] = row / heads;
        int h = h0 + row - tok[i] * heads;
        is_k[i] = h >= p.Hq;
        if (is_k[i]) h -= p.Hq;
        const AxesRows& r = is_k[i] ? p.k : p.q;
        const int64_t t = t0 + tok[i];
        const uint16_t* const x = r.x + t * r.x_tok + h * r.x_head;
        to[i] = r.out + t * r.o_tok + h * r.o_head;
        if (mine[i]) {
            lo[i] = *reinterpret_cast<const uint4*>(x + e0);
            hi[i] = *reinterpret_cast<const uint4*>(x + e1);
        }
    }
    for (int i = int(threadIdx.x); i < tokens * half; i += 256) {
        const int t = i / half, pair = i - t * half;
        uint32_t word = p.axis_bits[0];  // selected, not indexed: no load from the argument block in front of the position's
#pragma unroll
        for (int j = 1; j < 8; ++j) word = pair >> 4 == j ? p.axis_bits[j] : word;
        const int axis = int(word >> (2 * (pair & 15))) & 3;
        const int32_t at = p.pos[axis * p.pos_stride + t0 + t];
        float c = __builtin_nanf(""), s = c;  // a position outside the tables
        if (uint32_t(at) < uint32_t(p.max_seq)) {
            c = p.cos_tab[int64_t(at) * p.rope_dim + pair];
            s = p.sin_tab[int64_t(at) * p.rope_dim + pair];
        }
        s_tab[2 * t * half + pair] = c;
        s_tab[(2 * t + 1) * half + pair] = s;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        if (!mine[i]) break;  // whole rows: the lanes of one row leave together
        float y[16];
        unpack8<F16>(lo[i], y);
        unpack8<F16>(hi[i], y + 8);
        const float* const gamma = is_k[i] ? p.k.gamma : p.q.gamma;
        if (gamma) {
            const f32x4_t g[4] = {*reinterpret_cast<const f32x4_t*>(gamma + e0), *reinterpret_cast<const f32x4_t*>(gamma + e0 + 4),
                                  *reinterpret_cast<const f32x4_t*>(gamma + e1), *reinterpret_cast<const f32x4_t*>(gamma + e1 + 4)};
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) ss = __builtin_fmaf(y[j], y[j], ss);
            ss += dpp<kDppQuadXor1>(ss);
            ss += dpp<kDppQuadXor2>(ss);
            if constexpr (L >= 8) ss += dpp<kDppRowHalfMirror>(ss);
            if constexpr (L >= 16) ss += dpp<kDppRowMirror>(ss);
            const float f = 1.0f / __builtin_sqrtf(ss * (1.0f / D) + p.eps);
#pragma unroll
            for (int j = 0; j < 16; ++j) y[j] = y[j] * f * g[j >> 2][j & 3];
        }
        if (turns) {
            const f32x4_t* const tab = reinterpret_cast<const f32x4_t*>(s_tab + 2 * tok[i] * half + e0);
            const f32x4_t c[2] = {tab[0], tab[1]}, s[2] = {tab[half / 4], tab[half / 4 + 1]};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y0 = y[j], y1 = y[8 + j], cj = c[j >> 2][j & 3], sj = s[j >> 2][j & 3];
                y[j] = __builtin_fmaf(y0, cj, -(y1 * sj));
                y[8 + j] = __builtin_fmaf(y0, sj, y1 * cj);
            }
        }
        *reinterpret_cast<uint4*>(to[i] + e0) = pack8<F16>(y);
        *reinterpret_cast<uint4*>(to[i] + e1) = pack8<F16>(y + 8);
    }
}

template <int D, int NI, bool F16>
int launch_axes_rows(AxesParams& p, hipStream_t stream) {
    constexpr int kRows = 256 * NI / (D / 16), kMaxTokens = 16;
    const int64_t H = int64_t(p.Hq) + p.Hk;
    p.heads = int32_t(std::min<int64_t>(H, kRows));
    p.tokens = H > kRows ? 1 : std::min(kMaxTokens, int(kRows / H));
    const int64_t blocks = (int64_t(p.S) + p.tokens - 1) / p.tokens, parts = (H + p.heads - 1) / p.heads;
    if (blocks > INT_MAX / 256 || parts > 65535)
        return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: more rows than one launch takes");
    hipLaunchKernelGGL((norm_rope_axes_kernel<D, NI, F16>), dim3(unsigned(blocks), unsigned(parts)), dim3(256),
                       size_t(p.tokens) * p.rope_dim * sizeof(float), stream, p);
    GENLLM_LAUNCH_CHECK("norm_rope_axes_kernel");
    return GENLLM_OK;
}

// Four rows per lane where that still gives every CU four workgroups: a table row
// serves four times the heads and more loads are in flight per lane.  Else one (one
// against four, us: 32 / 8 heads of 128, 64 tokens 3.1 / 5.2, 1024 8.3 / 10.6, 4096
// 24.2 / 24.2, 8192 43.2 / 40.4, 32768 154 / 134; 8 / 2 of 256, 2048 8.7 / 10.8, 8192 24.7 /
// 25.5, 32768 79.0 / 77.8).
template <int D, bool F16>
int launch_axes_dim(AxesParams& p, hipStream_t stream) {
    const int64_t lanes = int64_t(p.S) * (int64_t(p.Hq) + p.Hk) * (D / 16);
    return lanes >= int64_t(device_cu_count()) * 4 * 256 * 4 ? launch_axes_rows<D, 4, F16>(p, stream)
                                                             : launch_axes_rows<D, 1, F16>(p, stream);
}

template <bool F16>
int launch_axes(AxesParams& p, int D, hipStream_t stream) {
    return D == 64 ? launch_axes_dim<64, F16>(p, stream)
                   : D == 128 ? launch_axes_dim<128, F16>(p, stream) : launch_axes_dim<256, F16>(p, stream);
}

bool rows_ok(const AxesRows& r) {
    return aligned_to(r.x, 16) && aligned_to(r.out, 16) && aligned_to(r.gamma, 16) &&
           ((r.x_tok | r.x_head | r.o_tok | r.o_head) & 7) == 0;
}

// "NAME overlaps NAME" where a row would be written that another workgroup reads.  An
// output may be its own input: a row is in registers before it is written.
std::string overlap_of(const AxesParams& p, int D, int n_axes) {
    const auto rows = [&](const uint16_t* at, int64_t tok, int64_t head, int32_t heads) {
        Rows r = Rows::whole(heads ? at : nullptr, 2 * D);
        r.n[0] = p.S, r.n[1] = heads, r.stride[0] = 2 * tok, r.stride[1] = 2 * head;
        return r;
    };
    const Rows q = rows(p.q.x, p.q.x_tok, p.q.x_head, p.Hq), k = rows(p.k.x, p.k.x_tok, p.k.x_head, p.Hk);
    const int64_t table = int64_t(p.max_seq) * p.rope_dim * 4;
    Rows pos = Rows::whole(p.pos, int64_t(p.S) * 4);
    pos.n[0] = n_axes, pos.stride[0] = p.pos_stride * 4;
    const NamedRows written[] = {{"q_out", rows(p.q.out, p.q.o_tok, p.q.o_head, p.Hq)}, {"k_out", rows(p.k.out, p.k.o_tok, p.k.o_head, p.Hk)}};
    const NamedRows read[] = {{"q", q},
                              {"k", k},
                              {"gamma_q", Rows::whole(p.Hq ? p.q.gamma : nullptr, D * 4)},
                              {"gamma_k", Rows::whole(p.Hk ? p.k.gamma : nullptr, D * 4)},
                              {"cos", Rows::whole(p.cos_tab, table)},
                              {"sin", Rows::whole(p.sin_tab, table)},
                              {"positions", pos}};
    const char *a, *b;
    const auto in_place = [&](const Rows& w, const Rows& r) {
        return w.same_as(r) && (&r == &read[0].rows ? &w == &written[0].rows : &r == &read[1].rows && &w == &written[1].rows);
    };
    if (find_overlap(written, read, in_place, a, b)) return std::string(a) + " overlaps " + b;
    for (const NamedRows& w : written)
        if (rows_shared_within(w.rows)) return std::string("rows of ") + w.name + " share memory";
    return {};
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
        p.axis_bits[i / 16] |= uint32_t(axis) << (2 * (i % 16));
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
    const auto moved = [](const AxesRows& r) { return r.x == r.out && (r.x_tok != r.o_tok || r.x_head != r.o_head); };
    if ((n_q_heads && moved(p.q)) || (n_k_heads && moved(p.k)))
        return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: an output over its input needs the same strides");
    if ((n_q_heads && !rows_ok(p.q)) || (n_k_heads && !rows_ok(p.k)))
        return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: q, k, their outputs and gammas must be 16-byte aligned");
    if (!aligned_to(cos_tab, 4) || !aligned_to(sin_tab, 4) || !aligned_to(positions, 4))
        return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: a pointer is not aligned to its type");
    p.Hq = n_q_heads, p.Hk = n_k_heads, p.S = seq_len, p.rope_dim = rope_dim, p.max_seq = max_seq;
    p.eps = eps, p.cos_tab = cos_tab, p.sin_tab = sin_tab, p.pos = positions, p.pos_stride = pos_stride;
    if (const std::string why = overlap_of(p, head_dim, n_axes); !why.empty())
        return fail(GENLLM_ERR_INVALID, "qk_norm_rope_axes: " + why);
    return dtype == GENLLM_DTYPE_F16 ? launch_axes<true>(p, head_dim, as_stream(stream))
                                     : launch_axes<false>(p, head_dim, as_stream(stream));
}
