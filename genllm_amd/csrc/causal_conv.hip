// causal_conv.hip -- the short causal depthwise convolution in front of a
// hybrid model's linear layers, with the last inputs of each sequence as its
// state.  Per channel, over the line (state rows, then the sequence's tokens):
//
//   y[t] = bias + sum_{j < W} w[j] line[t + j]      line[t + W - 1] = x[t]
//   out  = y / (1 + exp(-y))  with silu, else y
//
// in fp32, rounded once.  The new state is the line's last W - 1 rows.  Bound by
// memory: a thread keeps its window in registers, so that 8 tokens cost 11 loads, three
// of them from the cache (8192 channels: 2048 tokens 14.75 us in calls after each other, 4.6
// TB/s; behind a 1 GiB fill of other memory 22.6 us, 8192 tokens 73).  A single token is the
// launch and one load after another, id then state (4.4 us).
#include <algorithm>
#include <climits>
#include <string>

#include "common.hpp"
#include "kernels.hpp"
#include "rows.hpp"
#include "sequences.hpp"

namespace genllm {

namespace {

struct ConvParams {
    const uint16_t* x = nullptr;
    int64_t x_batch = 0, x_tok = 0;
    uint16_t* out = nullptr;
    int64_t o_batch = 0, o_tok = 0;
    const uint16_t* w = nullptr;  // [C][W]
    const uint16_t* bias = nullptr;
    uint16_t* state = nullptr;  // [n_states][W - 1][C], or null: zeros before each sequence
    Sequences seq;
    int32_t B = 0, C = 0, silu = 0;
    uint32_t c_blocks = 0, tiles = 0;
};

// V channels of one row: V = 8 one 16-byte access, V = 1 one element
template <int V>
struct Lane {
    uint32_t w[V == 8 ? 4 : 1];
};
template <int V>
__device__ __forceinline__ Lane<V> load_lane(const uint16_t* p) {
    Lane<V> r;
    if constexpr (V == 8) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        r.w[0] = u.x, r.w[1] = u.y, r.w[2] = u.z, r.w[3] = u.w;
    } else {
        r.w[0] = *p;
    }
    return r;
}
template <int V>
__device__ __forceinline__ void store_lane(uint16_t* p, const Lane<V>& r) {
    if constexpr (V == 8)
        *reinterpret_cast<uint4*>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    else
        *p = uint16_t(r.w[0]);
}
template <bool F16, int V>
__device__ __forceinline__ float elem(const Lane<V>& r, int i) {
    return i & 1 ? Elem<F16>::hi(r.w[i >> 1]) : Elem<F16>::lo(r.w[i >> 1]);
}

// The weights of V channels: with V = 8 they are 8 W elements in a row.
template <int W, int V, bool F16>
__device__ __forceinline__ void load_weights(const ConvParams& p, int c, float (&w)[W][V], float (&bias)[V]) {
    if constexpr (V == 8) {
        Lane<8> x[W], y{};
#pragma unroll
        for (int i = 0; i < W; ++i) x[i] = load_lane<8>(p.w + int64_t(c) * W + 8 * i);
        if (p.bias) y = load_lane<8>(p.bias + c);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            bias[i] = elem<F16, 8>(y, i);
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][i] = elem<F16, 8>(x[(i * W + j) / 8], (i * W + j) % 8);
        }
    } else {
        bias[0] = p.bias ? Elem<F16>::lo(p.bias[c]) : 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) w[j][0] = Elem<F16>::lo(p.w[int64_t(c) * W + j]);
    }
}

// One thread per V channels and TT tokens: all rows of its window are loaded
// before the first is used, and before its state's place is known.  Only the
// threads of a sequence's first tile touch its state: they read the old rows, then
// write the new ones.  x / (1 + exp(-x)) by the hardware's exp2 and reciprocal,
// each off by about one step of fp32, with both sides of the fraction divided by 2^8: the
// reciprocal gives 0 for what is above 2^126, and 1 + exp(-x) is from x = -87.3 on, where
// the result is still 2^-120 (one more product: 2048 tokens of 8192 channels 14.5 -> 14.75
// us; with the library's exp and division, behind a fill, 29.0 instead of 22.6).
template <int W, int V, int TT, bool F16>
__global__ __launch_bounds__(256) void causal_conv_kernel(ConvParams p) {
    static_assert(TT >= W - 1, "only a first tile may see the state");
    prefetch_kernargs<sizeof(ConvParams)>();
    const uint32_t cb = blockIdx.x % p.c_blocks, rest = blockIdx.x / p.c_blocks;
    const int b = int(rest / p.tiles);
    const int t0 = int(rest % p.tiles) * TT;
    const int c = int(cb * 256 + threadIdx.x) * V;
    const int len = entry_len(p.seq, b);
    if (t0 >= len) return;
    const int n = min(TT, len - t0);
    const bool mine = c < p.C;
    const uint16_t* const x = p.x + b * p.x_batch + c;
    Lane<V> row[TT + W - 1] = {};
    float w[W][V], bias[V];
    if (mine) {
#pragma unroll
        for (int j = 0; j < TT + W - 1; ++j) {
            const int t = t0 - (W - 1) + j;
            if (t >= 0 && j < n + W - 1) row[j] = load_lane<V>(x + t * p.x_tok);
        }
        load_weights<W, V, F16>(p, c, w, bias);
    }
    const int slot = entry_state(p.seq, b);
    if (!mine || slot == kEntryEmpty) return;
    uint16_t* const out = p.out + b * p.o_batch + c;
    if (slot == kEntryBad) {
        const uint32_t nan2 = Elem<F16>::pack_p(__builtin_nanf(""), __builtin_nanf(""));
        Lane<V> r;
        for (uint32_t& y : r.w) y = nan2;
        for (int t = t0; t < t0 + n; ++t) store_lane<V>(out + t * p.o_tok, r);
        return;
    }
    if (t0 == 0 && p.state) {
        uint16_t* const st = p.state + int64_t(slot) * (W - 1) * p.C + c;
        Lane<V> last[W - 1];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) row[j] = load_lane<V>(st + int64_t(j) * p.C);
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            const int t = len - (W - 1) + j;
            if (t >= 0)
                last[j] = load_lane<V>(x + t * p.x_tok);
            else  // a sequence shorter than the window: old rows move up
#pragma unroll
                for (int i = 0; i < W - 1; ++i)
                    if (i == t + W - 1) last[j] = row[i];
        }
#pragma unroll
        for (int j = 0; j < W - 1; ++j) store_lane<V>(st + int64_t(j) * p.C, last[j]);
    }
#pragma unroll
    for (int k = 0; k < TT; ++k) {
        if (k >= n) break;
        Lane<V> o;
        float y[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            y[i] = bias[i];
#pragma unroll
            for (int j = 0; j < W; ++j) y[i] = __builtin_fmaf(w[j][i], elem<F16, V>(row[k + j], i), y[i]);
            if (p.silu) y[i] = (y[i] * 0x1p-8f) * __builtin_amdgcn_rcpf(0x1p-8f + exp2_fast(__builtin_fmaf(-kLog2e, y[i], -8.0f)));
        }
        if constexpr (V == 8)
#pragma unroll
            for (int i = 0; i < 4; ++i) o.w[i] = Elem<F16>::pack_p(y[2 * i], y[2 * i + 1]);
        else
            o.w[0] = Elem<F16>::pack_p(y[0], 0.0f);
        store_lane<V>(out + (t0 + k) * p.o_tok, o);
    }
}

template <int W, int V, bool F16>
int launch_conv(ConvParams& p, hipStream_t stream) {
    constexpr int TT = 8;
    p.c_blocks = uint32_t((int64_t(p.C) + 256 * V - 1) / (256 * V));
    p.tiles = uint32_t((int64_t(p.seq.S) + TT - 1) / TT);
    const int64_t grid = int64_t(p.c_blocks) * p.tiles * p.B;
    if (grid > INT_MAX / 256) return fail(GENLLM_ERR_INVALID, "causal_conv: more elements than one launch takes");
    hipLaunchKernelGGL((causal_conv_kernel<W, V, TT, F16>), dim3(unsigned(grid)), dim3(256), 0, stream, p);
    GENLLM_LAUNCH_CHECK("causal_conv_kernel");
    return GENLLM_OK;
}

template <int V, bool F16>
int launch_conv_w(ConvParams& p, int width, hipStream_t stream) {
    return width == 2 ? launch_conv<2, V, F16>(p, stream)
                      : width == 3 ? launch_conv<3, V, F16>(p, stream) : launch_conv<4, V, F16>(p, stream);
}

// "NAME overlaps NAME" where rows would be written that another workgroup reads.
std::string overlap_of(const ConvParams& p, int width) {
    const auto rows = [&](const uint16_t* at, int64_t batch, int64_t tok) {
        Rows r = Rows::whole(at, int64_t(p.C) * 2);
        r.n[0] = p.B, r.n[1] = p.seq.S, r.stride[0] = 2 * batch, r.stride[1] = 2 * tok;
        return r;
    };
    const int64_t states = p.seq.ids ? p.seq.n_states : p.B;
    const NamedRows written[] = {{"out", rows(p.out, p.o_batch, p.o_tok)},
                                 {"the state", Rows::whole(p.state, states * (width - 1) * p.C * 2)}};
    const NamedRows read[] = {{"x", rows(p.x, p.x_batch, p.x_tok)},
                              {"the weight", Rows::whole(p.w, int64_t(p.C) * width * 2)},
                              {"the bias", Rows::whole(p.bias, int64_t(p.C) * 2)},
                              {"state_ids", Rows::whole(p.seq.ids, int64_t(p.B) * 4)},
                              {"seq_lens", Rows::whole(p.seq.lens, int64_t(p.B) * 4)}};
    const char *a, *b;
    if (find_overlap(written, read, [](const Rows&, const Rows&) { return false; }, a, b)) return std::string(a) + " overlaps " + b;
    return rows_shared_within(written[0].rows) ? "rows of out share memory" : std::string();
}

}  // namespace

}  // namespace genllm

using namespace genllm;

extern "C" int genllm_causal_conv(const void* x, int64_t x_batch_stride, int64_t x_tok_stride, const void* weight,
                                  const void* bias, void* out, int64_t o_batch_stride, int64_t o_tok_stride, void* state,
                                  int32_t n_states, const int32_t* state_ids, const int32_t* seq_lens, int32_t batch,
                                  int32_t seq_len, int32_t channels, int32_t width, int32_t dtype, int32_t silu,
                                  void* stream) {
    if (batch < 0 || seq_len < 0 || channels < 0 || n_states < 0)
        return fail(GENLLM_ERR_INVALID, "causal_conv: negative size");
    if (width < 2 || width > 4) return fail(GENLLM_ERR_UNSUPPORTED, "causal_conv: widths of 2, 3 and 4 are served");
    if (dtype != GENLLM_DTYPE_BF16 && dtype != GENLLM_DTYPE_F16)
        return fail(GENLLM_ERR_UNSUPPORTED, "causal_conv: bf16 or fp16 elements");
    if (batch == 0 || seq_len == 0 || channels == 0) return GENLLM_OK;
    if (!x || !weight || !out) return fail(GENLLM_ERR_INVALID, "causal_conv: null pointer");
    if (state_ids && !state) return fail(GENLLM_ERR_INVALID, "causal_conv: state_ids without a state");
    if (state && !state_ids && n_states < batch)
        return fail(GENLLM_ERR_INVALID, "causal_conv: fewer states than batch entries");
    if (!aligned_to(x, 2) || !aligned_to(weight, 2) || !aligned_to(bias, 2) || !aligned_to(out, 2) ||
        !aligned_to(state, 2) || !aligned_to(state_ids, 4) || !aligned_to(seq_lens, 4))
        return fail(GENLLM_ERR_INVALID, "causal_conv: a pointer is not aligned to its type");
    // the stride of a dim of one never matters
    if (batch == 1) x_batch_stride = o_batch_stride = 0;
    if (seq_len == 1) x_tok_stride = o_tok_stride = 0;
    if ((batch > 1 && !o_batch_stride) || (seq_len > 1 && !o_tok_stride))
        return fail(GENLLM_ERR_INVALID, "causal_conv: rows of out share memory");
    ConvParams p;
    p.x = static_cast<const uint16_t*>(x), p.x_batch = x_batch_stride, p.x_tok = x_tok_stride;
    p.out = static_cast<uint16_t*>(out), p.o_batch = o_batch_stride, p.o_tok = o_tok_stride;
    p.w = static_cast<const uint16_t*>(weight), p.bias = static_cast<const uint16_t*>(bias);
    p.state = static_cast<uint16_t*>(state);
    p.seq.ids = state_ids, p.seq.lens = seq_lens, p.seq.n_states = n_states, p.seq.S = seq_len;
    p.B = batch, p.C = channels, p.silu = silu != 0;
    if (const std::string why = overlap_of(p, width); !why.empty()) return fail(GENLLM_ERR_INVALID, "causal_conv: " + why);
    // 16 bytes per access, or one element where rows do not allow it (2048 tokens of 8192 channels, behind a 1 GiB fill, 22.6 against 34.3 us)
    const bool wide = channels % 8 == 0 && ((x_batch_stride | x_tok_stride | o_batch_stride | o_tok_stride) & 7) == 0 &&
                      aligned_to(x, 16) && aligned_to(out, 16) && aligned_to(state, 16) && aligned_to(weight, 16) &&
                      aligned_to(bias, 16);
    const hipStream_t s = as_stream(stream);
    if (dtype == GENLLM_DTYPE_F16) return wide ? launch_conv_w<8, true>(p, width, s) : launch_conv_w<1, true>(p, width, s);
    return wide ? launch_conv_w<8, false>(p, width, s) : launch_conv_w<1, false>(p, width, s);
}
