// pages_f8.hip -- rows of a batch quantised into 8-bit pages, and read back.
//
// A page of 16 tokens and a head have one scale 2^e, e the least with max |x| <= 448 2^e
// over what was written to it and at least -100, kept as the byte e + 127; a code is
// x 2^-e rounded to e4m3 (four significant bits, ties to even).  Powers of two make both
// directions exact but for that one rounding, and let a page grow: where a token raises
// e, the codes that the page already has are multiplied by 2^(old e - e), which rounds
// only those that end below 2^-6 (e4m3's subnormals).  So a page holds the same codes
// whether its tokens came at once or one by one, but for such.
//
// One wave per (K or V, page, head): lane l has token l / 4 and, of each 64 dims, 16 from
// 16 (l % 4) on: two 16-byte loads to one 16-byte store, 64 bytes of a row together.
//
// Bound by memory where there are many rows, else by the launch (8 heads of 128: 8192 tokens
// read back in 11.0 us, 91 % of a large copy's rate; 2048 written in 4.5 us, and one token of
// each of 64 entries in 4.4, of which the launch is 4.3).
#include <algorithm>
#include <climits>
#include <string>

#include "common.hpp"
#include "rows.hpp"
#include "sequences.hpp"

namespace genllm {

namespace {

constexpr int kLeastExponent = -100;

struct PagesF8 {
    // rows of elements: [B][S][Hkv][D], strides in elements; K, then V
    uint16_t* rows[2] = {};
    int64_t batch[2] = {}, tok[2] = {}, head[2] = {};
    // pools: strides in bytes
    uint8_t* pool[2] = {};
    int64_t block[2] = {}, p_tok[2] = {}, p_head[2] = {};
    uint8_t* scales[2] = {};  // [blocks][Hkv]
    const int32_t* ids[2] = {};
    int64_t ids_row[2] = {};
    const int32_t* start = nullptr;
    const int32_t* lens = nullptr;
    int32_t B = 0, S = 0, Hkv = 0, blocks = 0, max_pages = 0;
    uint32_t pages = 0;  // pages that an entry may touch
};

struct Place {
    int kind, b, h, page;  // page of the table
    int from, to;          // slots of the page within the entry's tokens
    int first;             // token of the entry in slot 0 (negative: before its first)
};

// What this wave does; false: nothing.
__device__ __forceinline__ bool place_of(const PagesF8& p, Place& r) {
    uint32_t w = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    r.h = int(w % uint32_t(p.Hkv)), w /= uint32_t(p.Hkv);
    const uint32_t j = w % p.pages;
    w /= p.pages;
    r.kind = int(w & 1), r.b = int(w >> 1);
    if (r.b >= p.B) return false;
    const int start = p.start[r.b];
    int n = p.lens ? p.lens[r.b] : p.S;
    n = min(max(n, 0), p.S);
    if (start < 0) return false;  // an idle entry
    r.page = start / kPage + int(j);
    r.first = int(j) * kPage - start % kPage;
    r.from = max(-r.first, 0), r.to = min(n - r.first, kPage);
    return r.from < r.to;
}

__device__ __forceinline__ float wave_max(float x) {
    x = row16_max(x);
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}

// the least e with x <= 448 2^e, from kLeastExponent on
__device__ __forceinline__ int exponent_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return max(int(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0), kLeastExponent);
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float(uint32_t(min(max(e, -126), 127) + 127) << 23); }

__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
}
__device__ __forceinline__ void values4(uint32_t w, float (&x)[4]) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
    x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
}

template <int D, bool F16>
__global__ __launch_bounds__(256) void scatter_f8_kernel(PagesF8 p) {
    using E = Elem<F16>;
    constexpr int C = D / 64;  // 16-dim chunks of a lane
    prefetch_kernargs<sizeof(PagesF8)>();
    Place at;
    if (!place_of(p, at) || at.page >= p.max_pages) return;
    const int k = at.kind, lane = threadIdx.x & 63, slot = lane >> 2;
    const int id = p.ids[k][at.b * p.ids_row[k] + at.page];
    const bool mine = slot >= at.from && slot < at.to;
    uint4 x[2 * C];
    if (mine) {
        const uint16_t* const row = p.rows[k] + at.b * p.batch[k] + int64_t(at.first + slot) * p.tok[k] + at.h * p.head[k] + 16 * (lane & 3);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            x[2 * c] = *reinterpret_cast<const uint4*>(row + 64 * c);
            x[2 * c + 1] = *reinterpret_cast<const uint4*>(row + 64 * c + 8);
        }
    } else {
#pragma unroll
        for (int c = 0; c < 2 * C; ++c) x[c] = make_uint4(0, 0, 0, 0);
    }
    if (unsigned(id) >= unsigned(p.blocks)) return;
    uint8_t* const scale = p.scales[k] + int64_t(id) * p.Hkv + at.h;
    uint8_t* const page = p.pool[k] + id * p.block[k] + at.h * p.p_head[k] + slot * p.p_tok[k] + 16 * (lane & 3);
    const bool grows = at.from > 0;  // the page has tokens from before
    const int had = grows ? *scale : 0;
    uint4 old[C];
    if (grows && !mine) {
#pragma unroll
        for (int c = 0; c < C; ++c) old[c] = *reinterpret_cast<const uint4*>(page + 64 * c);
    }
    float most = 0.0f;  // of the finite values
#pragma unroll
    for (int c = 0; c < 2 * C; ++c) {
        const uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = fabsf(E::lo(w[i])), b = fabsf(E::hi(w[i]));
            most = fmaxf(most, a <= __FLT_MAX__ ? a : 0.0f);
            most = fmaxf(most, b <= __FLT_MAX__ ? b : 0.0f);
        }
    }
    int e = exponent_of(wave_max(most));
    if (grows) e = max(e, had - 127);
    const float f = two_to(-e);
    if (mine) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            uint32_t r[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 u = x[2 * c + (i >> 1)];
                const uint32_t a = i & 1 ? u.z : u.x, b = i & 1 ? u.w : u.y;
                r[i] = codes4(E::lo(a) * f, E::hi(a) * f, E::lo(b) * f, E::hi(b) * f);
            }
            *reinterpret_cast<uint4*>(page + 64 * c) = make_uint4(r[0], r[1], r[2], r[3]);
        }
    } else if (grows && e != had - 127) {
        const float by = two_to(had - 127 - e);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint32_t w[4] = {old[c].x, old[c].y, old[c].z, old[c].w};
            uint32_t r[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[4];
                values4(w[i], v);
                r[i] = codes4(v[0] * by, v[1] * by, v[2] * by, v[3] * by);
            }
            *reinterpret_cast<uint4*>(page + 64 * c) = make_uint4(r[0], r[1], r[2], r[3]);
        }
    }
    if (lane == 0 && !(grows && had == 255)) *scale = uint8_t(e + 127);
}

template <int D, bool F16>
__global__ __launch_bounds__(256) void gather_f8_kernel(PagesF8 p) {
    using E = Elem<F16>;
    constexpr int C = D / 64;
    prefetch_kernargs<sizeof(PagesF8)>();
    Place at;
    if (!place_of(p, at)) return;
    const int k = at.kind, lane = threadIdx.x & 63, slot = lane >> 2;
    const int id = at.page < p.max_pages ? p.ids[k][at.b * p.ids_row[k] + at.page] : -1;
    const bool there = unsigned(id) < unsigned(p.blocks);
    if (slot < at.from || slot >= at.to) return;
    float s = __builtin_nanf("");
    uint4 w[C];
#pragma unroll
    for (int c = 0; c < C; ++c) w[c] = make_uint4(0, 0, 0, 0);
    if (there) {
        const uint8_t* const page = p.pool[k] + id * p.block[k] + at.h * p.p_head[k] + slot * p.p_tok[k] + 16 * (lane & 3);
#pragma unroll
        for (int c = 0; c < C; ++c) w[c] = *reinterpret_cast<const uint4*>(page + 64 * c);
        const int byte = p.scales[k][int64_t(id) * p.Hkv + at.h];
        if (byte != 255) s = __uint_as_float(byte ? uint32_t(byte) << 23 : 0x00400000u);
    }
    uint16_t* const row = p.rows[k] + at.b * p.batch[k] + int64_t(at.first + slot) * p.tok[k] + at.h * p.head[k] + 16 * (lane & 3);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t u[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
        uint32_t r[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v[4];
            values4(u[i], v);
            r[2 * i] = E::pack_p(v[0] * s, v[1] * s);
            r[2 * i + 1] = E::pack_p(v[2] * s, v[3] * s);
        }
        *reinterpret_cast<uint4*>(row + 64 * c) = make_uint4(r[0], r[1], r[2], r[3]);
        *reinterpret_cast<uint4*>(row + 64 * c + 8) = make_uint4(r[4], r[5], r[6], r[7]);
    }
}

template <bool kScatter, bool F16>
int launch(const PagesF8& p, int D, unsigned grid, hipStream_t s) {
    const dim3 block(256);
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), block, 0, s, p); };
    if constexpr (kScatter)
        D == 64 ? go(scatter_f8_kernel<64, F16>) : D == 128 ? go(scatter_f8_kernel<128, F16>) : go(scatter_f8_kernel<256, F16>);
    else
        D == 64 ? go(gather_f8_kernel<64, F16>) : D == 128 ? go(gather_f8_kernel<128, F16>) : go(gather_f8_kernel<256, F16>);
    GENLLM_LAUNCH_CHECK("pages_f8 kernel");
    return GENLLM_OK;
}

struct Call {
    void* k;
    int64_t k_batch, k_tok, k_head;
    void* v;
    int64_t v_batch, v_tok, v_head;
    void* k_pool;
    int64_t kp_block, kp_tok, kp_head;
    void* v_pool;
    int64_t vp_block, vp_tok, vp_head;
    uint8_t *k_scales, *v_scales;
    int32_t n_blocks;
    const int32_t* k_ids;
    int64_t k_ids_stride;
    const int32_t* v_ids;
    int64_t v_ids_stride;
    int32_t max_pages;
    const int32_t *start_pos, *seq_lens;
    int32_t batch, seq_len, n_kv_heads, head_dim, dtype;
    void* stream;
};

template <bool kScatter>
int run(const Call& c) {
    const char* const op = kScatter ? "kv_scatter_f8: " : "kv_gather_f8: ";
    const auto refuse = [&](int code, const std::string& why) { return fail(code, op + why); };
    if (c.batch < 0 || c.seq_len < 0 || c.n_kv_heads < 0 || c.n_blocks < 0 || c.max_pages < 0) return refuse(GENLLM_ERR_INVALID, "negative size");
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return refuse(GENLLM_ERR_UNSUPPORTED, "head_dim 64, 128 or 256");
    if (c.dtype != GENLLM_DTYPE_BF16 && c.dtype != GENLLM_DTYPE_F16) return refuse(GENLLM_ERR_UNSUPPORTED, "bf16 or fp16 elements");
    if (c.max_pages > 1 << 26) return refuse(GENLLM_ERR_INVALID, "tables of up to 2^26 pages");
    if (c.seq_len > 1 << 30) return refuse(GENLLM_ERR_INVALID, "up to 2^30 tokens");
    if (c.batch == 0 || c.seq_len == 0 || c.n_kv_heads == 0) return GENLLM_OK;
    if (!c.k || !c.v || !c.k_pool || !c.v_pool || !c.k_scales || !c.v_scales || (c.max_pages > 0 && (!c.k_ids || !c.v_ids)) || !c.start_pos)
        return refuse(GENLLM_ERR_INVALID, "null pointer");
    if (!aligned_to(c.k, 16) || !aligned_to(c.v, 16) || !aligned_to(c.k_pool, 16) || !aligned_to(c.v_pool, 16) ||
        ((c.k_batch | c.k_tok | c.k_head | c.v_batch | c.v_tok | c.v_head) & 7) ||
        ((c.kp_block | c.kp_tok | c.kp_head | c.vp_block | c.vp_tok | c.vp_head) & 15))
        return refuse(GENLLM_ERR_INVALID, "rows must be 16-byte aligned");
    if (!aligned_to(c.k_ids, 4) || !aligned_to(c.v_ids, 4) || !aligned_to(c.start_pos, 4) || !aligned_to(c.seq_lens, 4))
        return refuse(GENLLM_ERR_INVALID, "a pointer is not aligned to its type");

    PagesF8 p;
    const auto one = [](int64_t stride, int64_t n) { return n > 1 ? stride : 0; };  // the stride of a dim of one never matters
    void* const rows[2] = {c.k, c.v};
    void* const pools[2] = {c.k_pool, c.v_pool};
    const int64_t rs[2][3] = {{c.k_batch, c.k_tok, c.k_head}, {c.v_batch, c.v_tok, c.v_head}};
    const int64_t ps[2][3] = {{c.kp_block, c.kp_tok, c.kp_head}, {c.vp_block, c.vp_tok, c.vp_head}};
    Rows as_rows[2], as_pool[2], as_ids[2];
    for (int i = 0; i < 2; ++i) {
        p.rows[i] = static_cast<uint16_t*>(rows[i]), p.pool[i] = static_cast<uint8_t*>(pools[i]);
        p.batch[i] = one(rs[i][0], c.batch), p.tok[i] = one(rs[i][1], c.seq_len), p.head[i] = one(rs[i][2], c.n_kv_heads);
        p.block[i] = one(ps[i][0], c.n_blocks), p.p_tok[i] = ps[i][1], p.p_head[i] = one(ps[i][2], c.n_kv_heads);
        Rows r = Rows::whole(rows[i], int64_t(c.head_dim) * 2);
        r.n[0] = c.batch, r.n[1] = c.seq_len, r.n[2] = c.n_kv_heads;
        r.stride[0] = 2 * p.batch[i], r.stride[1] = 2 * p.tok[i], r.stride[2] = 2 * p.head[i];
        as_rows[i] = r;
        r = Rows::whole(pools[i], c.head_dim);
        r.n[0] = c.n_blocks, r.n[1] = kPage, r.n[2] = c.n_kv_heads;
        r.stride[0] = p.block[i], r.stride[1] = p.p_tok[i], r.stride[2] = p.p_head[i];
        as_pool[i] = r;
        r = Rows::whole(i ? c.v_ids : c.k_ids, int64_t(c.max_pages) * 4);
        r.n[0] = c.batch, r.stride[0] = 4 * one(i ? c.v_ids_stride : c.k_ids_stride, c.batch);
        as_ids[i] = r;
    }
    p.scales[0] = c.k_scales, p.scales[1] = c.v_scales;
    p.ids[0] = c.k_ids, p.ids[1] = c.v_ids;
    p.ids_row[0] = one(c.k_ids_stride, c.batch), p.ids_row[1] = one(c.v_ids_stride, c.batch);
    p.start = c.start_pos, p.lens = c.seq_lens;
    p.B = c.batch, p.S = c.seq_len, p.Hkv = c.n_kv_heads, p.blocks = c.n_blocks, p.max_pages = c.max_pages;
    p.pages = uint32_t((c.seq_len + 14) / kPage + 1);

    const Rows scales[2] = {Rows::whole(c.k_scales, int64_t(c.n_blocks) * c.n_kv_heads), Rows::whole(c.v_scales, int64_t(c.n_blocks) * c.n_kv_heads)};
    const Rows start = Rows::whole(c.start_pos, int64_t(c.batch) * 4), lens = Rows::whole(c.seq_lens, int64_t(c.batch) * 4);
    const char *a, *b;
    const auto never = [](const Rows&, const Rows&) { return false; };
    if constexpr (kScatter) {
        // one pool, with one or two arrays of scales, may hold K's and V's blocks: the tables then name different ones
        const bool one_pool = as_pool[1].same_as(as_pool[0]), one_scales = one_pool && scales[1].same_as(scales[0]);
        const NamedRows written[] = {{"k_pool", as_pool[0]}, {"v_pool", one_pool ? Rows() : as_pool[1]},
                                     {"k_scales", scales[0]}, {"v_scales", one_scales ? Rows() : scales[1]}};
        const NamedRows read[] = {{"k", as_rows[0]}, {"v", as_rows[1]}, {"k_ids", as_ids[0]}, {"v_ids", as_ids[1]}, {"start_pos", start}, {"seq_lens", lens}};
        if (find_overlap(written, read, never, a, b)) return refuse(GENLLM_ERR_INVALID, std::string(a) + " overlaps " + b);
        for (int i = 0; i < 2; ++i)
            if (rows_shared_within(as_pool[i])) return refuse(GENLLM_ERR_INVALID, std::string("rows of ") + (i ? "v_pool" : "k_pool") + " share memory");
    } else {
        const NamedRows written[] = {{"k_out", as_rows[0]}, {"v_out", as_rows[1]}};
        const NamedRows read[] = {{"k_pool", as_pool[0]}, {"v_pool", as_pool[1]}, {"k_scales", scales[0]}, {"v_scales", scales[1]},
                                  {"k_ids", as_ids[0]}, {"v_ids", as_ids[1]}, {"start_pos", start}, {"seq_lens", lens}};
        if (find_overlap(written, read, never, a, b)) return refuse(GENLLM_ERR_INVALID, std::string(a) + " overlaps " + b);
        for (int i = 0; i < 2; ++i)
            if (rows_shared_within(as_rows[i])) return refuse(GENLLM_ERR_INVALID, std::string("rows of ") + (i ? "v_out" : "k_out") + " share memory");
    }
    const __int128 waves = __int128(2) * c.batch * p.pages * c.n_kv_heads;
    if (waves > INT_MAX / 64) return refuse(GENLLM_ERR_INVALID, "more rows than one launch takes");
    const unsigned grid = unsigned((int64_t(waves) + 3) / 4);
    const hipStream_t s = as_stream(c.stream);
    return c.dtype == GENLLM_DTYPE_F16 ? launch<kScatter, true>(p, c.head_dim, grid, s) : launch<kScatter, false>(p, c.head_dim, grid, s);
}

}  // namespace

}  // namespace genllm

using namespace genllm;

extern "C" int genllm_kv_scatter_f8(const void* k, int64_t k_batch_stride, int64_t k_tok_stride, int64_t k_head_stride, const void* v,
                                    int64_t v_batch_stride, int64_t v_tok_stride, int64_t v_head_stride, void* k_pool,
                                    int64_t kp_block_stride, int64_t kp_tok_stride, int64_t kp_head_stride, void* v_pool,
                                    int64_t vp_block_stride, int64_t vp_tok_stride, int64_t vp_head_stride, uint8_t* k_scales,
                                    uint8_t* v_scales, int32_t n_blocks, const int32_t* k_ids, int64_t k_ids_stride,
                                    const int32_t* v_ids, int64_t v_ids_stride, int32_t max_pages, const int32_t* start_pos,
                                    const int32_t* seq_lens, int32_t batch, int32_t seq_len, int32_t n_kv_heads, int32_t head_dim,
                                    int32_t dtype, void* stream) {
    return run<true>({const_cast<void*>(k), k_batch_stride, k_tok_stride, k_head_stride, const_cast<void*>(v), v_batch_stride, v_tok_stride,
                      v_head_stride, k_pool, kp_block_stride, kp_tok_stride, kp_head_stride, v_pool, vp_block_stride, vp_tok_stride,
                      vp_head_stride, k_scales, v_scales, n_blocks, k_ids, k_ids_stride, v_ids, v_ids_stride, max_pages, start_pos,
                      seq_lens, batch, seq_len, n_kv_heads, head_dim, dtype, stream});
}

extern "C" int genllm_kv_gather_f8(const void* k_pool, int64_t kp_block_stride, int64_t kp_tok_stride, int64_t kp_head_stride,
                                   const void* v_pool, int64_t vp_block_stride, int64_t vp_tok_stride, int64_t vp_head_stride,
                                   const uint8_t* k_scales, const uint8_t* v_scales, int32_t n_blocks, const int32_t* k_ids,
                                   int64_t k_ids_stride, const int32_t* v_ids, int64_t v_ids_stride, int32_t max_pages,
                                   const int32_t* start_pos, const int32_t* seq_lens, void* k_out, int64_t k_batch_stride,
                                   int64_t k_tok_stride, int64_t k_head_stride, void* v_out, int64_t v_batch_stride,
                                   int64_t v_tok_stride, int64_t v_head_stride, int32_t batch, int32_t seq_len, int32_t n_kv_heads,
                                   int32_t head_dim, int32_t dtype, void* stream) {
    return run<false>({k_out, k_batch_stride, k_tok_stride, k_head_stride, v_out, v_batch_stride, v_tok_stride, v_head_stride,
                       const_cast<void*>(k_pool), kp_block_stride, kp_tok_stride, kp_head_stride, const_cast<void*>(v_pool),
                       vp_block_stride, vp_tok_stride, vp_head_stride, const_cast<uint8_t*>(k_scales), const_cast<uint8_t*>(v_scales),
                       n_blocks, k_ids, k_ids_stride, v_ids, v_ids_stride, max_pages, start_pos, seq_lens, batch, seq_len, n_kv_heads,
                       head_dim, dtype, stream});
}
