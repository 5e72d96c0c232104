// kv8_append.cu -- mg_kv8_append: new keys and values into the 8-bit paged
// cache, with the head norm and the position rotation on the way (the QK-norm,
// RoPE and cache write of layers.mojo:43-61), and the rotated queries.
//
// One CTA owns one block of 16 positions of one sequence and kv head: the
// block's scale is a maximum over its tokens, so the tokens of the call that
// fall into it, its earlier codes and its scale all belong to one CTA, and the
// q heads of the same tokens and kv head go along (they share the cos / sin
// rows).  A head vector is held by head_dim / 8 lanes, lane i with elements
// 4 i .. 4 i + 3 of each half, so that a rotation's pairs meet in one lane and
// loads are 4 elements wide.
//
// The work is memory traffic: the rows in, the rotated queries and one byte
// per value out; per element a norm and a rotation are a few operations.
#include "kv8.cuh"

#include <cstdio>

namespace mg {
namespace kv8 {
namespace {

constexpr int kThreads = 256;

struct AppendParams {
    Cache c;
    Batch b;
    const void *q, *k, *v;
    void *q_out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
    const float *q_norm, *k_norm, *cos_t, *sin_t;
    int group;            // q heads per kv head (0: no queries)
    int blocks_per_seq;   // > 0: block index = sequence * this + block; 0: by rows, seq_of_block
};

template <typename T>
__device__ __forceinline__ void load4(const T *p, float (&x)[4]);
template <>
__device__ __forceinline__ void load4<float>(const float *p, float (&x)[4]) {
    const float4 v = *reinterpret_cast<const float4 *>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
template <>
__device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16 *p, float (&x)[4]) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
}
template <>
__device__ __forceinline__ void load4<__half>(const __half *p, float (&x)[4]) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
__device__ __forceinline__ void store4(float *p, const float *x) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store4(__nv_bfloat16 *p, const float *x) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    *reinterpret_cast<uint2 *>(p) =
        make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}
__device__ __forceinline__ void store4(__half *p, const float *x) {
    const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
    *reinterpret_cast<uint2 *>(p) =
        make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

// A head vector's 8 elements of this lane: 0-3 from the first half, 4-7 from the second.
template <int HD, typename T>
__device__ __forceinline__ void load_vec(const T *p, int gl, float (&x)[8]) {
    float a[4], b[4];
    load4<T>(p + 4 * gl, a);
    load4<T>(p + HD / 2 + 4 * gl, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
}
// x <- rope(norm(x)) at position pos.
template <int HD>
__device__ __forceinline__ void turn(float (&x)[8], int gl, const float *w, const float *cos_t, const float *sin_t,
                                     int pos) {
    constexpr int kLanes = HD / 8;
    if (w) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = rms_inv(ss, 1.0f / HD);
        float nw[8];
        load_vec<HD, float>(w, gl, nw);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * (1.0f + nw[i]);
    }
    if (cos_t) {
        float c[4], s[4];
        load4<float>(cos_t + static_cast<int64_t>(pos) * (HD / 2) + 4 * gl, c);
        load4<float>(sin_t + static_cast<int64_t>(pos) * (HD / 2) + 4 * gl, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = x[i], b = x[4 + i];
            x[i] = a * c[i] - b * s[i];
            x[4 + i] = b * c[i] + a * s[i];
        }
    }
}
// The exponent of the smallest power of two s >= 2^-100 with amax <= 448 s, for finite amax >= 0 (as bits):
// 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
    const int e = static_cast<int>(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, -100);
}

// Blocks by rows: sequence b has the indices [q_start[b] / 16 + 2 b, q_start[b + 1] / 16 + 2 (b + 1)), at least as
// many as its q_len rows can touch.  Returns the sequence of `index` and its first index; -1 if none.
__device__ __forceinline__ int seq_of_block(const Batch &b, int index, int &base) {
    __shared__ int found;
    if (threadIdx.x == 0) found = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < b.batch; i += kThreads) {
        const int a = min(max(b.q_start[i], 0), b.total_q), e = min(max(b.q_start[i + 1], a), b.total_q);
        if (index >= a / kBlock + 2 * i && index < e / kBlock + 2 * (i + 1)) atomicMax(&found, i);
    }
    __syncthreads();
    const int i = found;
    if (i >= 0) base = min(max(b.q_start[i], 0), b.total_q) / kBlock + 2 * i;
    return i;
}

template <int HD, typename T, typename O>
__global__ void __launch_bounds__(kThreads) kv8_append_kernel(const AppendParams p) {
    constexpr int kLanes = HD / 8, kGroups = kThreads / kLanes, kPer = 2 * kBlock / kGroups;
    static_assert(kPer >= 1 && kPer * kGroups == 2 * kBlock, "32 K / V vectors over the groups");
    __shared__ uint32_t amax_s[2 * kBlock];  // K of tokens 0-15, V of tokens 0-15
    const int kvh = blockIdx.y, lane = threadIdx.x & 31;
    const int gi = threadIdx.x / kLanes, gl = threadIdx.x % kLanes;
    int si, j;
    if (p.blocks_per_seq > 0) {
        si = blockIdx.x / p.blocks_per_seq;
        j = blockIdx.x - si * p.blocks_per_seq;
    } else {
        int base = 0;
        si = seq_of_block(p.b, blockIdx.x, base);
        if (si < 0) return;
        j = blockIdx.x - base;
    }
    const Seq s = load_seq(p.b, si, j == 0 && kvh == 0 && threadIdx.x == 0);
    const int blk = max(s.pos0, 0) / kBlock + j;
    const int first = blk * kBlock;
    const int lo = max(max(s.pos0, 0), first), hi = min(s.pos0 + s.nq, first + kBlock);
    if (lo >= hi) return;
    // the block's place in the cache
    const int pt = first >> p.c.page_shift;
    const int page = p.b.table[si * p.b.table_stride + pt];
    const bool page_ok = page >= 0 && page < p.c.num_pages;
    if (!page_ok && threadIdx.x == 0) set_error(p.b.err, kErrPage);
    const int slot = first & ((1 << p.c.page_shift) - 1);
    const int64_t at = page * p.c.page_stride + kvh * p.c.head_stride + slot * p.c.token_stride;
    const int64_t sc = ((static_cast<int64_t>(page) * p.c.heads + kvh) << (p.c.page_shift - 4)) + slot / kBlock;
    const bool had = lo > first;  // the block holds earlier tokens
    float old_k = 0.f, old_v = 0.f;
    if (had && page_ok) {
        old_k = p.c.k_scale[sc];
        old_v = p.c.v_scale[sc];
    }
    const int64_t row0 = static_cast<int64_t>(s.q0) - s.pos0;  // row of a position

    // K and V vectors of the block: slot n = token n & 15 of K (n < 16) or V
    float x[kPer][8];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int n = i * kGroups + gi, pos = first + (n & 15);
        const bool on = pos >= lo && pos < hi;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
        if (on) {
            const int64_t row = row0 + pos;
            if (n < kBlock)
                load_vec<HD, T>(static_cast<const T *>(p.k) + row * p.k_row + kvh * p.k_head, gl, x[i]);
            else
                load_vec<HD, T>(static_cast<const T *>(p.v) + row * p.v_row + kvh * p.v_head, gl, x[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int n = i * kGroups + gi, pos = first + (n & 15);
        const bool on = pos >= lo && pos < hi;
        uint32_t most = 0;
        if (__any_sync(0xffffffffu, on)) {
            // a warp's vectors are all K or all V; absent tokens hold zeros and take a valid position
            if (n < kBlock) turn<HD>(x[i], gl, p.k_norm, p.cos_t, p.sin_t, on ? pos : lo);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                most = max(most, __float_as_uint(x[i][e]) & 0x7fffffffu);  // finite < infinity < NaN
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        if (gl == 0) amax_s[n] = on ? most : 0u;
    }
    // the q heads of the block's tokens, from the groups' other end: with one token they run beside its K and V
    const int nq = (hi - lo) * p.group;
    for (int n0 = 0; n0 < nq; n0 += kGroups) {
        const int n = n0 + kGroups - 1 - gi;
        const bool on = n < nq;
        const int pos = lo + (on ? n / p.group : 0), h = kvh * p.group + (on ? n % p.group : 0);
        const int64_t row = row0 + pos;
        float y[8];
        load_vec<HD, T>(static_cast<const T *>(p.q) + row * p.q_row + h * p.q_head, gl, y);
        turn<HD>(y, gl, p.q_norm, p.cos_t, p.sin_t, pos);
        if (on) {
            O *dst = static_cast<O *>(p.q_out) + row * p.out_row + h * p.out_head;
            store4(dst + 4 * gl, y);
            store4(dst + HD / 2 + 4 * gl, y + 4);
        }
    }
    __syncthreads();
    if (!page_ok) return;
    // lane n < 16: K of token n, lane 16 + n: V of it; a token with a non-finite vector counts for neither scale
    const uint32_t mine = amax_s[lane], other = __shfl_xor_sync(0xffffffffu, mine, 16);
    const bool bad = mine >= 0x7f800000u || other >= 0x7f800000u;
    const uint32_t bad_tokens = __ballot_sync(0xffffffffu, bad) & 0xffffu;
    uint32_t most = bad ? 0u : mine;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    float sk = __uint_as_float(static_cast<uint32_t>(scale_exponent(__shfl_sync(0xffffffffu, most, 0)) + 127) << 23);
    float sv = __uint_as_float(static_cast<uint32_t>(scale_exponent(__shfl_sync(0xffffffffu, most, 16)) + 127) << 23);
    if (had) {
        // earlier tokens of the block follow a scale that grows; K and V apart
        const float nk = fmaxf(sk, old_k), nv = fmaxf(sv, old_v);
        const int words = (lo - first) * (HD / 4);
        for (int w = threadIdx.x; w < 2 * words; w += kThreads) {
            const bool is_k = w < words;
            const int r = is_k ? w : w - words;
            const float ratio = is_k ? old_k / nk : old_v / nv;
            if (ratio == 1.0f) continue;
            uint32_t *cell = reinterpret_cast<uint32_t *>((is_k ? p.c.k : p.c.v) + at +
                                                          (r / (HD / 4)) * p.c.token_stride) + r % (HD / 4);
            uint32_t a, b;
            e4m3x4_to_h2x2(*cell, a, b);
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&a));
            const float2 g = __half22float2(*reinterpret_cast<const __half2 *>(&b));
            *cell = to_e4m3x4(f.x * ratio, f.y * ratio, g.x * ratio, g.y * ratio);
        }
        sk = nk;
        sv = nv;
    }
    if (threadIdx.x == 0) {
        p.c.k_scale[sc] = sk;
        p.c.v_scale[sc] = sv;
    }
    const float ik = 1.0f / sk, iv = 1.0f / sv;  // exact for the powers of two that this kernel writes
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int n = i * kGroups + gi, t = n & 15, pos = first + t;
        if (pos < lo || pos >= hi) continue;
        const float inv = n < kBlock ? ik : iv;
        uint32_t a = to_e4m3x4(x[i][0] * inv, x[i][1] * inv, x[i][2] * inv, x[i][3] * inv);
        uint32_t b = to_e4m3x4(x[i][4] * inv, x[i][5] * inv, x[i][6] * inv, x[i][7] * inv);
        if (bad_tokens >> t & 1u) a = b = n < kBlock ? 0x7f7f7f7fu : 0u;  // key NaN, value 0
        uint8_t *dst = (n < kBlock ? p.c.k : p.c.v) + at + t * p.c.token_stride;
        reinterpret_cast<uint32_t *>(dst)[gl] = a;
        reinterpret_cast<uint32_t *>(dst + HD / 2)[gl] = b;
    }
}

template <int HD, typename T, typename O>
cudaError_t launch(const AppendParams &p, dim3 grid, cudaStream_t s) {
    kv8_append_kernel<HD, T, O><<<grid, kThreads, 0, s>>>(p);
    return cudaGetLastError();
}
template <int HD>
cudaError_t launch_types(const AppendParams &p, dim3 grid, int in, int out, cudaStream_t s) {
    if (in == MG_BF16) return launch<HD, __nv_bfloat16, __nv_bfloat16>(p, grid, s);
    if (in == MG_F16) return launch<HD, __half, __half>(p, grid, s);
    if (out == MG_BF16) return launch<HD, float, __nv_bfloat16>(p, grid, s);
    if (out == MG_F16) return launch<HD, float, __half>(p, grid, s);
    return launch<HD, float, float>(p, grid, s);
}

bool known_type(int t) { return t == MG_F32 || t == MG_BF16 || t == MG_F16; }
}  // namespace

mg_status check_cache_batch(const char *who, const mg_kv8_cache *c, const mg_kv8_batch *b) {
    auto bad = [&](mg_status st, const char *what) {
        char buf[200];
        snprintf(buf, sizeof buf, "%s: %s", who, what);
        return report_error(st, buf);
    };
    if (!c || !b || c->struct_size != static_cast<int32_t>(sizeof *c) ||
        b->struct_size != static_cast<int32_t>(sizeof *b))
        return bad(MG_ERR_INVALID, "null argument or struct_size mismatch");
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return bad(MG_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256");
    if (c->page_size < kBlock || c->page_size > 256 || (c->page_size & (c->page_size - 1)) != 0)
        return bad(MG_ERR_UNSUPPORTED, "page_size must be a power of two in 16..256");
    if (c->num_pages <= 0 || c->num_kv_heads <= 0 || c->num_kv_heads > 65535)
        return bad(MG_ERR_INVALID, "need num_pages > 0 and num_kv_heads in 1..65535");
    if (!c->k_dev || !c->v_dev || !c->k_scale_dev || !c->v_scale_dev)
        return bad(MG_ERR_INVALID, "null cache pointer");
    if ((reinterpret_cast<uintptr_t>(c->k_dev) | reinterpret_cast<uintptr_t>(c->v_dev)) % 16 != 0 ||
        c->page_stride % 16 != 0 || c->head_stride % 16 != 0 || c->token_stride % 16 != 0)
        return bad(MG_ERR_INVALID, "cache data and strides must be multiples of 16 bytes");
    if (c->token_stride < c->head_dim || c->head_stride < c->head_dim || c->page_stride < c->head_dim)
        return bad(MG_ERR_INVALID, "cache strides must be at least head_dim bytes");
    if (b->batch <= 0 || b->total_q <= 0 || b->max_q <= 0 || b->max_ctx <= 0 || b->table_stride <= 0)
        return bad(MG_ERR_INVALID, "need batch, total_q, max_q, max_ctx and table_stride > 0");
    if (b->batch > (1 << 20) || b->total_q > (1 << 28) || b->max_q > (1 << 22) || b->max_ctx > (1 << 28))
        return bad(MG_ERR_UNSUPPORTED, "batch, total_q, max_q or max_ctx too large");
    if (b->max_ctx > b->table_stride * c->page_size)
        return bad(MG_ERR_INVALID, "max_ctx exceeds the page table (table_stride * page_size)");
    if (!b->q_start_dev || !b->ctx_len_dev || !b->page_table_dev || !b->err_dev)
        return bad(MG_ERR_INVALID, "null batch pointer");
    return MG_OK;
}

int log2_of(int n) {
    int s = 0;
    while ((1 << s) < n) ++s;
    return s;
}
Cache cache_of(const mg_kv8_cache *c) {
    return Cache{static_cast<uint8_t *>(c->k_dev), static_cast<uint8_t *>(c->v_dev), c->k_scale_dev, c->v_scale_dev,
                 c->page_stride, c->head_stride, c->token_stride, c->num_pages, log2_of(c->page_size),
                 c->num_kv_heads};
}
Batch batch_of(const mg_kv8_batch *b) {
    return Batch{b->q_start_dev, b->ctx_len_dev, b->page_table_dev, b->table_stride, b->err_dev,
                 b->batch, b->total_q, b->max_q, b->max_ctx};
}
}  // namespace kv8
}  // namespace mg

using namespace mg;

extern "C" mg_status mg_kv8_append(const mg_kv8_cache *cache, const mg_kv8_batch *batch,
                                   const mg_kv8_append_args *args, void *stream) {
    using namespace kv8;
    const mg_status st = check_cache_batch("mg_kv8_append", cache, batch);
    if (st != MG_OK) return st;
    if (!args || args->struct_size != static_cast<int32_t>(sizeof *args))
        return report_error(MG_ERR_INVALID, "mg_kv8_append: null argument or struct_size mismatch");
    if (!known_type(args->dtype) ||
        (args->num_heads > 0 && args->out_dtype != args->dtype &&
         !(args->dtype == MG_F32 && known_type(args->out_dtype))))
        return report_error(MG_ERR_UNSUPPORTED, "mg_kv8_append: dtype must be MG_F32, MG_BF16 or MG_F16, and out_dtype "
                                                "the same (for MG_F32 rows any of them)");
    if (!args->k_dev || !args->v_dev) return report_error(MG_ERR_INVALID, "mg_kv8_append: null k or v");
    if (args->num_heads < 0 || args->num_heads % cache->num_kv_heads != 0)
        return report_error(MG_ERR_INVALID, "mg_kv8_append: num_heads must be a multiple of num_kv_heads");
    if (args->num_heads > 0 && (!args->q_dev || !args->q_out_dev))
        return report_error(MG_ERR_INVALID, "mg_kv8_append: null q or q_out");
    if (!args->cos_dev != !args->sin_dev || (args->cos_dev && args->rope_len < batch->max_ctx))
        return report_error(MG_ERR_INVALID, "mg_kv8_append: need cos and sin with rope_len >= max_ctx, or neither");
    const uintptr_t in_align = args->dtype == MG_F32 ? 16 : 8, out_align = args->out_dtype == MG_F32 ? 16 : 8;
    uintptr_t in = reinterpret_cast<uintptr_t>(args->k_dev) | reinterpret_cast<uintptr_t>(args->v_dev);
    int64_t strides = args->k_row_stride | args->k_head_stride | args->v_row_stride | args->v_head_stride;
    uintptr_t out = 0, tables = reinterpret_cast<uintptr_t>(args->cos_dev) | reinterpret_cast<uintptr_t>(args->sin_dev) |
                                reinterpret_cast<uintptr_t>(args->k_norm_dev);
    if (args->num_heads > 0) {
        in |= reinterpret_cast<uintptr_t>(args->q_dev);
        out = reinterpret_cast<uintptr_t>(args->q_out_dev);
        tables |= reinterpret_cast<uintptr_t>(args->q_norm_dev);
        strides |= args->q_row_stride | args->q_head_stride | args->out_row_stride | args->out_head_stride;
    }
    if (in % in_align != 0 || out % out_align != 0 || strides % 4 != 0 || tables % 16 != 0)
        return report_error(MG_ERR_INVALID, "mg_kv8_append: rows must be aligned to 4 elements and their strides "
                                            "multiples of 4; norms and cos / sin aligned to 16 bytes");
    AppendParams p;
    p.c = cache_of(cache);
    p.b = batch_of(batch);
    p.q = args->q_dev, p.k = args->k_dev, p.v = args->v_dev, p.q_out = args->q_out_dev;
    p.q_row = args->q_row_stride, p.q_head = args->q_head_stride;
    p.k_row = args->k_row_stride, p.k_head = args->k_head_stride;
    p.v_row = args->v_row_stride, p.v_head = args->v_head_stride;
    p.out_row = args->out_row_stride, p.out_head = args->out_head_stride;
    p.q_norm = args->q_norm_dev, p.k_norm = args->k_norm_dev, p.cos_t = args->cos_dev, p.sin_t = args->sin_dev;
    p.group = args->num_heads / cache->num_kv_heads;
    // a sequence of max_q rows touches at most (max_q + 14) / 16 + 1 blocks
    const int64_t per_seq = (batch->max_q + kBlock - 2) / kBlock + 1;
    const int64_t by_rows = batch->total_q / kBlock + 2 * static_cast<int64_t>(batch->batch);
    p.blocks_per_seq = per_seq * batch->batch <= by_rows ? static_cast<int>(per_seq) : 0;
    const dim3 grid(static_cast<unsigned>(p.blocks_per_seq ? per_seq * batch->batch : by_rows), cache->num_kv_heads);
    cudaError_t e;
    if (cache->head_dim == 64) e = launch_types<64>(p, grid, args->dtype, args->out_dtype, static_cast<cudaStream_t>(stream));
    else if (cache->head_dim == 128) e = launch_types<128>(p, grid, args->dtype, args->out_dtype, static_cast<cudaStream_t>(stream));
    else e = launch_types<256>(p, grid, args->dtype, args->out_dtype, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) {
        char buf[160];
        snprintf(buf, sizeof buf, "mg_kv8_append: %s", cudaGetErrorString(e));
        return report_error(MG_ERR_CUDA, buf);
    }
    return MG_OK;
}
