// kv8_append.cu -- mg_kv8_append: new keys and values into the 8-bit paged
// cache, with the head norm and the position rotation on the way (the QK-norm,
// RoPE and cache write of layers.mojo:43-61), and the rotated queries.
//
// A block's scale is a maximum over its tokens, so the tokens of a call that
// fall into one block of 16 positions of a sequence and kv head, the block's
// earlier codes and its scale all belong to one owner, and the q heads of the
// same tokens and kv head go along (they share the cos / sin rows).  A head
// vector is held by head_dim / 8 lanes (a group), lane i with elements 4 i ..
// 4 i + 3 of each half, so that a rotation's pairs meet in one lane and loads
// are 4 elements wide.  Two forms:
//  * max_q 1 (a decode step): the owner is a group; nothing crosses groups;
//  * otherwise the owner is a CTA of 16 groups, one per token of the block.
//
// The work is memory traffic: the rows in, the rotated queries and one byte
// per value out; per element a norm and a rotation are a few operations.  What
// it costs is latency, so a token's K, V, q heads, cos and sin rows are all
// loaded before the first is used, and the page id and old scales, which only
// the stores need, are not waited for earlier.
//
// Measured (launches in a graph; a plain copy on this GPU reaches 6.46 TB/s):
// one token of 4 q and 1 kv heads of 256, 3.5 us, bound by the launch (4.8 in
// the block form); 128 tokens of 32 and 16 heads of 128 in fp16, 3.8 us (12.6
// in the block form); 5451 fp32 prompt tokens of 8 and 4 heads of 256, 31 us,
// 4.2 TB/s; one prompt of 16384 bf16 tokens of 32 and 16 heads of 128, 96 us,
// 5.0 TB/s (43 and 133 us while a token's rows were loaded one after another).
// Call by call, without a graph, 4.0 us for either decode step and 99 to 101 us
// (4.8 TB/s) for the long prompt.  The block form spills a little at 64 registers
// (fp32 32 bytes, fp16 8); with room for them an SM holds fewer CTAs.
#include "kv8.cuh"

#include <cstdio>
#include <type_traits>

namespace mg {
namespace kv8 {
namespace {

constexpr int kTokenThreads = 128;  // CTA of the one-token form

struct AppendParams {
    Cache c;
    Batch b;
    const void *q, *k, *v;
    void *q_out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
    const float *q_norm, *k_norm, *cos_t, *sin_t;
    int group;            // q heads per kv head (0: no queries)
    int blocks_per_seq;   // block form: > 0: block index = sequence * this + block; 0: by rows, seq_of_block
};

// Four elements as they lie in memory, and as floats.
template <typename T>
using Raw = typename std::conditional<sizeof(T) == 4, float4, uint2>::type;
template <typename T>
__device__ __forceinline__ void widen(const Raw<T> &v, float *x) {
    if constexpr (std::is_same<T, float>::value) {
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else if constexpr (std::is_same<T, __half>::value) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    } else {
        x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
        x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
    }
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
struct Vec {
    Raw<T> a, b;
    __device__ __forceinline__ void load(const T *p, int gl) {
        a = *reinterpret_cast<const Raw<T> *>(p + 4 * gl);
        b = *reinterpret_cast<const Raw<T> *>(p + HD / 2 + 4 * gl);
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
        widen<T>(a, x);
        widen<T>(b, x + 4);
    }
};
template <int HD>
__device__ __forceinline__ void load_weights(const float *w, int gl, float (&x)[8]) {
    Vec<HD, float> v;
    v.load(w, gl);
    v.floats(x);
}
__device__ __forceinline__ void rotate(float (&x)[8], const float4 &c, const float4 &s) {
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = x[i], b = x[4 + i];
        x[i] = a * cc[i] - b * ss[i];
        x[4 + i] = b * cc[i] + a * ss[i];
    }
}
template <int HD>
__device__ __forceinline__ void norm(float (&x)[8], const float (&w)[8]) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
    for (int o = HD / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rms_inv(ss, 1.0f / HD);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * (1.0f + w[i]);
}
// The same for a key, whose values are about to be rounded to 4 bits: the sum and the factor in 64 bits, so that what
// is left of its error (four roundings to 32 bits) moves hardly more values across a border than one rounding would: 10
// of 5.6 million codes, against 4 with the product and the rotation in 64 bits too, which takes 6 % longer.
template <int HD>
__device__ __forceinline__ void norm_key(float (&x)[8], const float (&w)[8]) {
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += static_cast<double>(x[i]) * static_cast<double>(x[i]);
#pragma unroll
    for (int o = HD / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const double m = ss * (1.0 / HD) + 1e-6;
    double inv = static_cast<double>(rsqrtf(static_cast<float>(m)));
    inv = inv * (1.5 - 0.5 * m * inv * inv);  // one Newton step from 2^-22 to 2^-44
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= static_cast<float>(inv * (1.0 + static_cast<double>(w[i])));
}
// The largest magnitude of a group's vector, as bits: finite < infinity < NaN.
template <int HD>
__device__ __forceinline__ uint32_t most_of(const float (&x)[8]) {
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
    if constexpr (HD == 256) {  // a group is a warp: one instruction (5451 fp32 prompt tokens: 32 us -> 31)
        return __reduce_max_sync(0xffffffffu, most);
    } else {
#pragma unroll
        for (int o = HD / 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        return most;
    }
}
// Eight codes of the lane at a token's row; `fill`: instead of them.
template <int HD>
__device__ __forceinline__ void store_codes(uint8_t *row, int gl, const float (&x)[8], float inv, bool bad, uint32_t fill) {
    const uint32_t a = to_e4m3x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    const uint32_t b = to_e4m3x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
    reinterpret_cast<uint32_t *>(row)[gl] = bad ? fill : a;
    reinterpret_cast<uint32_t *>(row + HD / 2)[gl] = bad ? fill : b;
}
// Four codes under a scale that grew: ratio = old / new.
__device__ __forceinline__ uint32_t requantise(uint32_t four, float ratio) {
    uint32_t a, b;
    e4m3x4_to_h2x2(four, a, b);
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&a));
    const float2 g = __half22float2(*reinterpret_cast<const __half2 *>(&b));
    return to_e4m3x4(f.x * ratio, f.y * ratio, g.x * ratio, g.y * ratio);
}
// The exponent of the smallest power of two s >= 2^-100 with amax <= 448 s, for finite amax >= 0 (as bits):
// 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
    const int e = static_cast<int>(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, -100);
}
__device__ __forceinline__ float scale_of(uint32_t amax_bits) {
    return __uint_as_float(static_cast<uint32_t>(scale_exponent(amax_bits) + 127) << 23);
}
constexpr uint32_t kInfBits = 0x7f800000u;
constexpr uint32_t kBadKey = 0x7f7f7f7fu;  // four e4m3 NaNs: the key of a token with a non-finite key or value

// Where a block lies: byte offset of its first token, index of its scales.
struct Spot {
    int64_t at, scale;
};
__device__ __forceinline__ Spot spot_of(const Cache &c, int page, int kvh, int first) {
    const int slot = first & ((1 << c.page_shift) - 1);
    return Spot{page * c.page_stride + kvh * c.head_stride + slot * c.token_stride,
                 ((static_cast<int64_t>(page) * c.heads + kvh) << (c.page_shift - 4)) + slot / kBlock};
}

// One token's vectors of a group: loaded together, then worked off.
template <int HD, int kQ, typename T, typename O>  // kQ: q heads in flight
struct Token {
    Vec<HD, T> k, v, q[kQ];
    float4 c, s;
    const T *qp;
    O *op;
    int64_t q_head, out_head;
    int group;
    __device__ __forceinline__ void load(const AppendParams &p, int64_t row, int pos, int kvh, int gl) {
        k.load(static_cast<const T *>(p.k) + row * p.k_row + kvh * p.k_head, gl);
        v.load(static_cast<const T *>(p.v) + row * p.v_row + kvh * p.v_head, gl);
        group = p.group;
        q_head = p.q_head, out_head = p.out_head;
        qp = static_cast<const T *>(p.q) + row * p.q_row + static_cast<int64_t>(kvh) * group * q_head;
        op = static_cast<O *>(p.q_out) + row * p.out_row + static_cast<int64_t>(kvh) * group * out_head;
#pragma unroll
        for (int i = 0; i < kQ; ++i)
            if (i < group) q[i].load(qp + i * q_head, gl);
        c = s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p.cos_t) {
            c = *reinterpret_cast<const float4 *>(p.cos_t + static_cast<int64_t>(pos) * (HD / 2) + 4 * gl);
            s = *reinterpret_cast<const float4 *>(p.sin_t + static_cast<int64_t>(pos) * (HD / 2) + 4 * gl);
        }
    }
    __device__ __forceinline__ void key(const AppendParams &p, int gl, float (&x)[8]) const {
        k.floats(x);
        if (p.k_norm) {
            float w[8];
            load_weights<HD>(p.k_norm, gl, w);
            norm_key<HD>(x, w);
        }
        if (p.cos_t) rotate(x, c, s);
    }
    // All lanes of the warp take part; `on`: of this group's token.
    __device__ __forceinline__ void queries(const AppendParams &p, int gl, bool on) {
        float w[8];
        if (p.q_norm) load_weights<HD>(p.q_norm, gl, w);
        for (int h0 = 0; h0 < group; h0 += kQ) {
#pragma unroll
            for (int i = 0; i < kQ; ++i) {
                if (h0 + i >= group) break;
                float x[8];
                q[i].floats(x);
                if (p.q_norm) norm<HD>(x, w);
                if (p.cos_t) rotate(x, c, s);
                if (on) {
                    store4(op + (h0 + i) * out_head + 4 * gl, x);
                    store4(op + (h0 + i) * out_head + HD / 2 + 4 * gl, x + 4);
                }
            }
#pragma unroll
            for (int i = 0; i < kQ; ++i)
                if (h0 + kQ + i < group) q[i].load(qp + (h0 + kQ + i) * q_head, gl);
        }
    }
};

// max_q 1: a group per (sequence, kv head).
template <int HD, typename T, typename O>
__global__ void __launch_bounds__(kTokenThreads) kv8_append_token_kernel(const AppendParams p) {
    constexpr int kLanes = HD / 8, kGroups = kTokenThreads / kLanes;
    kernel_begins();
    const int gl = threadIdx.x % kLanes;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / kLanes;
    const int si = min(static_cast<int>(item / p.c.heads), p.b.batch - 1), kvh = static_cast<int>(item % p.c.heads);
    const Seq s = load_seq(p.b, si, kvh == 0 && gl == 0);
    const int pos = s.pos0;
    const bool on = item < static_cast<int64_t>(p.b.batch) * p.c.heads && s.nq == 1 && pos >= 0;
    if (!__any_sync(0xffffffffu, on)) return;
    constexpr int kQ = 4;
    Token<HD, kQ, T, O> tk;
    int page = -1;
    if (on) {
        page = p.b.table[si * p.b.table_stride + (pos >> p.c.page_shift)];
        tk.load(p, s.q0, pos, kvh, gl);
    } else {
        tk.group = p.group;  // the warp's other groups run along with what the registers hold
        tk.k = tk.v = Vec<HD, T>{};
        tk.c = tk.s = make_float4(0.f, 0.f, 0.f, 0.f);
        tk.qp = static_cast<const T *>(p.q);
        tk.q_head = 0;
#pragma unroll
        for (int i = 0; i < kQ; ++i) tk.q[i] = Vec<HD, T>{};
    }
    float k[8], v[8];
    tk.key(p, gl, k);
    tk.v.floats(v);
    const uint32_t mk = most_of<HD>(k), mv = most_of<HD>(v);
    tk.queries(p, gl, on);
    if (!on) return;
    if (page < 0 || page >= p.c.num_pages) {
        if (gl == 0) set_error(p.b.err, kErrPage);
        return;
    }
    const int t = pos % kBlock;
    const Spot pl = spot_of(p.c, page, kvh, pos - t);
    const bool bad = mk >= kInfBits || mv >= kInfBits;
    float sk = scale_of(bad ? 0u : mk), sv = scale_of(bad ? 0u : mv);
    uint8_t *kb = p.c.k + pl.at, *vb = p.c.v + pl.at;
    if (t > 0) {  // the block's earlier tokens follow a scale that grows
        const float ok = p.c.k_scale[pl.scale], ov = p.c.v_scale[pl.scale];
        sk = fmaxf(sk, ok);
        sv = fmaxf(sv, ov);
        const float rk = ok / sk, rv = ov / sv;
        if (rk != 1.0f || rv != 1.0f) {
#pragma unroll 4
            for (int i = 0; i < 4 * t; ++i) {  // K, then V of a token's two halves
                uint8_t *row = (i & 1 ? vb : kb) + (i >> 2) * p.c.token_stride + (i & 2 ? HD / 2 : 0);
                const uint32_t old = reinterpret_cast<uint32_t *>(row)[gl];
                reinterpret_cast<uint32_t *>(row)[gl] = requantise(old, i & 1 ? rv : rk);
            }
        }
    }
    store_codes<HD>(kb + t * p.c.token_stride, gl, k, 1.0f / sk, bad, kBadKey);
    store_codes<HD>(vb + t * p.c.token_stride, gl, v, 1.0f / sv, bad, 0u);
    const uint32_t lanes = static_cast<uint32_t>((1ull << kLanes) - 1) << (threadIdx.x % 32 / kLanes * kLanes);
    __syncwarp(lanes);  // every lane of the group has read the old scales
    if (gl == 0) {
        p.c.k_scale[pl.scale] = sk;
        p.c.v_scale[pl.scale] = sv;
    }
}

// Blocks by rows: sequence b has the indices [q_start[b] / 16 + 2 b, q_start[b + 1] / 16 + 2 (b + 1)), at least as
// many as its q_len rows can touch.  Returns the sequence of `index` and its first index; -1 if none.
__device__ __forceinline__ int seq_of_block(const Batch &b, int index, int &base) {
    __shared__ int found;
    if (threadIdx.x == 0) found = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < b.batch; i += blockDim.x) {
        if (index == 0) load_seq(b, i, true);  // starts that fall back may leave their sequence no index to be seen at
        const int a = min(max(b.q_start[i], 0), b.total_q), e = min(max(b.q_start[i + 1], a), b.total_q);
        if (index >= a / kBlock + 2 * i && index < e / kBlock + 2 * (i + 1)) atomicMax(&found, i);
    }
    __syncthreads();
    const int i = found;
    if (i >= 0) base = min(max(b.q_start[i], 0), b.total_q) / kBlock + 2 * i;
    return i;
}

// A CTA of 16 groups per (sequence, block, kv head).
template <int HD, typename T, typename O>
__global__ void __launch_bounds__(2 * HD, 512 / HD) kv8_append_block_kernel(const AppendParams p) {
    constexpr int kLanes = HD / 8, kThreads = kBlock * kLanes;
    __shared__ uint32_t amax_s[2 * kBlock];  // K of tokens 0-15, V of tokens 0-15
    kernel_begins();
    const int kvh = blockIdx.y, lane = threadIdx.x & 31;
    const int t = threadIdx.x / kLanes, gl = threadIdx.x % kLanes;
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
    const int first = (max(s.pos0, 0) / kBlock + j) * kBlock;
    const int lo = max(max(s.pos0, 0), first), hi = min(s.pos0 + s.nq, first + kBlock);
    if (lo >= hi) return;
    const int page = p.b.table[si * p.b.table_stride + (first >> p.c.page_shift)];
    const int pos = first + t;
    const bool on = pos >= lo && pos < hi;
    Token<HD, 2, T, O> tk;  // 64 registers: twice the CTAs of 4 heads in flight
    // a group without a token runs along with the block's first new one
    const int at_pos = on ? pos : lo;
    tk.load(p, static_cast<int64_t>(s.q0) + at_pos - s.pos0, at_pos, kvh, gl);
    float k[8], v[8];
    tk.key(p, gl, k);
    tk.v.floats(v);
    const uint32_t mk = most_of<HD>(k), mv = most_of<HD>(v);
    if (gl == 0) {
        amax_s[t] = on ? mk : 0u;
        amax_s[kBlock + t] = on ? mv : 0u;
    }
    tk.queries(p, gl, on);
    __syncthreads();
    if (page < 0 || page >= p.c.num_pages) {
        if (threadIdx.x == 0) set_error(p.b.err, kErrPage);
        return;
    }
    const Spot pl = spot_of(p.c, page, kvh, first);
    // lane n < 16: K of token n, lane 16 + n: V of it; a token with a non-finite vector counts for neither scale
    const uint32_t mine = amax_s[lane], other = __shfl_xor_sync(0xffffffffu, mine, 16);
    const bool bad = mine >= kInfBits || other >= kInfBits;
    const uint32_t bad_tokens = __ballot_sync(0xffffffffu, bad) & 0xffffu;
    uint32_t most = bad ? 0u : mine;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    float sk = scale_of(__shfl_sync(0xffffffffu, most, 0)), sv = scale_of(__shfl_sync(0xffffffffu, most, 16));
    uint8_t *kb = p.c.k + pl.at, *vb = p.c.v + pl.at;
    if (lo > first) {  // the block's earlier tokens follow a scale that grows
        const float ok = p.c.k_scale[pl.scale], ov = p.c.v_scale[pl.scale];
        __syncthreads();  // every thread has read the old scales
        sk = fmaxf(sk, ok);
        sv = fmaxf(sv, ov);
        const int words = (lo - first) * (HD / 4);
        for (int w = threadIdx.x; w < 2 * words; w += kThreads) {
            const bool is_k = w < words;
            const int r = is_k ? w : w - words;
            const float ratio = is_k ? ok / sk : ov / sv;
            if (ratio == 1.0f) continue;
            uint32_t *cell = reinterpret_cast<uint32_t *>((is_k ? kb : vb) + (r / (HD / 4)) * p.c.token_stride) + r % (HD / 4);
            *cell = requantise(*cell, ratio);
        }
    }
    if (threadIdx.x == 0) {
        p.c.k_scale[pl.scale] = sk;
        p.c.v_scale[pl.scale] = sv;
    }
    if (!on) return;
    store_codes<HD>(kb + t * p.c.token_stride, gl, k, 1.0f / sk, bad_tokens >> t & 1u, kBadKey);
    store_codes<HD>(vb + t * p.c.token_stride, gl, v, 1.0f / sv, bad_tokens >> t & 1u, 0u);
}

template <int HD, typename T, typename O>
cudaError_t launch(const AppendParams &p, dim3 grid, cudaStream_t s) {
    if (p.b.max_q > 1) return launch_behind(kv8_append_block_kernel<HD, T, O>, grid, 2 * HD, 0, s, p);
    constexpr int kGroups = kTokenThreads / (HD / 8);
    const int64_t items = static_cast<int64_t>(p.b.batch) * p.c.heads;
    return launch_behind(kv8_append_token_kernel<HD, T, O>, dim3(static_cast<unsigned>((items + kGroups - 1) / kGroups)),
                         kTokenThreads, 0, s, p);
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
    if (b->table_width < 0) return bad(MG_ERR_INVALID, "need table_width >= 0");
    if (b->max_ctx > (b->table_width > 0 ? b->table_width : b->table_stride) * c->page_size)
        return bad(MG_ERR_INVALID, "max_ctx exceeds the page table (its width * page_size)");
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
    if (args->num_heads > 0 && args->q_out_dev == args->q_dev &&
        (args->out_dtype != args->dtype || args->out_row_stride != args->q_row_stride ||
         args->out_head_stride != args->q_head_stride))
        return report_error(MG_ERR_INVALID, "mg_kv8_append: q_out may be q only with its dtype and strides");
    // the one-token form: a group of head_dim / 8 lanes per sequence and kv head
    if (batch->max_q == 1 &&
        static_cast<int64_t>(batch->batch) * cache->num_kv_heads > INT32_MAX * static_cast<int64_t>(kTokenThreads / (cache->head_dim / 8)))
        return report_error(MG_ERR_UNSUPPORTED, "mg_kv8_append: batch * num_kv_heads too large");
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
