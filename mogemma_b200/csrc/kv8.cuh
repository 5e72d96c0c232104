// kv8.cuh -- the 8-bit paged key/value cache: what its append (kv8_append.cu)
// and its attention (kv8_attention.cu, kv8_prompt.cu) share.  Kernel
// parameters, e4m3 conversions, and the schedule that cuts the attention's
// work into equal shares.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/mogemma_b200.h"
#include "common.cuh"

namespace mg {
mg_status report_error(mg_status st, const char *msg);

namespace kv8 {

constexpr int kBlock = MG_KV8_BLOCK;  // tokens per scale
constexpr uint32_t kErrLens = MG_KV8_ERR_LENGTHS, kErrPage = MG_KV8_ERR_PAGE, kErrWait = MG_KV8_ERR_WAIT;

// The cache and the batch as the kernels see them.
struct Cache {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    int64_t page_stride, head_stride, token_stride;
    int num_pages, page_shift, heads;  // page_size = 1 << page_shift
};
struct Batch {
    const int32_t *q_start, *ctx_len, *table;
    int64_t table_stride;
    uint32_t *err;
    int batch, total_q, max_q, max_ctx;
};

// One sequence, with the device's lengths forced into the host's bounds: rows
// [q0, q0 + nq) at positions pos0 .. pos0 + nq - 1, of which those in
// [0, max_ctx) exist.
struct Seq {
    int q0, nq, pos0;
};
__device__ __forceinline__ Seq load_seq(const Batch &b, int i, bool report) {
    const int a = b.q_start[i], e = b.q_start[i + 1], ctx = b.ctx_len[i];
    Seq s;
    s.q0 = min(max(a, 0), b.total_q);
    s.nq = min(min(max(e, s.q0), b.total_q) - s.q0, b.max_q);
    // a length that breaks the bounds hides the whole sequence: positions below 0
    const bool bad = a < 0 || e < a || e > b.total_q || e - a > b.max_q || ctx < e - a || ctx > b.max_ctx;
    if (bad && report) set_error(b.err, kErrLens);
    s.pos0 = bad ? -s.nq : ctx - s.nq;
    return s;
}

// ---- launches.  A kernel is launched so that it may be set up while its
// predecessor on the stream ends (programmatic dependent launch), and waits for
// the predecessor's results itself, before its first access to memory.  No
// kernel lets its successor begin before it ends: a combine whose blocks came
// early cost the attention 1 to 2 us.
__device__ __forceinline__ void kernel_begins() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename... P, typename... A>
cudaError_t launch_behind(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// ---- e4m3 <-> wider.  Codes convert to fp16 exactly (448 and 2^-9 are both in its range).
// A word's codes 0, 1 and codes 2, 3.
__device__ __forceinline__ void e4m3x4_to_h2x2(uint32_t four, uint32_t &a, uint32_t &b) {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(a), "=r"(b)
        : "r"(four));
}
// Four floats to codes (nearest even, beyond 448 to 448, NaN to NaN), a in the lowest byte.
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}

__device__ __forceinline__ float ex2(float x) {  // PTX ex2.approx: one MUFU op, about 2 ulp
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float kInf = __builtin_huge_valf();
__device__ __forceinline__ float finite_or_0(float x) { return x == -kInf ? 0.f : x; }

// ---- query rows.  Two values of type T in a word, as floats and back.
template <typename T>
__device__ __forceinline__ float2 two(uint32_t w);
template <>
__device__ __forceinline__ float2 two<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 two<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
__device__ __forceinline__ uint32_t pack(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// The power of two that brings a row's largest magnitude (as bits) to [2^15, 2^16), fp16's last binade, and its inverse:
// fp16 rows then stay as they are, bf16 values exact down to 2^-32 of the largest.  A row with an infinity or NaN gets
// NaN for the inverse and answers NaN.
__device__ __forceinline__ void row_scale(uint32_t most, float &up, float &down) {
    const int e = static_cast<int>(most >> 23);
    up = down = 1.0f;
    if (e >= 255) {
        down = __int_as_float(0x7fc00000);
    } else if (most > 0) {  // bf16 subnormals too: e is 0
        const int sh = min(142 - e, 126);  // exponent of `up`; |sh| <= 126 keeps both normal
        up = __uint_as_float(static_cast<uint32_t>(127 + sh) << 23);
        down = __uint_as_float(static_cast<uint32_t>(127 - sh) << 23);
    }
}

// ---- the attention's schedule
// An item is (sequence, tile of ROWS query rows, kv head): the rows of a
// sequence and kv head are its (token, q head of the group) pairs, token major.
// Its cost is the number of units of 64 or 128 tokens its rows see, at least
// one (rows that see nothing still have an answer to write), plus a constant
// for its start and end that counts as units before the first.  Items are laid out head by
// head, sequence by sequence; CTA c of G takes the units [c W / G, (c+1) W / G)
// of all W, so the shares differ by one unit at most, whatever the lengths
// (with fewer units than CTAs, the first W CTAs take one each).
// Every CTA finds its place by the same scan over the items.
struct AttnShape {
    int group, rows, tiles, window;  // q heads per kv head; rows per tile; tiles per sequence (of max_q tokens)
    int unit, extra;                 // tokens of a unit of the schedule; cost of an item beside its units
};
struct Item {
    Seq seq;
    int row0, nrows;     // rows of the tile
    int lo, hi;          // positions its rows see lie in [lo, hi)
    int unit0, units;    // units unit0 .. unit0 + units - 1
    int cost;            // extra + units; 0: no rows
    // The pair to go on to: behind a tile without rows its sequence has no more.  (max_q may be far above most lengths:
    // one visit per tile kept the prompt kernel's roles waiting for the next item, 4 million tiles beyond 20 ms.)
    int after;
};
__device__ __forceinline__ Item load_item(const Batch &b, const AttnShape &a, int pair, bool report) {
    Item it;
    const int i = pair / a.tiles, t = pair - i * a.tiles;
    it.seq = load_seq(b, i, report);
    it.row0 = t * a.rows;
    it.nrows = min(a.rows, it.seq.nq * a.group - it.row0);
    it.units = it.cost = 0;
    it.after = it.nrows > 0 ? pair + 1 : (i + 1) * a.tiles;
    if (it.nrows <= 0) return it;
    const int first = it.seq.pos0 + it.row0 / a.group, last = it.seq.pos0 + (it.row0 + it.nrows - 1) / a.group;
    it.lo = a.window > 0 ? max(0, first - a.window + 1) : 0;
    it.hi = max(last + 1, it.lo);
    it.unit0 = it.lo / a.unit;
    it.units = max(1, (it.hi + a.unit - 1) / a.unit - it.unit0);
    it.cost = it.units + a.extra;
    return it;
}

// Where CTA `cta` of `ctas` starts: its range [w0, w1) of the whole cost, and
// the item (head, pair) and the place within it of w0.  All threads of the CTA
// call it; THREADS a multiple of 32.
struct Place {
    int64_t total;  // cost of all heads
    int64_t w0, w1;
    int ctas;  // CTAs that have a share
    int head, pair, skip;
};
template <int THREADS>
__device__ __forceinline__ Place find_place(const Batch &b, const AttnShape &a, int heads, int cta, int ctas) {
    constexpr int kWarps = THREADS / 32;
    __shared__ int64_t warp_sum_s[kWarps];
    __shared__ int found_pair, found_skip;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int pairs = b.batch * a.tiles, chunk = (pairs + THREADS - 1) / THREADS;
    const int p0 = min(pairs, tid * chunk), p1 = min(pairs, p0 + chunk);
    int64_t mine = 0;
    for (int p = p0; p < p1;) {
        const Item it = load_item(b, a, p, cta == 0);
        mine += it.cost;
        p = it.after;
    }
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t n = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += n;
    }
    if (lane == 31) warp_sum_s[warp] = upto;
    if (tid == 0) found_pair = found_skip = 0;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) upto += warp_sum_s[w];
        all += warp_sum_s[w];
    }
    Place pl;
    pl.total = all * heads;
    pl.ctas = static_cast<int>(min(pl.total, static_cast<int64_t>(ctas)));
    pl.w0 = cta < pl.ctas ? pl.total * cta / pl.ctas : 0;
    pl.w1 = cta < pl.ctas ? pl.total * (cta + 1) / pl.ctas : 0;
    pl.head = all > 0 ? static_cast<int>(pl.w0 / all) : 0;
    const int64_t in_head = pl.w0 - pl.head * all;
    if (mine > 0 && upto - mine <= in_head && in_head < upto) {
        int64_t left = in_head - (upto - mine);
        int p = p0;
        for (;;) {
            const Item it = load_item(b, a, p, false);
            const int next = it.after;
            if (left < it.cost || next >= p1) break;
            left -= it.cost;
            p = next;
        }
        found_pair = p;
        found_skip = static_cast<int>(left);
    }
    __syncthreads();
    pl.pair = found_pair;
    pl.skip = found_skip;
    return pl;
}
// The CTA that holds place w of the whole.
__device__ __forceinline__ int owner_of(const Place &pl, int64_t w) {
    return static_cast<int>(((w + 1) * pl.ctas - 1) / pl.total);
}

// The CTA's share, item by item: of the item's units, first .. first + take - 1.
struct Walk {
    int64_t w, w1;
    int head, pair, skip;  // skip: places of the current item before w
    int first, take;
    Item it;
    // The current item, or the next one of which the CTA has a unit; false at the end of the share.
    __device__ __forceinline__ bool settle(const Batch &b, const AttnShape &a) {
        while (w < w1) {
            it = load_item(b, a, pair, false);
            const int64_t end = min(static_cast<int64_t>(it.cost), skip + (w1 - w));
            first = max(0, skip - a.extra);
            take = max(0, static_cast<int>(end) - a.extra) - first;
            if (it.cost > 0 && take > 0) return true;
            step(b, a);
        }
        return false;
    }
    __device__ __forceinline__ void step(const Batch &b, const AttnShape &a) {
        w += it.cost > 0 ? it.cost - skip : 0;
        skip = 0;
        pair = it.after;
        if (pair >= b.batch * a.tiles) pair = 0, ++head;
    }
    __device__ __forceinline__ bool start(const Batch &b, const AttnShape &a, const Place &pl) {
        w = pl.w0, w1 = pl.w1, head = pl.head, pair = pl.pair, skip = pl.skip;
        return settle(b, a);
    }
    __device__ __forceinline__ bool next(const Batch &b, const AttnShape &a) {
        step(b, a);
        return settle(b, a);
    }
    __device__ __forceinline__ bool whole() const { return take == it.units; }
    // The item's units after this CTA's are others': the CTA of the last one.
    __device__ __forceinline__ int last_cta(const Place &pl) const { return owner_of(pl, w - skip + it.cost - 1); }
    // The partial answer's slot: a part with the item's first unit, or a later one; a CTA has one of each at most.
    __device__ __forceinline__ int slot(int cta) const { return 2 * cta + (first == 0 ? 1 : 0); }
};

// Items of which several CTAs have a part: the CTA with the first unit names it
// in split[c], for the combine; the others are the CTAs up to last_cta.
struct Split {
    int pair, head, nrows;  // nrows 0: no such item
    int last_cta;
};
struct Partials {
    Split *split;  // [ctas]
    float *ml;     // [2 ctas][rows][2]: running maximum (log2 units) and sum
    float *o;      // [2 ctas][rows][head dim], divided by the sum
};
inline size_t partials_bytes(int ctas, int rows, int hd) {
    return static_cast<size_t>(ctas) * (sizeof(Split) + 2 * static_cast<size_t>(rows) * (hd + 2) * sizeof(float));
}
inline Partials partials_at(void *ws, int ctas, int rows) {
    Partials p;
    p.split = static_cast<Split *>(ws);
    p.ml = reinterpret_cast<float *>(p.split + ctas);
    p.o = p.ml + 4 * static_cast<size_t>(ctas) * rows;
    return p;
}

struct AttnArgs {
    Cache c;
    Batch b;
    AttnShape a;
    Partials part;
    const void *q;
    void *out;
    int64_t q_row, q_head, out_row, out_head;
    float scale_log2;  // scale * log2(e)
    uint64_t wait_ns;  // budget of a wait inside the prompt kernel
    int stall;         // mg_kv8_set_debug: the hand-off that CTA 0 withholds; -1: none
};
// Hand-offs of the prompt kernel, as mg_kv8_set_debug counts them.
enum Handoff : int {
    kItemFull, kItemEmpty, kKFull, kKEmpty, kVFull, kVEmpty, kQFull, kSFull, kPFull, kPvDone, kScales, kPair, kDrained,
    kHandoffs
};
}  // namespace kv8
}  // namespace mg
