// kv8_prompt.cu -- mg_kv8_attention for many query rows per kv head (prompts,
// prompt chunks, drafts of several tokens): the 5th-generation tensor cores on
// the 8-bit paged cache.
//
// An item's query rows ((token, q head of the group) pairs of one kv head) are
// one or two tiles of 128 (two for head dims 64 and 128, which then share every
// widened key and value); its keys run in units of 64 tokens.  Both products
// are tcgen05.mma kind::f16 with fp32 accumulators in TMEM:
//   S [128 x 64] = Q . K^T        Q and K fp16 in shared memory, K-major
//   O [128 x hd] += P . V         P fp16 in TMEM (over S), V fp16 MN-major
// The cache's codes are widened to fp16, which is exact, on their way into
// shared memory; q is brought into fp16's range by a power of two per row.  The
// block scales of K multiply the score columns, those of V ride in P's
// exponent: with s = scale log2(e) k_scale <q, k>, m = max s and
// M = max(s + log2 v_scale), P = 2^(s + log2 v_scale - M) and l = sum 2^(s - m),
// so P is bounded whatever the scales and fp16 holds it to 2^-12.
//
// Warps of a CTA (640 threads, one CTA per SM):
//  * warps 0-7: softmax.  Two row tiles: warpgroup g has tile g, a row per
//    thread (TMEM lane = row).  One row tile (hd 256): warpgroup g has columns
//    32 g .. 32 g + 31 of every row, and the two threads of a row exchange their
//    maxima.  They also bring the item's Q into shared memory and write the
//    answers;
//  * warps 8-11 load K, 12-15 V: codes from the pages into registers one or two units
//    ahead (page ids one further), widened and stored in the 128-byte swizzled
//    layout (token rows of 64 dims); tokens that no row sees become zeros, so
//    that stale codes behind the context cannot reach a product;
//  * warp 16: allocates TMEM; one lane issues the MMAs: S of unit j + 1 before
//    P V of unit j, so that it runs under the softmax of unit j;
//  * warp 17: one lane walks the CTA's share of the schedule and hands the
//    items to the others through a ring in shared memory.  Warps 18 and 19 only
//    complete the warpgroup, whose registers go to the softmax.
// K, V and each tile's S have two stages.  P overwrites the S stage it was made
// from; the tensor pipe runs one thread's MMAs in order, so S of unit j + 2
// lands after P V of unit j has read it.  O is rescaled only when M grows by
// more than 8 (P stays below 2^8, within fp16's range).  A row tile takes no
// part in units that none of its rows see.
//
// Every wait is bounded; on expiry the kernel records kErrWait, every role
// leaves its loop, TMEM is freed and the kernel returns.
#include <cstdio>
#include <type_traits>

#include "kv8.cuh"
#include "tc_common.cuh"

namespace mg {
namespace kv8 {
namespace {
constexpr int kM = 128;   // rows of a tile
constexpr int kN = kUnit; // tokens of a unit
constexpr int kThreads = 640;
// Registers per thread: the block is launched with 96 (5 warps on an SM sub-partition); loaders and the issuing
// warpgroup give up what the softmax takes: 2 x 120 + 2 x 80 + 80 = 5 x 96.
constexpr int kSoftmaxRegs = 120, kLoadRegs = 80, kIssueRegs = 80;
constexpr uint32_t kErrWait = 0x90000u;
constexpr float kInf = __builtin_huge_valf();
constexpr float kRescale = 8.0f;
constexpr int kRing = 8;  // units whose scales are at hand: K's loader runs up to five units ahead of a softmax

template <int HD>
struct Cfg {
    static constexpr bool kTwo = HD <= 128;                 // two row tiles (O and S of both fit TMEM)
    static constexpr int kRows = kTwo ? 2 * kM : kM;        // rows of an item
    static constexpr int kCols = kTwo ? kN : kN / 2;        // score columns of a softmax thread
    static constexpr int kAtoms = HD / 64;
    static constexpr int kDepth = HD == 256 ? 1 : 2;        // units of codes that a loader holds: 32 registers at most
    static constexpr uint32_t kQBytes = kRows * HD * 2, kTileBytes = kN * HD * 2;
    static constexpr uint32_t kS = (kTwo ? 2 : 1) * HD;     // TMEM: O of each tile, then S stages
    static constexpr size_t kSmem = 1024 + kQBytes + 4 * kTileBytes;
};
constexpr uint32_t kTmemCols = 512;

// kind::f16, A and B fp16, D fp32; B transposed: MN-major.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, int b_mn) {
    return (1u << 4) | (static_cast<uint32_t>(b_mn) << 16) | ((static_cast<uint32_t>(n) >> 3) << 17) |
           ((static_cast<uint32_t>(m) >> 4) << 24);
}
// MN-major tile in the 128-byte swizzle: rows (k) of 64 elements 128 bytes apart, 8-row groups 1024 bytes apart
// (stride byte offset), the next 64 elements `lead` bytes further (leading byte offset).
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, uint32_t lead) {
    return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(lead >> 4) << 16) | (64ull << 32) |
           (1ull << 46) | (2ull << 61);
}
// The issuing warp runs converged and one elected lane issues.  The instruction takes its operands from uniform
// registers: they are constants off a few bases, with the stage a template argument and the accumulate flag a
// constant; computed per MMA from loop variables, moving them there took longer than the MMA itself.
template <uint32_t IDESC, bool ACC>
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %3, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %4, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "n"(ACC ? 1 : 0), "r"(IDESC)
        : "memory");
}
template <uint32_t IDESC, bool ACC>
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %3, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %4, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "n"(ACC ? 1 : 0), "r"(IDESC)
        : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
        : "memory");
}
// 32 columns of this thread's TMEM row; the caller waits (tmem_ld_wait) before it reads them.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, float *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
          "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr));
}
template <int N>
__device__ __forceinline__ void tmem_ld_wait(float (&v)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));  // the values exist only after the wait
}

__device__ __forceinline__ uint4 ldg16(const uint8_t *p) {
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
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

// Bounded wait.  err_dev may hold a bad page's code already, so a stop is announced in shared memory.
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, volatile int *stop, uint32_t *err) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t n = 1;; ++n) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((n & 15u) == 0u) {
            if (*stop) return false;
            if (globaltimer_ns() - t0 > kWaitBudgetNs) {
                *stop = 1;
                set_error(err, kErrWait);
                return false;
            }
        }
    }
}

// Two floats in one register pair: the packed fp32 operations.
struct F2 {
    uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void un2(F2 x, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float finite_or_0(float x) { return x == -kInf ? 0.f : x; }

template <int N>
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&v)[N]) {
    static_assert(N == 16 || N == 32, "16 or 32 columns");
    if constexpr (N == 32) {
        tc::tmem_st32(taddr, v);
    } else {
        asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
            "%14, %15, %16};" ::"r"(taddr),
            "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
            "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
            : "memory");
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    }
}

// The CTA's share of the schedule, item by item.
struct Walk {
    int64_t w, w1;
    int head, pair, skip, take;
    bool first;
    Item it;
    // The current item, or the next one with rows; false at the end of the share.
    __device__ __forceinline__ bool settle(const AttnArgs &p) {
        const int pairs = p.b.batch * p.a.tiles;
        while (w < w1) {
            it = load_item(p.b, p.a, pair, false);
            if (it.units > 0) {
                take = static_cast<int>(min(static_cast<int64_t>(it.units - skip), w1 - w));
                return true;
            }
            if (++pair == pairs) pair = 0, ++head;
        }
        return false;
    }
    __device__ __forceinline__ bool start(const AttnArgs &p, const Place &pl) {
        w = pl.w0, w1 = pl.w1, head = pl.head, pair = pl.pair, skip = pl.skip, first = true;
        return settle(p);
    }
    __device__ __forceinline__ bool next(const AttnArgs &p) {
        w += take;
        skip = 0;
        first = false;
        if (++pair == p.b.batch * p.a.tiles) pair = 0, ++head;
        return settle(p);
    }
};
// An item as the walker hands it out.
struct Desc {
    int take;              // units of this CTA's share; 0: the share has ended
    int tok0, lo, hi;      // first token of the first unit; positions seen by any row (lo rounded down to a block)
    int seq, head;
    int q0, pos0;          // first row and position of the sequence's new tokens
    int row0, nrows;
    int t_rows[2], t_lo[2], t_hi[2];  // per row tile: its rows and the positions they see
    int slot;              // of the partial answer; -1: the item is whole
    __device__ __forceinline__ int token(int j) const { return tok0 + j * kN; }
    __device__ __forceinline__ bool sees(int g, int tok, int n = 1) const {  // tile g, n units from tok
        return tok < t_hi[g] && tok + n * kN > t_lo[g];
    }
};
constexpr int kItems = 4;

template <int HD, typename T>
__global__ void __launch_bounds__(kThreads, 1) kv8_prompt_kernel(const AttnArgs p) {
    using C = Cfg<HD>;
    constexpr int kAtoms = C::kAtoms, kTiles = C::kTwo ? 2 : 1, kCols = C::kCols;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], sc_full[kRing], q_full[2], pair_bar[4][2], q_pair[4];
    __shared__ __align__(8) uint64_t item_full[kItems], item_empty[kItems];
    __shared__ Desc items_s[kItems];
    __shared__ __align__(8) uint64_t s_full[2][2], p_full[2][2], pv_done[2][2];  // [tile][stage]
    __shared__ float sc_k[kRing][4], sc_v[kRing][4];  // scales of a unit's four blocks: K, log2 of V
    __shared__ int sc_ok[kRing][4];
    __shared__ float q_down[C::kRows];
    __shared__ float2 xch[2][2][kM];  // one row tile: the two halves' maxima (by unit parity)
    __shared__ uint32_t tmem_slot;
    __shared__ int stop_s;
    volatile int *stop = &stop_s;
    uint32_t *err = p.b.err;
    asm volatile("griddepcontrol.launch_dependents;");
    const uintptr_t base = (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023);
    unsigned char *gen = reinterpret_cast<unsigned char *>(base);
    const uint32_t sq = smem_u32(gen), sk = sq + C::kQBytes, sv = sk + 2 * C::kTileBytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = blockIdx.x;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 4);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 4);
            mbar_init(&v_empty[i], 1);
            mbar_init(&q_full[i], C::kTwo ? 4 : 8);
            for (int g = 0; g < 2; ++g) {
                mbar_init(&s_full[g][i], 1);
                mbar_init(&p_full[g][i], C::kTwo ? 4 : 8);
                mbar_init(&pv_done[g][i], 1);
            }
        }
        for (int i = 0; i < kRing; ++i) mbar_init(&sc_full[i], 8);
        for (int i = 0; i < kItems; ++i) {
            mbar_init(&item_full[i], 1);
            mbar_init(&item_empty[i], 17);  // 8 softmax warps, 8 loaders, the MMA issuer
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&pair_bar[i][0], 2);
            mbar_init(&pair_bar[i][1], 2);
            mbar_init(&q_pair[i], 2);
        }
        stop_s = 0;
        fence_barrier_init();
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const Place pl = find_place<kThreads>(p.b, p.a, p.c.heads, cta, gridDim.x);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const uint32_t units = static_cast<uint32_t>(pl.w1 - pl.w0);
    // The i-th item; null at the end of the share, or (stop set) when a wait ran out.
    auto item = [&](uint32_t i) -> const Desc * {
        const bool ok = wait(&item_full[i % kItems], (i / kItems) & 1u, stop, err);
        return ok && items_s[i % kItems].take > 0 ? &items_s[i % kItems] : nullptr;
    };
    // The same, and a wait, for a whole warp.
    auto warp_item = [&](uint32_t i) -> const Desc * {
        const Desc *x = item(i);
        return __all_sync(0xffffffffu, x != nullptr) ? x : nullptr;
    };
    auto warp_wait = [&](uint64_t *bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, wait(bar, parity, stop, err));
    };

    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (warp == 16) {  // ---- MMA issuer
            constexpr uint32_t kIdS = idesc_f16(kM, kN, 0), kIdO = idesc_f16(kM, HD, 1);
            // descriptors count in 16 bytes; shared memory ends below their 2^14
            const uint64_t qd = tc::sw128_desc(sq), kd = tc::sw128_desc(sk), vd = sw128_mn_desc(sv, kN * 128);
            uint32_t n = 0;                                       // units so far
            uint32_t acts[2] = {0, 0};                            // a tile's items so far in which it sees something
            uint32_t uses[2][2] = {{0, 0}, {0, 0}};               // [tile][stage] P V issued
            bool ok = true;
            for (uint32_t i = 0; ok; ++i) {
                const Desc *d = warp_item(i);
                if (!d) break;
                const int take = d->take;
                bool begun[2] = {false, false};
                auto s_of = [&](auto stage, uint32_t u, int j) -> bool {  // S of unit u, the item's j-th
                    constexpr uint32_t ST = decltype(stage)::value;
                    if (!warp_wait(&k_full[ST], (u >> 1) & 1u)) return false;
                    tc::tc_fence_after();
#pragma unroll
                    for (int g = 0; g < kTiles; ++g) {
                        if (!d->sees(g, d->token(j))) continue;
                        const uint32_t t = tmem + C::kS + (2 * g + ST) * kN;
#pragma unroll
                        for (int kk = 0; kk < HD / 16; ++kk) {
                            const uint64_t qa = qd + (((kk >> 2) * C::kRows * 128 + g * kM * 128 + (kk & 3) * 32) >> 4);
                            const uint64_t kb = kd + ((ST * C::kTileBytes + (kk >> 2) * kN * 128 + (kk & 3) * 32) >> 4);
                            if (kk == 0) umma_ss<kIdS, false>(t, qa, kb);
                            else umma_ss<kIdS, true>(t, qa, kb);
                        }
                        commit(&s_full[g][ST]);
                    }
                    commit(&k_empty[ST]);
                    return true;
                };
                auto pv_of = [&](auto stage, uint32_t u, int j) -> bool {  // P V of unit u
                    constexpr uint32_t ST = decltype(stage)::value;
                    if (!warp_wait(&v_full[ST], (u >> 1) & 1u)) return false;
#pragma unroll
                    for (int g = 0; g < kTiles; ++g) {
                        if (!d->sees(g, d->token(j))) continue;
                        if (!warp_wait(&p_full[g][ST], uses[g][ST]++ & 1u)) return false;
                        tc::tc_fence_after();
                        const uint32_t o = tmem + g * HD, t = tmem + C::kS + (2 * g + ST) * kN;
                        const uint64_t vb = vd + ((ST * C::kTileBytes) >> 4);
                        if (begun[g]) umma_ts<kIdO, true>(o, t, vb);
                        else umma_ts<kIdO, false>(o, t, vb);
                        begun[g] = true;
#pragma unroll
                        for (int kk = 1; kk < kN / 16; ++kk) umma_ts<kIdO, true>(o, t + kk * 8, vb + ((kk * 2048) >> 4));
                        commit(&pv_done[g][ST]);
                    }
                    commit(&v_empty[ST]);
                    return true;
                };
                using S0 = std::integral_constant<uint32_t, 0>;
                using S1 = std::integral_constant<uint32_t, 1>;
#pragma unroll
                for (int g = 0; g < kTiles; ++g)
                    if (d->sees(g, d->tok0, take)) ok = ok && warp_wait(&q_full[g], acts[g]++ & 1u);
                if (ok) ok = n & 1 ? s_of(S1(), n, 0) : s_of(S0(), n, 0);
                for (int j = 0; ok && j < take; ++j, ++n) {
                    if (n & 1) ok = (j + 1 == take || s_of(S0(), n + 1, j + 1)) && pv_of(S1(), n, j);
                    else ok = (j + 1 == take || s_of(S1(), n + 1, j + 1)) && pv_of(S0(), n, j);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&item_empty[i % kItems]);
            }
        } else if (warp == 17 && lane == 0) {  // ---- walker
            Walk wk;
            p.part.split[cta].nrows = 0;
            bool more = wk.start(p, pl);
            for (uint32_t i = 0;; ++i) {
                if (i >= kItems && !wait(&item_empty[i % kItems], (i / kItems - 1) & 1u, stop, err)) break;
                Desc &d = items_s[i % kItems];
                d.take = more ? wk.take : 0;
                if (more) {
                    const Item &it = wk.it;
                    const bool whole = wk.take == it.units;
                    const int slot = 2 * cta + (wk.first ? 0 : 1);
                    d.tok0 = (it.unit0 + wk.skip) * kN;
                    d.lo = it.lo & ~(kBlock - 1);
                    d.hi = it.hi;
                    d.seq = wk.pair / p.a.tiles;
                    d.head = wk.head;
                    d.q0 = it.seq.q0;
                    d.pos0 = it.seq.pos0;
                    d.row0 = it.row0;
                    d.nrows = it.nrows;
                    for (int g = 0; g < 2; ++g) {
                        const int rows = min(kM, it.nrows - g * kM);
                        d.t_rows[g] = rows;
                        d.t_lo[g] = d.t_hi[g] = 0;
                        if (rows > 0) {
                            const int first = it.seq.pos0 + (it.row0 + g * kM) / p.a.group;
                            d.t_lo[g] = p.a.window > 0 ? max(0, first - p.a.window + 1) : 0;
                            d.t_hi[g] = it.seq.pos0 + (it.row0 + g * kM + rows - 1) / p.a.group + 1;
                        }
                    }
                    d.slot = whole ? -1 : slot;
                    if (wk.skip == 0 && !whole)
                        p.part.split[cta] = Split{wk.pair, wk.head, it.nrows, slot, owner_of(pl, wk.w + it.units - 1), {0, 0, 0}};
                }
                mbar_arrive(&item_full[i % kItems]);
                if (!more) break;
                more = wk.next(p);
            }
        }
    } else if (warp >= 8) {  // ---- loaders: K or V
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
        const bool is_k = warp < 12;
        const int u = (threadIdx.x - 256) & 127, quad = u >> 2, sub = u & 3;
        const bool leader = sub == 0 && (quad & 15) == 0;  // holds the scales of blocks quad / 16 and quad / 16 + 2
        const uint8_t *codes = (is_k ? p.c.k : p.c.v) + 16 * sub;
        const float *scales = is_k ? p.c.k_scale : p.c.v_scale;
        uint64_t *full = is_k ? k_full : v_full, *empty = is_k ? k_empty : v_empty;
        unsigned char *stage0 = gen + C::kQBytes + (is_k ? 0 : 2 * C::kTileBytes);
        const int slot_mask = (1 << p.c.page_shift) - 1;
        // the unit whose page ids are being read: the j-th of item i_at
        int j = 0, pg[2], pg_tok = 0, pg_head = 0;
        uint32_t i_at = 0;
        bool pg_on[2] = {false, false};
        const Desc *d = warp_item(0);
        auto read_pages = [&]() {
            if (!d) return;
            pg_tok = d->token(j) + quad;
            pg_head = d->head;
            const int32_t *table = p.b.table + d->seq * p.b.table_stride;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int tok = pg_tok + 32 * i;
                pg_on[i] = tok >= d->lo && tok < d->hi;  // pages before a window may be gone
                pg[i] = pg_on[i] ? table[tok >> p.c.page_shift] : 0;
            }
            if (++j == d->take) {
                j = 0;
                __syncwarp();
                if (lane == 0) mbar_arrive(&item_empty[i_at % kItems]);
                d = warp_item(++i_at);
            }
        };
        uint4 r[C::kDepth][2][kAtoms];
        float sc[C::kDepth][2];
        int ok_b[C::kDepth][2];
        auto read_codes = [&](int b) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int page = pg[i], slot = (pg_tok + 32 * i) & slot_mask;
                bool on = pg_on[i];
                if (on && (page < 0 || page >= p.c.num_pages)) {
                    set_error(err, kErrPage);
                    on = false;
                }
                const uint8_t *src = codes + page * p.c.page_stride + pg_head * p.c.head_stride + slot * p.c.token_stride;
#pragma unroll
                for (int a = 0; a < kAtoms; ++a) r[b][i][a] = on ? ldg16(src + 64 * a) : make_uint4(0, 0, 0, 0);
                if (leader) {
                    const int64_t at =
                        ((static_cast<int64_t>(page) * p.c.heads + pg_head) << (p.c.page_shift - 4)) + (slot >> 4);
                    sc[b][i] = on ? scales[at] : 1.f;
                    ok_b[b][i] = on ? 1 : 0;
                }
            }
        };
        // unit n from buffer b; false when a wait ran out
        auto store = [&](uint32_t n, int b) -> bool {
            if (leader) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int blk = (quad >> 4) + 2 * i;
                    if (is_k) {
                        sc_k[n % kRing][blk] = sc[b][i];
                        sc_ok[n % kRing][blk] = ok_b[b][i];
                    } else {
                        sc_v[n % kRing][blk] = __log2f(sc[b][i]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sc_full[n % kRing]);
            const uint32_t st = n & 1;
            if (n >= 2 && !warp_wait(&empty[st], ((n >> 1) - 1) & 1u)) return false;
            unsigned char *tile = stage0 + st * C::kTileBytes;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = quad + 32 * i;
#pragma unroll
                for (int a = 0; a < kAtoms; ++a) {  // 16 codes -> two 16-byte chunks of the 128-byte row, swizzled
                    uint4 lo, hi;
                    e4m3x4_to_h2x2(r[b][i][a].x, lo.x, lo.y);
                    e4m3x4_to_h2x2(r[b][i][a].y, lo.z, lo.w);
                    e4m3x4_to_h2x2(r[b][i][a].z, hi.x, hi.y);
                    e4m3x4_to_h2x2(r[b][i][a].w, hi.z, hi.w);
                    unsigned char *dst = tile + a * kN * 128 + row * 128;
                    *reinterpret_cast<uint4 *>(dst + (((2 * sub) ^ (row & 7)) << 4)) = lo;
                    *reinterpret_cast<uint4 *>(dst + (((2 * sub + 1) ^ (row & 7)) << 4)) = hi;
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[st]);
            return true;
        };
        read_pages();
#pragma unroll
        for (int b = 0; b < C::kDepth; ++b) {
            if (static_cast<uint32_t>(b) < units) read_codes(b);
            read_pages();
        }
        bool ok = true;
        for (uint32_t n0 = 0; ok && n0 < units; n0 += C::kDepth) {
#pragma unroll
            for (int b = 0; b < C::kDepth; ++b) {
                const uint32_t n = n0 + b;
                if (!ok || n >= units) continue;
                ok = store(n, b);
                if (ok && n + C::kDepth < units) read_codes(b);
                read_pages();
            }
        }
    } else {  // ---- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int wg = warp >> 2, tg = C::kTwo ? wg : 0, r = 32 * (warp & 3) + lane;  // tile and row of this thread
        const int col0 = C::kTwo ? 0 : wg * kCols;
        const uint32_t lane_off = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t t_o = tmem + tg * HD + lane_off, t_s0 = tmem + C::kS + 2 * tg * kN + lane_off;
        uint32_t n = 0, acts = 0;         // units of the share; items in which this tile sees something
        uint32_t uses = 0;                // bit st: parity of the tile's uses of stage st
        bool ok = true;
        for (uint32_t i_at = 0;; ++i_at) {
            const Desc *d = warp_item(i_at);
            if (!d) break;
            const int t_rows = d->t_rows[tg], take = d->take;
            const bool active = d->sees(tg, d->tok0, take);
            // Q: a warp brings kQR rows, lane d with HD / 32 values of each; a row's largest becomes 2^7 .. 2^8
            if (active) {
                constexpr int kW = HD / 64, kQR = C::kTwo ? 32 : 16, kBatch = kW == 4 ? 8 : 16;
                const int qr0 = kQR * warp;  // of the item
                int64_t off = 0;
                const int nrows = d->nrows;
                if (lane < kQR && qr0 + lane < nrows) {
                    const int row = d->row0 + qr0 + lane, tok = row / p.a.group;
                    off = (static_cast<int64_t>(d->q0) + tok) * p.q_row +
                          (d->head * p.a.group + row - tok * p.a.group) * p.q_head;
                }
#pragma unroll 1
                for (int r0 = 0; r0 < kQR && qr0 + r0 < nrows; r0 += kBatch) {
                    uint32_t q[kBatch][kW];
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) {
                        const T *src = static_cast<const T *>(p.q) + __shfl_sync(0xffffffffu, off, r0 + i) + lane * 2 * kW;
#pragma unroll
                        for (int w = 0; w < kW; ++w) q[i][w] = 0;
                        if (qr0 + r0 + i < nrows) {
                            if constexpr (kW == 1) {
                                q[i][0] = *reinterpret_cast<const uint32_t *>(src);
                            } else if constexpr (kW == 2) {
                                const uint2 v = *reinterpret_cast<const uint2 *>(src);
                                q[i][0] = v.x, q[i][1] = v.y;
                            } else {
                                const uint4 v = *reinterpret_cast<const uint4 *>(src);
                                q[i][0] = v.x, q[i][1] = v.y, q[i][2] = v.z, q[i][3] = v.w;
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) {
                        const int lr = qr0 + r0 + i;
                        uint32_t most = 0;
#pragma unroll
                        for (int w = 0; w < kW; ++w) {
                            const float2 f = two<T>(q[i][w]);
                            most = max(most, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
                        }
                        most = __reduce_max_sync(0xffffffffu, most);
                        const int e = static_cast<int>(most >> 23);
                        float up = 1.0f, down = 1.0f;
                        if (e >= 255) {  // a row with an infinity or NaN answers NaN
                            down = __int_as_float(0x7fc00000);
                        } else if (e > 0) {
                            const int sh = min(134 - e, 126);
                            up = __uint_as_float(static_cast<uint32_t>(127 + sh) << 23);
                            down = __uint_as_float(static_cast<uint32_t>(127 - sh) << 23);
                        }
                        if (p.scale_log2 < 0.f) up = -up;  // factors of S stay positive
                        if (lane == 0) q_down[lr] = down;
                        uint32_t hw[kW];
#pragma unroll
                        for (int w = 0; w < kW; ++w) {
                            const float2 f = two<T>(q[i][w]);
                            hw[w] = pack(f.x * up, f.y * up, __half());
                        }
                        // byte 4 kW lane of the row: atom, chunk and offset
                        const int byte = 4 * kW * lane, atom = byte >> 7, chunk = (byte >> 4) & 7, in = byte & 15;
                        unsigned char *dst = gen + atom * C::kRows * 128 + lr * 128 + ((chunk ^ (lr & 7)) << 4) + in;
                        if constexpr (kW == 1) *reinterpret_cast<uint32_t *>(dst) = hw[0];
                        else if constexpr (kW == 2) *reinterpret_cast<uint2 *>(dst) = make_uint2(hw[0], hw[1]);
                        else *reinterpret_cast<uint4 *>(dst) = make_uint4(hw[0], hw[1], hw[2], hw[3]);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[tg]);
                ok = warp_wait(&q_full[tg], acts++ & 1u);
                if (!ok) break;
            }
            const bool any_rows = 32 * (warp & 3) < t_rows, row_on = r < t_rows;
            const float factor = active && row_on ? fabsf(p.scale_log2) * q_down[tg * kM + r] : 0.f;
            const int pos = d->pos0 + (d->row0 + tg * kM + r) / p.a.group;
            const int hi = row_on ? pos + 1 : 0, lo = p.a.window > 0 ? pos - p.a.window + 1 : 0;

            float m = -kInf, mref = -kInf, l = 0.f;
            bool begun = false;
            uint32_t last = 0;  // stage of the tile's latest unit
            for (int j = 0; j < take; ++j, ++n) {
                const int t0 = d->token(j);
                if (!d->sees(tg, t0)) continue;
                const uint32_t st = n & 1, ph = uses >> st & 1u;
                // S first: a tile that sat out many units is then within one phase of the scales' barrier
                ok = warp_wait(&s_full[tg][st], ph) && warp_wait(&sc_full[n % kRing], (n / kRing) & 1u);
                if (!ok) break;
                tc::tc_fence_after();
                if (any_rows) {
                    const uint32_t t_s = t_s0 + st * kN;
                    constexpr int kB = kCols / 16;  // scale blocks of this thread's columns
                    float s[kCols], cf[kB], lv[kB];
                    tmem_ld32_async(t_s + col0, s);
                    if constexpr (kCols == 64) tmem_ld32_async(t_s + 32, s + 32);
                    bool blocks_ok = true;
#pragma unroll
                    for (int b = 0; b < kB; ++b) {
                        cf[b] = factor * sc_k[n % kRing][col0 / 16 + b];
                        lv[b] = sc_v[n % kRing][col0 / 16 + b];
                        blocks_ok = blocks_ok && sc_ok[n % kRing][col0 / 16 + b] != 0;
                    }
                    tmem_ld_wait(s);
                    const int tc0 = t0 + col0;
                    const bool all = !row_on || (blocks_ok && lo <= tc0 && tc0 + kCols <= hi);
                    if (!__all_sync(0xffffffffu, all)) {
#pragma unroll
                        for (int b = 0; b < kB; ++b) {
                            const bool on = sc_ok[n % kRing][col0 / 16 + b] != 0;
#pragma unroll
                            for (int i = 16 * b; i < 16 * b + 16; ++i)
                                s[i] = on && tc0 + i >= lo && tc0 + i < hi ? s[i] * cf[b] : -kInf;
                            cf[b] = 1.0f;
                        }
                    }
                    float mn = -kInf, vn = -kInf;
#pragma unroll
                    for (int b = 0; b < kB; ++b) {
                        const float *x = s + 16 * b;
                        float a0 = max3(x[0], x[1], x[2]), a1 = max3(x[3], x[4], x[5]);
                        a0 = max3(a0, x[6], x[7]), a1 = max3(a1, x[8], x[9]);
                        a0 = max3(a0, x[10], x[11]), a1 = max3(a1, x[12], x[13]);
                        const float t = fmaxf(max3(a0, x[14], x[15]), a1) * cf[b];
                        mn = fmaxf(mn, t);
                        vn = fmaxf(vn, t + lv[b]);
                    }
                    if constexpr (!C::kTwo) {  // the other half's columns
                        xch[st][wg][r] = make_float2(mn, vn);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&pair_bar[warp & 3][st]);
                        ok = warp_wait(&pair_bar[warp & 3][st], ph);
                        if (!ok) break;
                        const float2 o = xch[st][wg ^ 1][r];
                        mn = fmaxf(mn, o.x);
                        vn = fmaxf(vn, o.y);
                    }
                    mn = fmaxf(mn, m);
                    const float mb = finite_or_0(mn);
                    l *= ex2(m - mb);
                    m = mn;
                    const bool move = vn > mref + kRescale || (mref == -kInf && vn > -kInf);
                    const float old = mref;
                    if (move) mref = vn;
                    const float rb = finite_or_0(mref);
                    if (begun && __any_sync(0xffffffffu, move)) {
                        // O holds P V of this tile's units so far once the last one is done
                        ok = warp_wait(&pv_done[tg][st ^ 1], (uses >> (st ^ 1) & 1u) ^ 1u);
                        if (!ok) break;
                        tc::tc_fence_after();
                        const float f = move ? ex2(old - rb) : 1.0f;
                        constexpr int kOc = C::kTwo ? HD : HD / 2;
#pragma unroll 1
                        for (int x = 0; x < kOc; x += 32) {
                            uint32_t o[32];
                            const uint32_t at = t_o + (C::kTwo ? 0 : wg * kOc) + x;
                            tc::tmem_ld32(at, o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tc::tmem_st32(at, o);
                        }
                    }
                    uint32_t pk[kCols / 2];
                    F2 sum = f2(0.f, 0.f);
                    const F2 nm = f2(-mb, -mb);
#pragma unroll
                    for (int b = 0; b < kB; ++b) {
                        const float wv = ex2(fminf(lv[b] + mb - rb, 126.f));
                        const F2 w2 = f2(wv, wv), c2 = f2(cf[b], cf[b]);
#pragma unroll
                        for (int i = 16 * b; i < 16 * b + 16; i += 2) {
                            float e0, e1;
                            un2(fma2(f2(s[i], s[i + 1]), c2, nm), e0, e1);
                            const F2 e = f2(ex2(e0), ex2(e1));
                            sum = add2(sum, e);
                            un2(mul2(e, w2), e0, e1);
                            pk[i / 2] = pack(e0, e1, __half());
                        }
                    }
                    float s0, s1;
                    un2(sum, s0, s1);
                    l += s0 + s1;
                    tmem_st(t_s + col0 / 2, pk);
                }
                begun = true;
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[tg][st]);
                uses ^= 1u << st;
                last = st;
            }
            if (!ok) break;
            if (begun) {
                ok = warp_wait(&pv_done[tg][last], (uses >> last & 1u) ^ 1u);
                if (!ok) break;
                tc::tc_fence_after();
            }
            if constexpr (!C::kTwo) {  // the two halves' sums; the pair's barrier has another phase per item
                xch[0][wg][r] = make_float2(l, 0.f);
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_pair[warp & 3]);
                ok = warp_wait(&q_pair[warp & 3], i_at & 1u);
                if (!ok) break;
                l = xch[0][0][r].x + xch[0][1][r].x;
            }
            if (any_rows) {
                const int slot = d->slot;
                const bool whole = slot < 0;
                const float f = l == 0.f || !begun ? 0.f : ex2(finite_or_0(mref) - finite_or_0(m)) / l;
                const int row = d->row0 + tg * kM + r, tok = row / p.a.group, hq = d->head * p.a.group + row - tok * p.a.group;
                T *dst = static_cast<T *>(p.out) + (static_cast<int64_t>(d->q0) + tok) * p.out_row + hq * p.out_head;
                const int64_t at = static_cast<int64_t>(slot) * C::kRows + tg * kM + r;
                if (!whole && row_on && col0 == 0) *reinterpret_cast<float2 *>(p.part.ml + 2 * at) = make_float2(m, l);
                constexpr int kOc = C::kTwo ? HD : HD / 2;
#pragma unroll 1
                for (int x0 = 0; x0 < kOc; x0 += 32) {
                    const int x = x0 + (C::kTwo ? 0 : wg * kOc);
                    float o[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0.f;
                    if (begun) {
                        tmem_ld32_async(t_o + x, o);
                        tmem_ld_wait(o);
                    }
                    if (!row_on) continue;
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] *= f;
                    if (whole) {
                        uint4 *d4 = reinterpret_cast<uint4 *>(dst + x);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            d4[i] = make_uint4(pack(o[8 * i], o[8 * i + 1], T()), pack(o[8 * i + 2], o[8 * i + 3], T()),
                                               pack(o[8 * i + 4], o[8 * i + 5], T()), pack(o[8 * i + 6], o[8 * i + 7], T()));
                    } else {
                        float4 *d4 = reinterpret_cast<float4 *>(p.part.o + at * HD + x);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            d4[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
            }
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[i_at % kItems]);
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        tc::tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    }
}

template <int HD, typename T>
cudaError_t launch(const AttnArgs &p, int ctas, cudaStream_t s) {
    const cudaError_t e = cudaFuncSetAttribute(kv8_prompt_kernel<HD, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(Cfg<HD>::kSmem));
    if (e != cudaSuccess) return e;
    kv8_prompt_kernel<HD, T><<<ctas, kThreads, Cfg<HD>::kSmem, s>>>(p);
    return cudaGetLastError();
}
}  // namespace

int prompt_rows(int hd) { return hd == 256 ? Cfg<256>::kRows : Cfg<128>::kRows; }

cudaError_t launch_prompt(const AttnArgs &p, int hd, bool f16, int ctas, cudaStream_t s) {
    if (hd == 64) return f16 ? launch<64, __half>(p, ctas, s) : launch<64, __nv_bfloat16>(p, ctas, s);
    if (hd == 128) return f16 ? launch<128, __half>(p, ctas, s) : launch<128, __nv_bfloat16>(p, ctas, s);
    return f16 ? launch<256, __half>(p, ctas, s) : launch<256, __nv_bfloat16>(p, ctas, s);
}

}  // namespace kv8
}  // namespace mg
