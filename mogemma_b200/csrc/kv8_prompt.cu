// kv8_prompt.cu -- mg_kv8_attention for many query rows per kv head (prompts,
// prompt chunks, drafts of several tokens): the 5th-generation tensor cores on
// the 8-bit paged cache.
//
// An item's query rows ((token, q head of the group) pairs of one kv head) are
// one or two tiles of 128 (two for head dims 64 and 128, which then share every
// widened key and value); its keys run in units of 128 tokens.  Both products
// are tcgen05.mma kind::f16 with fp32 accumulators in TMEM:
//   S [128 x 128] = Q . K^T       Q and K fp16 in shared memory, K-major
//   O [128 x hd] += P . V         P fp16 in TMEM (over S), V fp16 MN-major
// The cache's codes are widened to fp16, which is exact, on their way into
// shared memory; q is brought into fp16's range by a power of two per row.  The
// block scales of K multiply the score columns, those of V ride in P's
// exponent: with s = scale log2(e) k_scale <q, k>, m = max s and
// M = max(s + log2 v_scale), P = 2^(s + log2 v_scale - M + 8) and l = sum
// 2^(s - m), so P is bounded whatever the scales.  fp16, the MMA operand's type,
// holds P to 2^-11 of itself down to 2^-22 of the row's largest, below that to
// 2^-33 of the largest, where a term also ends; m and M may lag (kRescale),
// which only widens that.
//
// Warps of a CTA (640 threads, one CTA per SM):
//  * warps 0-7: softmax.  Two row tiles: warpgroup g has tile g, a row per
//    thread (TMEM lane = row).  One row tile (hd 256): warpgroup g has columns
//    64 g .. 64 g + 63 of every row, and the two threads of a row exchange their
//    maxima.  They also bring the item's Q into shared memory and write the
//    answers;
//  * warps 8-11 load K, 12-15 V: a unit's codes from the pages into registers
//    one unit ahead (page ids two ahead), widened and stored in the 128-byte
//    swizzled layout (token rows of 64 dims); tokens that no row sees become
//    zeros, so that stale codes behind the context cannot reach a product.  The
//    loads go out behind the fence that publishes the unit before: a fence waits
//    for the loads in flight;
//  * warps 16 and 17: issue the MMAs, one warp per row tile (16 also allocates
//    TMEM);
//  * warp 18: one lane walks the CTA's share of the schedule and hands the
//    items to the others through a ring in shared memory.
//
// Two row tiles have one S stage each and take turns: P V and the next S of one
// run under the softmax of the other.  One row tile has two S stages: S of unit
// j + 1 is issued before P V of unit j and runs under its softmax.  P overwrites
// the S it was made from; the tensor pipe runs one thread's MMAs in order, so
// the next S on a stage lands after P V has read P.  K and V have two stages
// each (hd 256: one; S and P V alternate, and either is reloaded under the
// other).  O is rescaled only when m or M grows by more than 7.9 (P stays within
// fp16's range).  A row tile takes no part in units that none of its
// rows see.
//
// Units of 64 tokens were the first form: N = 64 reads Q from shared memory for
// half the work (48 cycles per MMA against 64 for N = 128), and the waits
// between roles (200 to 300 cycles each) came twice as often.
//
// Measured (in a graph, with the combine; then without loads, without softmax,
// without either): 4096 bf16 tokens of 32 q and 16 kv heads of 128 in one prompt,
// 273 us, 504 TFLOP/s of the masked products (252, 151, 134); chunks of 512 and
// 365 tokens that end at 8192 and 5844 positions, 8 / 4 heads of 256, 102 us, 492
// TFLOP/s (83, 82, 60); seven prompts of 246 to 777 tokens, 12 / 4 heads of 64,
// 40 us (40, 28, 27).  What bounds it: at hd 128 the softmax, two warps on an SM
// sub-partition not hiding each other's latencies (TMEM loads, the row's serial
// maximum, the exponentials, the store of P); at hd 256, with one row tile and
// one stage of K and V, the hand-offs between MMAs, loads and softmax in equal
// parts; short prompts, the launches, Q, the first K and the join.
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
constexpr int kN = 128;   // tokens of a unit
constexpr int kThreads = 640;
// log2 of P at a row's reference M, and how far the maximum may grow past M before O is rescaled: P stays below
// 2^15.9, within fp16.  A higher lift keeps more of the weights far below the row's largest (down to 2^(-24 - kLift)) and
// rescales more often: lift 0, 6, 8, 13 take 261, 266, 272, 284 us for the 27B prompt below, whose key scales lie 8
// times apart, and 259 us each where they are alike.
constexpr float kLift = 8.0f, kUnlift = 1.0f / 256.0f;  // 2^-kLift apart from ex2, which ends at 2^-126
constexpr float kRescale = 15.9f - kLift;
constexpr int kRing = 4;  // units whose scales are at hand

template <int HD>
struct Cfg {
    static constexpr bool kTwo = HD <= 128;                 // two row tiles (O and S of both fit TMEM)
    static constexpr int kRows = kTwo ? 2 * kM : kM;        // rows of an item
    static constexpr int kCols = kTwo ? kN : kN / 2;        // score columns of a softmax thread
    static constexpr int kChunk = kTwo ? 64 : 32;           // of which it holds so many at a time
    // Registers per thread: the block is launched with 96 (5 warps on an SM sub-partition); the softmax holds kChunk
    // scores, a loader 32 registers of codes (hd 256: 64).  2 softmax + 2 load + issue = 5 x 96.
    static constexpr int kSoftmaxRegs = kTwo ? 120 : 96, kLoadRegs = kTwo ? 80 : 104, kIssueRegs = 80;
    static constexpr int kStages = kTwo ? 2 : 1;            // of K and of V
    static constexpr int kSStages = kTwo ? 1 : 2;           // of each tile's S
    static constexpr uint32_t kQBytes = kRows * HD * 2, kTileBytes = kN * HD * 2;
    static constexpr uint32_t kS = (kTwo ? 2 : 1) * HD;     // TMEM: O of each tile, then the S stages
    static constexpr size_t kSmem = 1024 + kQBytes + 2 * kStages * kTileBytes;
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
// The whole issuing warp runs this code and lane 0 (`lead`) issues: one thread's MMAs run in order, and nothing depends
// on the warp being converged, as an elect.sync here would.  The operands are constants off a few bases, with the
// stage a template argument and the accumulate flag a constant.
template <uint32_t IDESC, bool ACC>
__device__ __forceinline__ void umma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 p, %3, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %4, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "n"(ACC ? 1 : 0), "r"(IDESC), "r"(lead)
        : "memory");
}
template <uint32_t IDESC, bool ACC>
__device__ __forceinline__ void umma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 p, %3, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %4, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "n"(ACC ? 1 : 0), "r"(IDESC), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t lead, uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(lead)
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
// Bounded wait.  err_dev may hold a bad page's code already, so a stop is announced in shared memory.
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, volatile int *stop, uint32_t *err,
                                     const volatile uint64_t *budget) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t n = 1;; ++n) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((n & 15u) == 0u) {
            if (*stop) return false;
            if (globaltimer_ns() - t0 > *budget) {
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
    constexpr int kTiles = C::kTwo ? 2 : 1, kCols = C::kCols, kSt = C::kStages, kSS = C::kSStages;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], sc_full[kRing], q_full[2], pair_bar[4][2], q_pair[4];
    __shared__ __align__(8) uint64_t item_full[kItems], item_empty[kItems];
    __shared__ __align__(8) uint64_t s_full[2][2], p_full[2][2], pv_done[2][2];  // [tile][S stage]
    __shared__ __align__(8) uint64_t drained[2];  // a tile's MMAs have all run
    __shared__ Desc items_s[kItems];
    __shared__ __align__(16) float sc_k[kRing][8], sc_v[kRing][8];  // scales of a unit's eight blocks: K, log2 of V
    __shared__ __align__(8) uint8_t sc_ok[kRing][8];
    __shared__ float q_down[C::kRows];
    __shared__ float2 xch[2][2][kM];  // one row tile: the two halves' maxima (by S stage)
    __shared__ uint32_t tmem_slot;
    __shared__ int stop_s;
    __shared__ uint64_t budget_s;  // of a wait; in shared memory, read by a wait that lasts, it takes no registers
    volatile int *stop = &stop_s;
    const volatile uint64_t *budget = &budget_s;
    uint32_t *err = p.b.err;
    const uintptr_t base = (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023);
    unsigned char *gen = reinterpret_cast<unsigned char *>(base);
    const uint32_t sq = smem_u32(gen), sk = sq + C::kQBytes, sv = sk + kSt * C::kTileBytes;
    // broadcast, so that what depends on the warp alone is warp-uniform to the compiler (the MMAs' operands)
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int cta = blockIdx.x;

    if (threadIdx.x == 0) {
        // one arrival more than there will be withholds a hand-off (a test of the bounded waits)
        auto init = [&](uint64_t *bar, int arrivals, Handoff h) {
            mbar_init(bar, arrivals + (cta == 0 && p.stall == h ? 1 : 0));
        };
        for (int i = 0; i < 2; ++i) {
            init(&k_full[i], 4, kKFull);
            init(&k_empty[i], kTiles, kKEmpty);
            init(&v_full[i], 4, kVFull);
            init(&v_empty[i], kTiles, kVEmpty);
            init(&q_full[i], C::kTwo ? 4 : 8, kQFull);
            for (int g = 0; g < 2; ++g) {
                init(&s_full[g][i], 1, kSFull);
                init(&p_full[g][i], C::kTwo ? 4 : 8, kPFull);
                init(&pv_done[g][i], 1, kPvDone);
            }
            init(&drained[i], 1, kDrained);
        }
        for (int i = 0; i < kRing; ++i) init(&sc_full[i], 8, kScales);
        for (int i = 0; i < kItems; ++i) {
            init(&item_full[i], 1, kItemFull);
            init(&item_empty[i], 16 + kTiles, kItemEmpty);  // 8 softmax warps, 8 loaders, the MMA issuers
        }
        for (int i = 0; i < 4; ++i) {
            init(&pair_bar[i][0], 2, kPair);
            init(&pair_bar[i][1], 2, kPair);
            init(&q_pair[i], 2, kPair);
        }
        stop_s = 0;
        budget_s = p.wait_ns;
        fence_barrier_init();
    }
    // before the allocation: a predecessor that lets this kernel begin early may still have to allocate TMEM itself, and
    // would wait for this kernel, which waits for it
    kernel_begins();
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
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
    // The i-th item; null at the end of the share, or (stop set) when a wait ran out.
    auto item = [&](uint32_t i) -> const Desc * {
        const bool ok = wait(&item_full[i % kItems], (i / kItems) & 1u, stop, err, budget);
        return ok && items_s[i % kItems].take > 0 ? &items_s[i % kItems] : nullptr;
    };
    // The same, and a wait, for a whole warp.
    auto warp_item = [&](uint32_t i) -> const Desc * {
        const Desc *x = item(i);
        return __all_sync(0xffffffffu, x != nullptr) ? x : nullptr;
    };
    auto warp_wait = [&](uint64_t *bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, wait(bar, parity, stop, err, budget));
    };

    if (warp >= 16) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kIssueRegs));
    if (warp >= 16 && warp < 16 + kTiles) {  // ---- MMA issuers: warp 16 + g has row tile g
        constexpr uint32_t kIdS = idesc_f16(kM, kN, 0), kIdO = idesc_f16(kM, HD, 1);
        const int g = warp - 16;
        const uint32_t lead = lane == 0 ? 1u : 0u;
        auto commit = [&](uint64_t *bar) { commit_if(lead, bar); };
        // descriptors count in 16 bytes; shared memory ends below their 2^14
        const uint64_t qd = tc::sw128_desc(sq + g * kM * 128), kd = tc::sw128_desc(sk), vd = sw128_mn_desc(sv, kN * 128);
        const uint32_t t_o = tmem + g * HD, t_s = tmem + C::kS + kSS * g * kN;
        uint32_t n = 0;     // units so far
        uint32_t acts = 0;  // the tile's items so far in which it sees something
        uint32_t uses = 0;  // bit st: parity of the tile's uses of S stage st
        bool ok = true;
        for (uint32_t i = 0; ok; ++i) {
            const Desc *d = warp_item(i);
            if (!d) break;
            const int take = d->take;
            bool begun = false;
            auto sees = [&](int j) { return d->sees(g, d->token(j)); };
            // S of unit u, the item's j-th
            auto s_at = [&](auto parity, uint32_t u, int j) -> bool {
                constexpr uint32_t st = decltype(parity)::value % kSt, ss = decltype(parity)::value % kSS;
                if (!warp_wait(&k_full[st], (u / kSt) & 1u)) return false;
                tc::tc_fence_after();
                if (sees(j)) {
                    const uint64_t kb = kd + ((st * C::kTileBytes) >> 4);
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {
                        const uint64_t a = qd + (((kk >> 2) * C::kRows * 128 + (kk & 3) * 32) >> 4);
                        const uint64_t b = kb + (((kk >> 2) * kN * 128 + (kk & 3) * 32) >> 4);
                        if (kk == 0) umma_ss<kIdS, false>(lead, t_s + ss * kN, a, b);
                        else umma_ss<kIdS, true>(lead, t_s + ss * kN, a, b);
                    }
                    commit(&s_full[g][ss]);
                }
                commit(&k_empty[st]);
                return true;
            };
            // P V of unit n, the item's j-th
            auto pv_at = [&](auto parity, int j) -> bool {
                constexpr uint32_t st = decltype(parity)::value % kSt, ss = decltype(parity)::value % kSS;
                if (!warp_wait(&v_full[st], (n / kSt) & 1u)) return false;
                if (sees(j)) {
                    if (!warp_wait(&p_full[g][ss], uses >> ss & 1u)) return false;
                    uses ^= 1u << ss;
                    tc::tc_fence_after();
                    const uint32_t t = t_s + ss * kN;
                    const uint64_t vb = vd + ((st * C::kTileBytes) >> 4);
                    if (begun) umma_ts<kIdO, true>(lead, t_o, t, vb);
                    else umma_ts<kIdO, false>(lead, t_o, t, vb);
                    begun = true;
#pragma unroll
                    for (int kk = 1; kk < kN / 16; ++kk) {
                        // P's columns: 8 per step of 16 tokens; one row tile: the second half's behind column kN / 2
                        const uint32_t col = C::kTwo || kk < 4 ? kk * 8 : kN / 2 + (kk - 4) * 8;
                        umma_ts<kIdO, true>(lead, t_o, t + col, vb + ((kk * 2048) >> 4));
                    }
                    commit(&pv_done[g][ss]);
                }
                commit(&v_empty[st]);
                return true;
            };
            using Even = std::integral_constant<uint32_t, 0>;  // stages are constants to the MMAs
            using Odd = std::integral_constant<uint32_t, 1>;
            auto s_of = [&](uint32_t u, int j) { return u & 1 ? s_at(Odd(), u, j) : s_at(Even(), u, j); };
            auto pv_of = [&](int j) { return n & 1 ? pv_at(Odd(), j) : pv_at(Even(), j); };
            if (d->sees(g, d->tok0, take)) ok = warp_wait(&q_full[g], acts++ & 1u);
            ok = ok && s_of(n, 0);
            for (int j = 0; ok && j < take; ++j, ++n) {
                if constexpr (C::kTwo) ok = pv_of(j) && (j + 1 == take || s_of(n + 1, j + 1));
                else ok = (j + 1 == take || s_of(n + 1, j + 1)) && pv_of(j);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[i % kItems]);
        }
        commit(&drained[g]);  // after a wait that ran out MMAs may be in flight: TMEM and shared memory are held for them
        volatile int never = 0;
        wait(&drained[g], 0, &never, err, budget);
    } else if (warp == 18) {  // ---- walker
        if (lane == 0) {
            Walk wk;
            p.part.split[cta].nrows = 0;
            bool more = wk.start(p.b, p.a, pl);
            for (uint32_t i = 0;; ++i) {
                if (i >= kItems && !wait(&item_empty[i % kItems], (i / kItems - 1) & 1u, stop, err, budget)) break;
                Desc &d = items_s[i % kItems];
                d.take = more ? wk.take : 0;
                if (more) {
                    const Item &it = wk.it;
                    const bool whole = wk.whole();
                    d.tok0 = (it.unit0 + wk.first) * kN;
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
                    d.slot = whole ? -1 : wk.slot(cta);
                    if (wk.first == 0 && !whole) p.part.split[cta] = Split{wk.pair, wk.head, it.nrows, wk.last_cta(pl)};
                }
                mbar_arrive(&item_full[i % kItems]);
                if (!more) break;
                more = wk.next(p.b, p.a);
            }
        }
    } else if (warp >= 8 && warp < 16) {  // ---- loaders: K or V
        if constexpr (C::kLoadRegs < 96) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kLoadRegs));
        if constexpr (C::kLoadRegs > 96) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kLoadRegs));
        const bool is_k = warp < 12;
        const int u = (threadIdx.x - 256) & 127, quad = u >> 2, sub = u & 3;  // tokens quad + 32 i, 16 bytes of each 64
        const bool leader = sub == 0 && (quad & 15) == 0;  // holds the scales of blocks quad / 16 + 2 i
        const uint8_t *codes = (is_k ? p.c.k : p.c.v) + 16 * sub;
        const float *scales = is_k ? p.c.k_scale : p.c.v_scale;
        uint64_t *full = is_k ? k_full : v_full, *empty = is_k ? k_empty : v_empty;
        unsigned char *stage0 = gen + C::kQBytes + (is_k ? 0 : kSt * C::kTileBytes);
        const int slot_mask = (1 << p.c.page_shift) - 1;
        // the unit whose page ids are being read: the j-th of item i_at
        int j = 0, pg[4] = {0, 0, 0, 0}, pg_tok = 0, pg_head = 0, pg_lo = 0, pg_hi = 0;
        uint32_t i_at = 0;
        const Desc *d = warp_item(0);
        auto seen = [&](int i) { return pg_tok + 32 * i >= pg_lo && pg_tok + 32 * i < pg_hi; };
        auto read_pages = [&]() -> bool {  // false: the share has ended
            if (!d) return false;
            pg_tok = d->token(j) + quad;
            pg_head = d->head;
            pg_lo = d->lo;  // pages before a window may be gone
            pg_hi = d->hi;
            const int32_t *table = p.b.table + d->seq * p.b.table_stride;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (seen(i)) pg[i] = table[(pg_tok + 32 * i) >> p.c.page_shift];
            if (++j == d->take) {
                j = 0;
                __syncwarp();
                if (lane == 0) mbar_arrive(&item_empty[i_at % kItems]);
                d = warp_item(++i_at);
            }
            return true;
        };
        uint4 r[4][HD / 64];
        float sc[4];
        uint32_t ok_b = 0;  // bit i: block quad / 16 + 2 i is there
        auto read_codes = [&]() {
            ok_b = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int page = pg[i], slot = (pg_tok + 32 * i) & slot_mask;
                bool on = seen(i);
                if (on && (page < 0 || page >= p.c.num_pages)) {
                    set_error(err, kErrPage);
                    on = false;
                }
                const uint8_t *src = codes + page * p.c.page_stride + pg_head * p.c.head_stride + slot * p.c.token_stride;
#pragma unroll
                for (int a = 0; a < HD / 64; ++a) r[i][a] = on ? ldg16(src + 64 * a) : make_uint4(0, 0, 0, 0);
                sc[i] = 1.0f;
                if (leader && on) {
                    sc[i] = scales[((static_cast<int64_t>(page) * p.c.heads + pg_head) << (p.c.page_shift - 4)) + (slot >> 4)];
                    ok_b |= 1u << i;
                }
            }
        };
        // unit n; false when a wait ran out
        auto store = [&](uint32_t n) -> bool {
            const uint32_t st = n % kSt;
            if (n >= kSt && !warp_wait(&empty[st], (n / kSt - 1) & 1u)) return false;
            if (leader) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int blk = (quad >> 4) + 2 * i;
                    if (is_k) {
                        sc_k[n % kRing][blk] = sc[i];
                        sc_ok[n % kRing][blk] = static_cast<uint8_t>(ok_b >> i & 1u);
                    } else {
                        sc_v[n % kRing][blk] = __log2f(sc[i]);
                    }
                }
            }
            unsigned char *row = stage0 + st * C::kTileBytes + quad * 128;  // token quad + 32 i: (quad + 32 i) & 7 = quad & 7
            const int lo_at = ((2 * sub) ^ (quad & 7)) << 4, hi_at = ((2 * sub + 1) ^ (quad & 7)) << 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int a = 0; a < HD / 64; ++a) {  // 16 codes -> two 16-byte chunks of the 128-byte row, swizzled
                    uint4 lo, hi;
                    e4m3x4_to_h2x2(r[i][a].x, lo.x, lo.y);
                    e4m3x4_to_h2x2(r[i][a].y, lo.z, lo.w);
                    e4m3x4_to_h2x2(r[i][a].z, hi.x, hi.y);
                    e4m3x4_to_h2x2(r[i][a].w, hi.z, hi.w);
                    *reinterpret_cast<uint4 *>(row + a * kN * 128 + i * 32 * 128 + lo_at) = lo;
                    *reinterpret_cast<uint4 *>(row + a * kN * 128 + i * 32 * 128 + hi_at) = hi;
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sc_full[n % kRing]);
                mbar_arrive(&full[st]);
            }
            return true;
        };
        bool held = read_pages(), ok = true;
        if (held) read_codes();
        bool have = read_pages();
        for (uint32_t n = 0; ok && held; ++n) {
            ok = store(n);
            held = have;
            if (ok && have) read_codes();
            have = read_pages();
        }
    } else if (warp < 8) {  // ---- softmax
        if constexpr (C::kSoftmaxRegs > 96) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
        const int wg = warp >> 2, tg = C::kTwo ? wg : 0, r = 32 * (warp & 3) + lane;  // tile and row of this thread
        const int col0 = C::kTwo ? 0 : wg * kCols;
        const uint32_t lane_off = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t t_o = tmem + tg * HD + lane_off, t_s0 = tmem + C::kS + kSS * tg * kN + lane_off;
        uint32_t n = 0, acts = 0;         // units of the share; items in which this tile sees something
        uint32_t uses = 0;                // bit st: parity of the tile's uses of S stage st
        uint32_t met = 0;                 // bit st: parity of this warp's exchanges with its other half
        bool ok = true;
        for (uint32_t i_at = 0;; ++i_at) {
            const Desc *d = warp_item(i_at);
            if (!d) break;
            const int t_rows = d->t_rows[tg], take = d->take;
            const bool active = d->sees(tg, d->tok0, take);
            if (active) {
                // Q: a warp brings kQR rows, 8 kB at a time, 4 lanes to a row; a row's largest becomes 2^15 .. 2^16
                constexpr int kQR = C::kTwo ? 32 : 16, kCh = HD / 32;  // 16-byte chunks of a lane: 4 i + lane % 4
                constexpr int kB = kCh >= 8 ? 1 : 8 / kCh < kQR / 8 ? 8 / kCh : kQR / 8;  // rows of a lane: 32 registers
                const int nrows = d->nrows, sub = lane & 3;
#pragma unroll 1
                for (int r0 = kQR * warp; r0 < kQR * (warp + 1) && r0 < nrows; r0 += 8 * kB) {
                    uint4 q[kB][kCh];
#pragma unroll
                    for (int y = 0; y < kB; ++y) {
                        const int lr = min(r0 + 8 * y + (lane >> 2), nrows - 1);  // row of the item
                        const int row = d->row0 + lr, tok = row / p.a.group;
                        const T *src = static_cast<const T *>(p.q) + (static_cast<int64_t>(d->q0) + tok) * p.q_row +
                                       (d->head * p.a.group + row - tok * p.a.group) * p.q_head + 8 * sub;
#pragma unroll
                        for (int i = 0; i < kCh; ++i) q[y][i] = *reinterpret_cast<const uint4 *>(src + 32 * i);
                    }
#pragma unroll
                    for (int y = 0; y < kB; ++y) {
                        const int lr = r0 + 8 * y + (lane >> 2);
                        uint32_t most = 0;
#pragma unroll
                        for (int i = 0; i < kCh; ++i) {
                            const uint32_t w[4] = {q[y][i].x, q[y][i].y, q[y][i].z, q[y][i].w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 f = two<T>(w[e]);
                                most = max(most, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
                            }
                        }
                        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
                        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
                        float up, down;
                        row_scale(most, up, down);
                        if (p.scale_log2 < 0.f) up = -up;  // factors of S stay positive
                        if (lr < nrows) {
                            if (sub == 0) q_down[lr] = down;
#pragma unroll
                            for (int i = 0; i < kCh; ++i) {
                                const uint32_t w[4] = {q[y][i].x, q[y][i].y, q[y][i].z, q[y][i].w};
                                uint32_t h[4];
#pragma unroll
                                for (int x = 0; x < 4; ++x) {
                                    const float2 f = two<T>(w[x]);
                                    h[x] = pack(f.x * up, f.y * up, __half());
                                }
                                const int chunk = 4 * (i & 1) + sub;  // of atom i / 2
                                *reinterpret_cast<uint4 *>(gen + (i >> 1) * C::kRows * 128 + lr * 128 +
                                                           ((chunk ^ (lr & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
                            }
                        }
                        __syncwarp();
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
            uint32_t last = 0;  // S stage of the tile's latest unit
            for (int j = 0; j < take; ++j, ++n) {
                const int t0 = d->token(j);
                if (!d->sees(tg, t0)) continue;
                const uint32_t st = n % kSS, ph = uses >> st & 1u, ring = n % kRing;
                // S first: a tile that sat out many units is then within one phase of the scales' barrier
                ok = warp_wait(&s_full[tg][st], ph) && warp_wait(&sc_full[ring], (n / kRing) & 1u);
                if (!ok) break;
                tc::tc_fence_after();
                if (any_rows) {
                    const uint32_t t_s = t_s0 + st * kN + col0;
                    const int tc0 = t0 + col0;
                    const uint64_t flags = *reinterpret_cast<const uint64_t *>(sc_ok[ring]);
                    const bool blocks_ok =
                        C::kTwo ? flags == 0x0101010101010101ull : static_cast<uint32_t>(flags >> (4 * col0 / 8)) == 0x01010101u;
                    const bool full =
                        __all_sync(0xffffffffu, !row_on || (blocks_ok && lo <= tc0 && tc0 + kCols <= hi));
                    constexpr int kCh = C::kChunk, kB = kCh / 16;
                    // kChunk columns: scores and their factors; in partly seen units the masked products with factors of 1
                    auto scores = [&](int x, float (&s)[kCh], float (&cf)[kB], float (&lv)[kB]) {
                        tmem_ld32_async(t_s + kCh * x, s);
                        if constexpr (kCh == 64) tmem_ld32_async(t_s + kCh * x + 32, s + 32);
#pragma unroll
                        for (int b = 0; b < kB; ++b) {
                            cf[b] = factor * sc_k[ring][col0 / 16 + kB * x + b];
                            lv[b] = sc_v[ring][col0 / 16 + kB * x + b];
                        }
                        tmem_ld_wait(s);
                        if (!full) {
                            const int at = tc0 + kCh * x;
#pragma unroll
                            for (int b = 0; b < kB; ++b) {
                                const bool on = sc_ok[ring][col0 / 16 + kB * x + b] != 0;
#pragma unroll
                                for (int i = 16 * b; i < 16 * b + 16; ++i)
                                    s[i] = on && at + i >= lo && at + i < hi ? s[i] * cf[b] : -kInf;
                                cf[b] = 1.0f;
                            }
                        }
                    };
                    // their maxima: of the scores, and with log2 of the value scales
                    auto maxima = [&](const float (&s)[kCh], const float (&cf)[kB], const float (&lv)[kB], float &mn, float &vn) {
#pragma unroll
                        for (int b = 0; b < kB; ++b) {
                            const float *y = s + 16 * b;
                            float a0 = max3(y[0], y[1], y[2]), a1 = max3(y[3], y[4], y[5]);
                            a0 = max3(a0, y[6], y[7]), a1 = max3(a1, y[8], y[9]);
                            a0 = max3(a0, y[10], y[11]), a1 = max3(a1, y[12], y[13]);
                            const float t = fmaxf(max3(a0, y[14], y[15]), a1) * cf[b];
                            mn = fmaxf(mn, t);
                            vn = fmaxf(vn, t + lv[b]);
                        }
                    };
                    // P of kChunk columns, and their sum
                    auto weigh = [&](int x, const float (&s)[kCh], const float (&cf)[kB], const float (&lv)[kB]) {
                        const float mb = finite_or_0(m), rb = finite_or_0(mref);
                        const F2 nm = f2(-mb, -mb);
                        F2 sum[kB];
                        uint32_t pk[kCh / 2];
#pragma unroll
                        for (int b = 0; b < kB; ++b) {
                            const float wv = ex2(fminf(lv[b] + mb - rb + kLift, 126.f));
                            const F2 w2 = f2(wv, wv), c2 = f2(cf[b], cf[b]);
                            sum[b] = f2(0.f, 0.f);
#pragma unroll
                            for (int i = 16 * b; i < 16 * b + 16; i += 2) {
                                float e0, e1;
                                un2(fma2(f2(s[i], s[i + 1]), c2, nm), e0, e1);
                                const F2 e = f2(ex2(e0), ex2(e1));
                                sum[b] = add2(sum[b], e);
                                un2(mul2(e, w2), e0, e1);
                                pk[i / 2] = pack(e0, e1, __half());
                            }
                        }
                        float s0, s1;
                        F2 all = add2(sum[0], sum[1]);
                        if constexpr (kB == 4) all = add2(all, add2(sum[2], sum[3]));
                        un2(all, s0, s1);
                        l += s0 + s1;
                        tmem_st(t_s + kCh / 2 * x, pk);  // over columns that have been read
                    };
                    // m and mref move to mn and vn for the rows in which either grows by more than kRescale (P and the
                    // terms of l stay below 2^15); what was formed with the old ones follows: l, O, and P of `done` chunks
                    // of this unit.  O must hold P V of all this tile's units so far: with one S stage S of this unit was
                    // issued after them.
                    auto move_to = [&](float mn, float vn, int done) -> bool {
                        const bool move = mn > m + kRescale || vn > mref + kRescale || (m == -kInf && mn > -kInf);
                        if (!__any_sync(0xffffffffu, move)) return true;
                        float fl = 1.0f, fo = 1.0f;
                        if (move) {
                            const float m2 = fmaxf(m, mn), r2 = fmaxf(mref, vn);
                            fl = ex2(m - finite_or_0(m2));
                            fo = ex2(mref - finite_or_0(r2));
                            m = m2;
                            mref = r2;
                        }
                        l *= fl;
                        if (begun) {
                            if constexpr (!C::kTwo) {
                                if (!warp_wait(&pv_done[tg][st ^ 1], (uses >> (st ^ 1) & 1u) ^ 1u)) return false;
                                tc::tc_fence_after();
                            }
                            constexpr int kOc = C::kTwo ? HD : HD / 2;
#pragma unroll 1
                            for (int x = 0; x < kOc; x += 32) {
                                uint32_t o[32];
                                const uint32_t at = t_o + (C::kTwo ? 0 : wg * kOc) + x;
                                tc::tmem_ld32(at, o);
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fo);
                                tc::tmem_st32(at, o);
                            }
                        }
                        if constexpr (C::kTwo) {
#pragma unroll 1
                            for (int x = 0; x < done; ++x) {
                                uint32_t o[32];
                                tc::tmem_ld32(t_s + 32 * x, o);
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&o[i]));
                                    o[i] = pack(f.x * fo, f.y * fo, __half());
                                }
                                tc::tmem_st32(t_s + 32 * x, o);
                            }
                        }
                        return true;
                    };
                    if constexpr (C::kTwo) {  // one pass, chunk by chunk
#pragma unroll 1
                        for (int x = 0; x < kCols / kCh; ++x) {
                            float s[kCh], cf[kB], lv[kB], mn = -kInf, vn = -kInf;
                            scores(x, s, cf, lv);
                            maxima(s, cf, lv, mn, vn);
                            move_to(mn, vn, x);
                            weigh(x, s, cf, lv);
                        }
                    } else {  // the maxima first: the other half's columns share O's scale
                        float mn = -kInf, vn = -kInf;
#pragma unroll 1
                        for (int x = 0; x < kCols / kCh; ++x) {
                            float s[kCh], cf[kB], lv[kB];
                            scores(x, s, cf, lv);
                            maxima(s, cf, lv, mn, vn);
                        }
                        xch[st][wg][r] = make_float2(mn, vn);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&pair_bar[warp & 3][st]);
                        ok = warp_wait(&pair_bar[warp & 3][st], met >> st & 1u);
                        if (!ok) break;
                        met ^= 1u << st;  // not `uses`: a warp without rows in an item exchanges nothing
                        const float2 o = xch[st][wg ^ 1][r];
                        ok = move_to(fmaxf(mn, o.x), fmaxf(vn, o.y), 0);
                        if (!ok) break;
#pragma unroll 1
                        for (int x = 0; x < kCols / kCh; ++x) {
                            float s[kCh], cf[kB], lv[kB];
                            scores(x, s, cf, lv);
                            weigh(x, s, cf, lv);
                        }
                    }
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
            if constexpr (!C::kTwo) {  // the two halves' sums
                xch[i_at & 1][wg][r] = make_float2(l, 0.f);
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_pair[warp & 3]);
                ok = warp_wait(&q_pair[warp & 3], i_at & 1u);
                if (!ok) break;
                l = xch[i_at & 1][0][r].x + xch[i_at & 1][1][r].x;
            }
            if (any_rows) {
                const int slot = d->slot;
                const bool whole = slot < 0;
                const float f = l == 0.f || !begun ? 0.f : ex2(finite_or_0(mref) - finite_or_0(m)) * kUnlift / l;
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
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] *= f;
                    if (row_on && whole) {
                        uint4 *d4 = reinterpret_cast<uint4 *>(dst + x);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            d4[i] = make_uint4(pack(o[8 * i], o[8 * i + 1], T()), pack(o[8 * i + 2], o[8 * i + 3], T()),
                                               pack(o[8 * i + 4], o[8 * i + 5], T()), pack(o[8 * i + 6], o[8 * i + 7], T()));
                    } else if (row_on) {
                        float4 *d4 = reinterpret_cast<float4 *>(p.part.o + at * HD + x);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            d4[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                    __syncwarp();  // the TMEM loads are warp-wide
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
    return e != cudaSuccess ? e : launch_behind(kv8_prompt_kernel<HD, T>, dim3(ctas), kThreads, Cfg<HD>::kSmem, s, p);
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
