// kv8_prompt.cu -- mg_kv8_attention for many query rows per kv head (prompts,
// prompt chunks, drafts of several tokens): the 5th-generation tensor cores on
// the 8-bit paged cache.
//
// An item is a tile of 128 query rows ((token, q head of the group) pairs of
// one kv head); its keys run in tiles of 64 tokens.  Both products are
// tcgen05.mma kind::f16 with fp32 accumulators in TMEM:
//   S [128 x 64] = Q . K^T        Q and K fp16 in shared memory, K-major
//   O [128 x hd] += P . V         P fp16 in TMEM (over S), V fp16 MN-major
// The cache's codes are widened to fp16, which is exact, on their way into
// shared memory; q is brought into fp16's range by a power of two per row.  The
// block scales of K multiply the score columns, those of V ride in P's
// exponent: with s = scale log2(e) k_scale <q, k>, m = max s and
// M = max(s + log2 v_scale), P = 2^(s + log2 v_scale - M) and l = sum 2^(s - m),
// so P is bounded whatever the scales and fp16 holds it to 2^-12.
//
// Warps of a CTA (288 threads):
//  * warps 0-3: softmax, one row per thread (TMEM lane = row); they also bring
//    the item's Q tile into shared memory and write the answer;
//  * warps 4-7: loaders -- codes from the pages into registers one tile ahead,
//    widened and stored in the 128-byte swizzled layout (token rows of 64
//    dims); tokens that are not seen become zeros, so that stale codes behind
//    the context cannot reach a product;
//  * warp 8: allocates TMEM; one lane issues the MMAs: S of tile j + 1 before
//    P V of tile j, so that it runs under the softmax of tile j.
// K, V and S have two stages.  P overwrites the S stage it was made from; the
// tensor pipe runs one thread's MMAs in order, so S of tile j + 2 lands after
// P V of tile j has read it.  O is rescaled only when M grows by more than 2^8
// (P stays below 2^8, exact in fp16's range).
//
// Every wait is bounded; on expiry the kernel records kErrWait, every role
// leaves its loop, TMEM is freed and the kernel returns.
#include <cstdio>

#include "kv8.cuh"
#include "tc_common.cuh"

namespace mg {
namespace kv8 {
namespace {
constexpr int kM = 128;   // rows of an item
constexpr int kN = kUnit; // tokens of a tile
constexpr int kThreads = 288;
constexpr uint32_t kErrWait = 0x90000u;
constexpr float kInf = __builtin_huge_valf();
constexpr float kRescale = 8.0f;

template <int HD>
struct Cfg {
    static constexpr int kAtoms = HD / 64;
    static constexpr uint32_t kQBytes = kM * HD * 2, kTileBytes = kN * HD * 2;
    static constexpr uint32_t kTmem = HD == 256 ? 512 : 256;  // O: HD columns, S: 2 x 64
    static constexpr int kPerSm = HD == 256 ? 1 : 2;
    static constexpr size_t kSmem = 1024 + kQBytes + 4 * kTileBytes;
};

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
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    tc::umma_bf16(d, a, b, idesc, acc);  // kind::f16; the operand types are the descriptor's
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %3, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %4, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(acc), "r"(idesc)
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
        if (mbar_try_wait_sleep(bar, parity, kMbarSleepNs)) return true;
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
    __device__ __forceinline__ int tile_token(int j) const { return (it.unit0 + skip + j) * kN; }
};

template <int HD, typename T>
__global__ void __launch_bounds__(kThreads, Cfg<HD>::kPerSm) kv8_prompt_kernel(const AttnArgs p) {
    using C = Cfg<HD>;
    constexpr int kAtoms = C::kAtoms;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t k_full[2], k_empty[2], v_full[2], pv_done[2], s_full[2], p_full[2], sc_full[4], q_full;
    __shared__ float sc_k[4][4], sc_v[4][4];  // scales of a tile's four blocks: K, log2 of V
    __shared__ int sc_ok[4][4];
    __shared__ float q_down[kM];
    __shared__ uint32_t tmem_slot;
    __shared__ int stop_s;
    volatile int *stop = &stop_s;
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
            mbar_init(&pv_done[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&sc_full[i], 4);
        mbar_init(&q_full, 4);
        stop_s = 0;
        p.part.split[cta].nrows = 0;
        fence_barrier_init();
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(C::kTmem)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const Place pl = find_place<kThreads>(p.b, p.a, p.c.heads, cta, gridDim.x);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = tmem_slot, t_o = tmem, t_s0 = tmem + HD;
    Walk wk;
    bool more = wk.start(p, pl);

    if (warp == 8) {
        if (lane == 0) {  // ---- MMA issuer
            constexpr uint32_t kIdS = idesc_f16(kM, kN, 0), kIdO = idesc_f16(kM, HD, 1);
            uint32_t n = 0, items = 0;  // tiles and items so far
            auto issue_s = [&](uint32_t j) -> bool {
                const uint32_t st = j & 1;
                if (!wait(&k_full[st], (j >> 1) & 1u, stop, p.b.err)) return false;
                tc::tc_fence_after();
                const uint32_t kb = sk + st * C::kTileBytes;
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk)
                    umma_ss(t_s0 + st * kN, tc::sw128_desc(sq + (kk >> 2) * kM * 128 + (kk & 3) * 32),
                            tc::sw128_desc(kb + (kk >> 2) * kN * 128 + (kk & 3) * 32), kIdS, kk > 0 ? 1u : 0u);
                tc::umma_commit(smem_u32(&s_full[st]));
                tc::umma_commit(smem_u32(&k_empty[st]));
                return true;
            };
            bool ok = true;
            while (ok && more) {
                ok = wait(&q_full, items & 1u, stop, p.b.err) && issue_s(n);
                const int take = wk.take;
                for (int j = 0; ok && j < take; ++j, ++n) {
                    if (j + 1 < take && !issue_s(n + 1)) {
                        ok = false;
                        break;
                    }
                    const uint32_t st = n & 1, ph = (n >> 1) & 1u;
                    if (!wait(&p_full[st], ph, stop, p.b.err) || !wait(&v_full[st], ph, stop, p.b.err)) {
                        ok = false;
                        break;
                    }
                    tc::tc_fence_after();
                    const uint32_t vb = sv + st * C::kTileBytes;
#pragma unroll
                    for (int kk = 0; kk < kN / 16; ++kk)
                        umma_ts(t_o, t_s0 + st * kN + kk * 8, sw128_mn_desc(vb + kk * 2048, kN * 128), kIdO,
                                (j | kk) != 0 ? 1u : 0u);
                    tc::umma_commit(smem_u32(&pv_done[st]));
                }
                ++items;
                more = wk.next(p);
            }
        }
    } else if (warp >= 4) {  // ---- loaders
        const int u = threadIdx.x - 128, quad = u >> 2, sub = u & 3;
        // a tile's page ids, read one tile before its codes
        struct Ref {
            int tok0, lo, hi, head, page[2];  // page -2: no position that a row sees
        } ref;
        int j = 0;  // tile of the item that `ref` names
        auto look = [&]() {
            ref.tok0 = wk.tile_token(j);
            ref.lo = wk.it.lo & ~(kBlock - 1);  // pages before a window may be gone
            ref.hi = wk.it.hi;
            ref.head = wk.head;
            const int32_t *table = p.b.table + (wk.pair / p.a.tiles) * p.b.table_stride;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int tok = ref.tok0 + quad + 32 * i;
                ref.page[i] = -2;
                if (tok >= ref.lo && tok < ref.hi) {
                    ref.page[i] = table[tok >> p.c.page_shift];
                    if (ref.page[i] < 0 || ref.page[i] >= p.c.num_pages) {
                        set_error(p.b.err, kErrPage);
                        ref.page[i] = -2;
                    }
                }
            }
        };
        auto advance = [&]() {
            if (++j == wk.take) {
                j = 0;
                more = wk.next(p);
            }
            if (more) look();
        };
        uint4 kr[2][kAtoms], vr[2][kAtoms];
        float ks[2], vs[2];
        int okb[2];
        const uint8_t *vsrc[2];
        auto fetch_k = [&]() {  // resolves ref; V follows from vsrc
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int page = ref.page[i];
                const bool on = page >= 0;
                const int tok = ref.tok0 + quad + 32 * i, slot = tok & ((1 << p.c.page_shift) - 1);
                const int64_t at = page * p.c.page_stride + ref.head * p.c.head_stride + slot * p.c.token_stride + 16 * sub;
                vsrc[i] = on ? p.c.v + at : nullptr;
#pragma unroll
                for (int a = 0; a < kAtoms; ++a) kr[i][a] = on ? ldg16(p.c.k + at + 64 * a) : make_uint4(0, 0, 0, 0);
                if (sub == 0 && (quad & 15) == 0) {
                    const int64_t sc = ((static_cast<int64_t>(page) * p.c.heads + ref.head) << (p.c.page_shift - 4)) +
                                       (slot >> 4);
                    ks[i] = on ? p.c.k_scale[sc] : 1.f;
                    vs[i] = on ? p.c.v_scale[sc] : 1.f;
                    okb[i] = on ? 1 : 0;
                }
            }
        };
        auto fetch_v = [&]() {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int a = 0; a < kAtoms; ++a) vr[i][a] = vsrc[i] ? ldg16(vsrc[i] + 64 * a) : make_uint4(0, 0, 0, 0);
        };
        // 16 codes -> two 16-byte chunks of the token's 128-byte row, swizzled
        auto put = [&](unsigned char *tile, const uint4 (&r)[2][kAtoms]) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = quad + 32 * i;
#pragma unroll
                for (int a = 0; a < kAtoms; ++a) {
                    uint4 lo, hi;
                    e4m3x4_to_h2x2(r[i][a].x, lo.x, lo.y);
                    e4m3x4_to_h2x2(r[i][a].y, lo.z, lo.w);
                    e4m3x4_to_h2x2(r[i][a].z, hi.x, hi.y);
                    e4m3x4_to_h2x2(r[i][a].w, hi.z, hi.w);
                    unsigned char *dst = tile + a * kN * 128 + row * 128;
                    *reinterpret_cast<uint4 *>(dst + (((2 * sub) ^ (row & 7)) << 4)) = lo;
                    *reinterpret_cast<uint4 *>(dst + (((2 * sub + 1) ^ (row & 7)) << 4)) = hi;
                }
            }
        };
        unsigned char *gk = gen + C::kQBytes, *gv = gk + 2 * C::kTileBytes;
        if (more) {
            look();
            fetch_k();
            fetch_v();
            advance();
        }
        const uint32_t tiles = static_cast<uint32_t>(pl.w1 - pl.w0);
        for (uint32_t n = 0; n < tiles; ++n) {
            const uint32_t st = n & 1, prev = ((n >> 1) - 1) & 1u;
            if (n >= 2 && !__all_sync(0xffffffffu, wait(&k_empty[st], prev, stop, p.b.err))) break;
            put(gk + st * C::kTileBytes, kr);
            if (sub == 0 && (quad & 15) == 0) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int b = (quad >> 4) + 2 * i;
                    sc_k[n & 3][b] = ks[i];
                    sc_v[n & 3][b] = __log2f(vs[i]);
                    sc_ok[n & 3][b] = okb[i];
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sc_full[n & 3]);
                mbar_arrive(&k_full[st]);
            }
            if (n + 1 < tiles) fetch_k();
            if (n >= 2 && !__all_sync(0xffffffffu, wait(&pv_done[st], prev, stop, p.b.err))) break;
            put(gv + st * C::kTileBytes, vr);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[st]);
            if (n + 1 < tiles) {
                fetch_v();
                advance();
            }
        }
    } else {  // ---- softmax: thread = row
        const int r = threadIdx.x;
        const uint32_t lane_off = static_cast<uint32_t>(warp * 32) << 16;
        uint32_t n = 0;
        bool ok = true;
        while (more) {
            const Item it = wk.it;
            const bool any_rows = warp * 32 < it.nrows;
            // Q: a warp brings its 32 rows, lane d with HD / 32 values; the largest becomes 2^7 .. 2^8
            constexpr int kW = HD / 64;  // 32-bit words of a lane
            if (any_rows) {
#pragma unroll 1
                for (int r0 = 0; r0 < 32; r0 += 8) {
                    uint32_t q[8][kW];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int row = it.row0 + warp * 32 + r0 + i;
                        const bool on = warp * 32 + r0 + i < it.nrows;
                        const int tok = on ? row / p.a.group : 0;
                        const int h = wk.head * p.a.group + (on ? row - tok * p.a.group : 0);
                        const T *src = static_cast<const T *>(p.q) + (static_cast<int64_t>(it.seq.q0) + tok) * p.q_row +
                                       h * p.q_head + lane * 2 * kW;
#pragma unroll
                        for (int w = 0; w < kW; ++w) q[i][w] = 0;
                        if (on) {
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
                    for (int i = 0; i < 8; ++i) {
                        const int lr = warp * 32 + r0 + i;
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
                        unsigned char *dst = gen + atom * kM * 128 + lr * 128 + ((chunk ^ (lr & 7)) << 4) + in;
                        if constexpr (kW == 1) *reinterpret_cast<uint32_t *>(dst) = hw[0];
                        else if constexpr (kW == 2) *reinterpret_cast<uint2 *>(dst) = make_uint2(hw[0], hw[1]);
                        else *reinterpret_cast<uint4 *>(dst) = make_uint4(hw[0], hw[1], hw[2], hw[3]);
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full);
            const float factor = any_rows ? fabsf(p.scale_log2) * q_down[r] : 0.f;
            const bool row_on = r < it.nrows;
            const int pos = it.seq.pos0 + (it.row0 + r) / p.a.group;
            const int hi = row_on ? pos + 1 : 0, lo = p.a.window > 0 ? pos - p.a.window + 1 : 0;

            float m = -kInf, mref = -kInf, l = 0.f;
            for (int j = 0; j < wk.take; ++j, ++n) {
                const uint32_t st = n & 1, ph = (n >> 1) & 1u;
                ok = wait(&sc_full[n & 3], (n >> 2) & 1u, stop, p.b.err) && wait(&s_full[st], ph, stop, p.b.err);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                tc::tc_fence_after();
                if (any_rows) {
                    const uint32_t t_s = t_s0 + st * kN + lane_off;
                    float s[kN];
                    tmem_ld32_async(t_s, s);
                    tmem_ld32_async(t_s + 32, s + 32);
                    float c[4], lv[4];
                    bool blocks_ok = true;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        c[b] = factor * sc_k[n & 3][b];
                        lv[b] = sc_v[n & 3][b];
                        blocks_ok = blocks_ok && sc_ok[n & 3][b] != 0;
                    }
                    tmem_ld_wait(s);
                    const int t0 = wk.tile_token(j);
                    const bool all = !row_on || (blocks_ok && lo <= t0 && t0 + kN <= hi);
                    if (!__all_sync(0xffffffffu, all)) {
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            const bool okb = sc_ok[n & 3][b] != 0;
#pragma unroll
                            for (int i = 16 * b; i < 16 * b + 16; ++i)
                                s[i] = okb && t0 + i >= lo && t0 + i < hi ? s[i] * c[b] : -kInf;
                            c[b] = 1.0f;
                        }
                    }
                    float mn = m, vn = -kInf;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        float t = s[16 * b];
#pragma unroll
                        for (int i = 1; i < 16; ++i) t = fmaxf(t, s[16 * b + i]);
                        t *= c[b];
                        mn = fmaxf(mn, t);
                        vn = fmaxf(vn, t + lv[b]);
                    }
                    const float mb = mn == -kInf ? 0.f : mn;
                    l *= ex2(m - mb);
                    m = mn;
                    const bool move = vn > mref + kRescale || (mref == -kInf && vn > -kInf);
                    const float old = mref;
                    if (move) mref = vn;
                    const float rb = mref == -kInf ? 0.f : mref;
                    if (j > 0 && __any_sync(0xffffffffu, move)) {
                        // O holds P V of the tiles up to j - 1 once that of j - 1 is done
                        ok = wait(&pv_done[(n - 1) & 1], ((n - 1) >> 1) & 1u, stop, p.b.err);
                        if (!__all_sync(0xffffffffu, ok)) {
                            ok = false;
                            break;
                        }
                        tc::tc_fence_after();
                        const float f = move ? ex2(old - rb) : 1.0f;
#pragma unroll 1
                        for (int x = 0; x < HD / 32; ++x) {
                            uint32_t o[32];
                            tc::tmem_ld32(t_o + lane_off + 32 * x, o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tc::tmem_st32(t_o + lane_off + 32 * x, o);
                        }
                    }
                    uint32_t pk[kN / 2];
                    float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const float wv = ex2(fminf(lv[b] + mb - rb, 126.f));
#pragma unroll
                        for (int i = 16 * b; i < 16 * b + 16; i += 2) {
                            const float e0 = ex2(fmaf(s[i], c[b], -mb)), e1 = ex2(fmaf(s[i + 1], c[b], -mb));
                            sum0 += e0;
                            sum1 += e1;
                            pk[i / 2] = pack(e0 * wv, e1 * wv, __half());
                        }
                    }
                    l += sum0 + sum1;
                    tc::tmem_st32(t_s, pk);
                }
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[st]);
            }
            if (!ok) break;
            ok = wait(&pv_done[(n - 1) & 1], ((n - 1) >> 1) & 1u, stop, p.b.err);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc::tc_fence_after();
            const bool whole = wk.take == it.units;
            const int slot = 2 * cta + (wk.first ? 0 : 1);
            if (any_rows) {
                const float f = l == 0.f ? 0.f : ex2((mref == -kInf ? 0.f : mref) - (m == -kInf ? 0.f : m)) / l;
                const int row = it.row0 + r, tok = row / p.a.group, hq = wk.head * p.a.group + row - tok * p.a.group;
                T *dst = static_cast<T *>(p.out) + (static_cast<int64_t>(it.seq.q0) + tok) * p.out_row + hq * p.out_head;
                const int64_t at = static_cast<int64_t>(slot) * kM + r;
                if (!whole && row_on) *reinterpret_cast<float2 *>(p.part.ml + 2 * at) = make_float2(m, l);
#pragma unroll 1
                for (int x = 0; x < HD / 32; ++x) {
                    float o[32];
                    tmem_ld32_async(t_o + lane_off + 32 * x, o);
                    tmem_ld_wait(o);
                    if (!row_on) continue;
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] *= f;
                    if (whole) {
                        uint4 *d4 = reinterpret_cast<uint4 *>(dst + 32 * x);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            d4[i] = make_uint4(pack(o[8 * i], o[8 * i + 1], T()), pack(o[8 * i + 2], o[8 * i + 3], T()),
                                               pack(o[8 * i + 4], o[8 * i + 5], T()), pack(o[8 * i + 6], o[8 * i + 7], T()));
                    } else {
                        float4 *d4 = reinterpret_cast<float4 *>(p.part.o + at * HD + 32 * x);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            d4[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
            }
            if (threadIdx.x == 0 && wk.skip == 0 && !whole)
                p.part.split[cta] =
                    Split{wk.pair, wk.head, it.nrows, slot, owner_of(pl, wk.w + it.units - 1), {0, 0, 0}};
            tc::tc_fence_before();
            more = wk.next(p);
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc::tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmem));
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

int prompt_ctas_per_sm(int hd) { return hd == 256 ? Cfg<256>::kPerSm : Cfg<128>::kPerSm; }

cudaError_t launch_prompt(const AttnArgs &p, int hd, bool f16, int ctas, cudaStream_t s) {
    if (hd == 64) return f16 ? launch<64, __half>(p, ctas, s) : launch<64, __nv_bfloat16>(p, ctas, s);
    if (hd == 128) return f16 ? launch<128, __half>(p, ctas, s) : launch<128, __nv_bfloat16>(p, ctas, s);
    return f16 ? launch<256, __half>(p, ctas, s) : launch<256, __nv_bfloat16>(p, ctas, s);
}

}  // namespace kv8
}  // namespace mg
