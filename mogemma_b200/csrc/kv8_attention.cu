// kv8_attention.cu -- mg_kv8_attention: attention over the 8-bit paged cache
// (the attention of layers.mojo:63-94), for few query rows per kv head; the
// combine of partial answers; and the entry points.
//
// kv8_rows_kernel takes items of up to 8 or 16 query rows.  It is bound by
// reading the cache: one code byte feeds few rows' products, so the legacy
// warp-level MMA is fast enough.  A warp takes 16 tokens (one scale block) at a time and
// computes transposed products, tokens and head dims on the MMA's 16 rows, the
// query rows on its 8 columns:
//   S^T[16 tokens][8 rows] = K . Q^T     A = K codes, widened to fp16 (exact)
//   O^T[16 dims][8 rows]  += V^T . P^T   A = V codes of 4 tokens a lane,
//                                        byte-interleaved, widened to fp16
// The k index of an MMA may be any order of the head dims as long as A and B
// agree, so a lane's K fragment is 16 consecutive bytes of a token's row, and
// the m index any order of the output dims, so its V fragment is too.
// S^T's accumulator layout transposes into P^T's operand layout by movmatrix.
//
// Every warp has a ring of its own in shared memory, filled by asynchronous
// 16-byte copies kStages - 1 steps (8 KB each, hd 64: 4 KB) ahead, and nothing
// but its own copies to wait for; token rows are padded by 16 bytes, so that the fragments'
// loads meet no bank twice.  With the codes in registers instead, one step
// ahead, 64 KB per SM at most were in flight: 4.3 TB/s on 1.37 GB of cache
// where the ring reaches 5.8.
//
// Measured (in a graph, with the combine): 32 tokens over 4096 to 16384 positions
// each, 10.4 thousand on average, 32 / 16 heads of 128, 226 to 236 us, 5.8 to 6.1
// TB/s (255 us, 5.4 TB/s, call by call); one token over 131072 positions, 4 / 1
// heads of 256, 24 us, 2.8 TB/s; one over 640 positions, 10 us, which is latency
// alone: two launches, the scan for a CTA's place, the page look-up, two steps
// and the join.
//
// With s = scale log2(e) k_scale <q, k> the state per row is m = max s,
// l = sum 2^(s - m) and the sum of P V with P = 2^(s + log2 v_scale - M + 15),
// M = max(s + log2 v_scale): the value scale rides in the exponent, so that P
// is at most 2^15 whatever the scales.  P is fp16 because it is an MMA operand:
// held to 2^-11 of itself down to 2^-29 of the row's largest, below that to
// 2^-40 of the largest, where a term also ends.  (With a largest P of 1 a long
// tail of weights at 2^-25 of one token's, 0.4 % of a softmax over 131072
// positions, was lost from the sum of P V while l counted it.)
#include <cfloat>
#include <cmath>
#include <cstdio>
#include <type_traits>

#include "kv8.cuh"

namespace mg {
namespace kv8 {

mg_status check_cache_batch(const char *who, const mg_kv8_cache *c, const mg_kv8_batch *b);
Cache cache_of(const mg_kv8_cache *c);
Batch batch_of(const mg_kv8_batch *b);
// kv8_prompt.cu
constexpr int kPromptUnit = 128;
// What an item's start and end cost, in units: with 0, 3, 6 the 27B prompt takes 322, 270, 282 us, chunks of 512 and 365
// tokens at 8192 and 5844 positions (hd 256) 105, 97, 101, ragged prompts of hd 64 41.8, 39.4, 41.4, two prompts of 300
// tokens 23.4 each.
constexpr int kPromptExtra = 3;
int prompt_rows(int hd);
cudaError_t launch_prompt(const AttnArgs &p, int hd, bool f16, int ctas, cudaStream_t s);

namespace {
constexpr int kRows = 8;       // query rows of an MMA; an item has 8 or 16
constexpr int kUnit = 64;      // tokens of a unit of the schedule
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr float kLift = 15.0f;  // log2 of a row's largest P: 2^15 is the largest power of two in fp16
constexpr float kUnlift = 1.0f / 32768.0f;  // 2^-kLift; apart from ex2, which ends at 2^-126: value scales may be as small

// D += A . B, 16 x 8 x 16, fp16 operands, fp32 accumulators.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void store_out4(__half *p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack(a, b, __half()), pack(c, d, __half()));
}
__device__ __forceinline__ void store_out4(__nv_bfloat16 *p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack(a, b, __nv_bfloat16()), pack(c, d, __nv_bfloat16()));
}
__device__ __forceinline__ float max_over_rows(float v) {  // over the 8 lanes that share lane % 4
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

template <int HD>
struct RowsCfg {
    static constexpr int kTiles = HD == 256 ? 1 : 2;    // 16-token tiles of a warp's step
    static constexpr int kVB = HD / 8 < 16 ? HD / 8 : 16;  // V bytes per load: 8 (hd 64) or 16
    static constexpr int kVH = HD / (8 * kVB);          // loads along the head dims
    static constexpr int kM = HD / 16;                  // MMAs along the output dims
    static constexpr int kRow = HD + 16;                // bytes of a token's padded row
    static constexpr int kStep = 2 * kTiles * 16 * kRow;  // K rows, then V rows
    static constexpr int kStages = HD == 64 ? 5 : 3;    // 100 to 110 KB for four warps: two CTAs per SM
    static constexpr size_t kSmem = static_cast<size_t>(kWarps) * kStages * kStep;
    static_assert(sizeof(float) * 2 * kRows * (HD + 4) <= kStages * kStep, "the merge takes the place of a warp's ring");
};

// 16 bytes to shared memory, asynchronously; zeros where !on.
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t *src, bool on) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {  // all but the latest N groups have landed
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// A tile's 16 token rows (K or V) of which the first `live` are real.
template <int HD>
__device__ __forceinline__ void copy_tile(uint32_t dst, const uint8_t *tile, int64_t stride, int live, int lane) {
    constexpr int kChunks = HD / 16, kRowsAt = 32 / kChunks;  // 16-byte chunks of a row; rows per pass of the warp
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += kRowsAt) {
        const int r = r0 + lane / kChunks, c = lane % kChunks;
        const bool on = r < live;
        copy16(dst + r * RowsCfg<HD>::kRow + 16 * c, on ? tile + r * stride + 16 * c : tile, on);
    }
}

template <int HD, int NT, typename T>  // NT: 8-row tiles of an item
__global__ void __launch_bounds__(kThreads) kv8_rows_kernel(const AttnArgs p) {
    using Cfg = RowsCfg<HD>;
    extern __shared__ __align__(16) unsigned char smem[];  // rings by warp; at an item's end [row][HD + 4] floats each
    __shared__ float mlm[kWarps][NT * kRows][3];
    kernel_begins();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int cta = blockIdx.x, ctas = gridDim.x;
    unsigned char *ring = smem + warp * Cfg::kStages * Cfg::kStep;
    const uint32_t ring_s = smem_u32(ring);
    constexpr int kMerge = Cfg::kStages * Cfg::kStep / 4;  // floats from one warp's merge rows to the next's
    const Place pl = find_place<kThreads>(p.b, p.a, p.c.heads, cta, ctas);
    if (threadIdx.x == 0) p.part.split[cta].nrows = 0;
    Walk wk;
    for (bool more = wk.start(p.b, p.a, pl); more; more = wk.next(p.b, p.a)) {
        const Item &it = wk.it;
        const int head = wk.head, pair = wk.pair;
        const bool whole = wk.whole();
        // this CTA's 16-token tiles of the item
        const int ta = max((it.unit0 + wk.first) * (kUnit / 16), it.lo / 16);
        const int tb = min((it.unit0 + wk.first + wk.take) * (kUnit / 16), (it.hi + 15) / 16);
        const int si = pair / p.a.tiles;
        const int32_t *table = p.b.table + si * p.b.table_stride;

        // ---- the warp's tiles, kTiles neighbours per step: its n-th is ta + ((n / kTiles) kWarps + warp) kTiles + n % kTiles
        auto tile_at = [&](int n) { return ta + ((n / Cfg::kTiles) * kWarps + warp) * Cfg::kTiles + n % Cfg::kTiles; };
        // lane i holds the place and scales of tile number base + i (place -1: none), and the scales of the 32 before
        int64_t place = -1;
        float ks = 0.f, lvs = 0.f, ks_old = 0.f, lvs_old = 0.f;
        uint32_t there = 0, there_old = 0;  // bit i: tile number base + i has a place
        auto look_up = [&](int base) {
            const int tile = tile_at(base + lane);
            place = -1;
            ks_old = ks;
            lvs_old = lvs;
            there_old = there;
            ks = 0.f;
            lvs = 1.f;
            if (tile < tb) {
                const int tok = tile * 16, slot = tok & ((1 << p.c.page_shift) - 1);
                const int page = table[tok >> p.c.page_shift];
                if (page >= 0 && page < p.c.num_pages) {
                    const int64_t sc = ((static_cast<int64_t>(page) * p.c.heads + head) << (p.c.page_shift - 4)) +
                                       (slot >> 4);
                    place = page * p.c.page_stride + head * p.c.head_stride + slot * p.c.token_stride;
                    ks = p.c.k_scale[sc];
                    lvs = p.c.v_scale[sc];
                } else {
                    set_error(p.b.err, kErrPage);
                }
            }
            there = __ballot_sync(0xffffffffu, place >= 0);
        };
        const int steps = (tb - ta + kWarps * Cfg::kTiles - 1) / (kWarps * Cfg::kTiles);
        // A step's copies; the scales, read along with the places, have until the step is worked on to arrive.
        auto fetch = [&](int step, int stage) {
            if (step < steps) {
                const int n0 = step * Cfg::kTiles;
                if ((n0 & 31) == 0) look_up(n0);
#pragma unroll
                for (int i = 0; i < Cfg::kTiles; ++i) {
                    const int64_t at = __shfl_sync(0xffffffffu, place, (n0 + i) & 31);
                    const int live = at < 0 ? 0 : it.hi - tile_at(n0 + i) * 16;
                    const int64_t src = at < 0 ? 0 : at;
                    const uint32_t dst = ring_s + stage * Cfg::kStep + i * 16 * Cfg::kRow;
                    copy_tile<HD>(dst, p.c.k + src, p.c.token_stride, live, lane);
                    copy_tile<HD>(dst + Cfg::kTiles * 16 * Cfg::kRow, p.c.v + src, p.c.token_stride, live, lane);
                }
            }
            copies_commit();  // an empty group past the end: the count of groups stays that of steps
        };
#pragma unroll
        for (int i = 0; i < Cfg::kStages - 1; ++i) fetch(i, i);

        // ---- query rows: B fragments, row g, k order as the K fragments
        uint32_t qf[NT][HD / 64][4][2];
        float factor[NT][2];
        int lo[NT][2], hi[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = it.row0 + nt * kRows + g;
            const bool on = nt * kRows + g < it.nrows;
            const int tok = on ? r / p.a.group : 0, h = head * p.a.group + (on ? r - tok * p.a.group : 0);
            const T *src = static_cast<const T *>(p.q) + (static_cast<int64_t>(it.seq.q0) + tok) * p.q_row +
                           h * p.q_head + 16 * t;
            uint32_t raw[HD / 64][8];
            uint32_t most = 0;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint4 v = on ? reinterpret_cast<const uint4 *>(src + 64 * c)[i] : make_uint4(0, 0, 0, 0);
                    raw[c][4 * i] = v.x, raw[c][4 * i + 1] = v.y, raw[c][4 * i + 2] = v.z, raw[c][4 * i + 3] = v.w;
                }
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 f = two<T>(raw[c][i]);
                    most = max(most, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
                }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            float up, down;
            row_scale(most, up, down);
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 f = two<T>(raw[c][i]);
                    qf[nt][c][i >> 1][i & 1] = pack(f.x * up, f.y * up, __half());
                }
            // columns 2 t, 2 t + 1 of the accumulators are rows held by lanes 8 t, 8 t + 4
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                factor[nt][i] = p.scale_log2 * __shfl_sync(0xffffffffu, down, 8 * t + 4 * i);
                const int ri = nt * kRows + 2 * t + i;
                const int pos = it.seq.pos0 + (it.row0 + ri) / p.a.group;
                hi[nt][i] = ri < it.nrows ? pos + 1 : 0;
                lo[nt][i] = p.a.window > 0 ? pos - p.a.window + 1 : 0;
            }
        }

        float o[NT][Cfg::kM][4], m[NT][2], mv[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < Cfg::kM; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
            m[nt][0] = m[nt][1] = mv[nt][0] = mv[nt][1] = -kInf;
            l[nt][0] = l[nt][1] = 0.f;
        }
        auto work = [&](int step, int stage) {
            const int n0 = step * Cfg::kTiles;
            copies_wait<Cfg::kStages - 1>();
            __syncwarp();
            const unsigned char *kt = ring + stage * Cfg::kStep, *vt = kt + Cfg::kTiles * 16 * Cfg::kRow;
            // S^T
            float s[Cfg::kTiles][NT][4];
#pragma unroll
            for (int i = 0; i < Cfg::kTiles; ++i) {
#pragma unroll
                for (int e = 0; e < 4 * NT; ++e) s[i][e / 4][e % 4] = 0.f;
                // lane's K: tokens g and g + 8, bytes 64 c + 16 t .. + 15
                const unsigned char *row = kt + (16 * i + g) * Cfg::kRow + 16 * t;
#pragma unroll
                for (int c = 0; c < HD / 64; ++c) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(row + 64 * c);
                    const uint4 y = *reinterpret_cast<const uint4 *>(row + 8 * Cfg::kRow + 64 * c);
                    const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t a0, a1, a2, a3;
                        e4m3x4_to_h2x2(xw[j], a0, a2);
                        e4m3x4_to_h2x2(yw[j], a1, a3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma16816(s[i][nt], a0, a1, a2, a3, qf[nt][c][j][0], qf[nt][c][j][1]);
                    }
                }
            }
            // masked, scaled scores
            float sk[Cfg::kTiles], lv[Cfg::kTiles];
            bool seen[Cfg::kTiles];
#pragma unroll
            for (int i = 0; i < Cfg::kTiles; ++i) {
                const int n = n0 + i;  // the copies are up to kStages - 1 steps ahead: perhaps in the next window
                const bool old = n / 32 != min(step + Cfg::kStages - 1, steps - 1) * Cfg::kTiles / 32;
                sk[i] = __shfl_sync(0xffffffffu, old ? ks_old : ks, n & 31);
                lv[i] = __log2f(__shfl_sync(0xffffffffu, old ? lvs_old : lvs, n & 31));
                seen[i] = (old ? there_old : there) >> (n & 31) & 1u;
            }
            float base[NT][2], basev[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float top[2] = {-kInf, -kInf}, topv[2] = {-kInf, -kInf};
#pragma unroll
                for (int i = 0; i < Cfg::kTiles; ++i) {
                    const int tok = tile_at(n0 + i) * 16 + g;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int c = e & 1, at = tok + 8 * (e >> 1);
                        float &x = s[i][nt][e];
                        x = seen[i] && at >= lo[nt][c] && at < hi[nt][c] ? x * (factor[nt][c] * sk[i]) : -kInf;
                        top[c] = fmaxf(top[c], x);
                        topv[c] = fmaxf(topv[c], x + lv[i]);
                    }
                }
                bool moved = false;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float mn = fmaxf(m[nt][c], max_over_rows(top[c]));
                    const float vn = fmaxf(mv[nt][c], max_over_rows(topv[c]));
                    base[nt][c] = finite_or_0(mn);
                    basev[nt][c] = finite_or_0(vn);
                    l[nt][c] *= ex2(m[nt][c] - base[nt][c]);
                    moved |= vn != mv[nt][c];
                    top[c] = ex2(mv[nt][c] - basev[nt][c]);  // O's factor
                    m[nt][c] = mn;
                    mv[nt][c] = vn;
                }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int i = 0; i < Cfg::kM; ++i) {
                        o[nt][i][0] *= top[0], o[nt][i][2] *= top[0];
                        o[nt][i][1] *= top[1], o[nt][i][3] *= top[1];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < Cfg::kTiles; ++i) {
                uint32_t b0[NT], b1[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float pr[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        l[nt][e & 1] += ex2(s[i][nt][e] - base[nt][e & 1]);
                        pr[e] = ex2(s[i][nt][e] + (lv[i] + kLift) - basev[nt][e & 1]);
                    }
                    b0[nt] = transpose8x8(pack(pr[0], pr[1], __half()));
                    b1[nt] = transpose8x8(pack(pr[2], pr[3], __half()));
                }
                // lane's V: tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9, bytes kVB (8 h + g) .. of each
                const unsigned char *row = vt + (16 * i + 2 * t) * Cfg::kRow + Cfg::kVB * g;
#pragma unroll
                for (int h = 0; h < Cfg::kVH; ++h) {
                    uint32_t w[4][Cfg::kVB / 4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const unsigned char *at = row + ((r & 1) + 8 * (r >> 1)) * Cfg::kRow + 8 * Cfg::kVB * h;
                        if constexpr (Cfg::kVB == 16) {
                            const uint4 x = *reinterpret_cast<const uint4 *>(at);
                            w[r][0] = x.x, w[r][1] = x.y, w[r][2] = x.z, w[r][3] = x.w;
                        } else {
                            const uint2 x = *reinterpret_cast<const uint2 *>(at);
                            w[r][0] = x.x, w[r][1] = x.y;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < Cfg::kVB / 4; ++j) {
                        // tokens 2 t and 2 t + 1 (then + 8) of dims 4 j .. 4 j + 3, interleaved
                        uint32_t a[4], b[4];
                        e4m3x4_to_h2x2(__byte_perm(w[0][j], w[1][j], 0x5140), a[0], a[1]);
                        e4m3x4_to_h2x2(__byte_perm(w[0][j], w[1][j], 0x7362), a[2], a[3]);
                        e4m3x4_to_h2x2(__byte_perm(w[2][j], w[3][j], 0x5140), b[0], b[1]);
                        e4m3x4_to_h2x2(__byte_perm(w[2][j], w[3][j], 0x7362), b[2], b[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const int d = h * (Cfg::kVB / 2) + 2 * j;
                            mma16816(o[nt][d], a[0], a[1], b[0], b[1], b0[nt], b1[nt]);
                            mma16816(o[nt][d + 1], a[2], a[3], b[2], b[3], b0[nt], b1[nt]);
                        }
                    }
                }
            }
            __syncwarp();  // the stage has been read
        };
        for (int step0 = 0; step0 < steps; step0 += Cfg::kStages) {
#pragma unroll
            for (int st = 0; st < Cfg::kStages; ++st) {
                if (step0 + st >= steps) continue;
                fetch(step0 + st + Cfg::kStages - 1, (st + Cfg::kStages - 1) % Cfg::kStages);
                work(step0 + st, st);
            }
        }
        copies_wait<0>();

        // ---- merge the warps
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], x);
                if (g == 0) {
                    float *row = mlm[warp][nt * kRows + 2 * t + c];
                    row[0] = m[nt][c], row[1] = l[nt][c], row[2] = mv[nt][c];
                }
            }
            // o[..][e]: dim kVB (8 h + g) + 2 j + (e >> 1), row 2 t + (e & 1), for MMA h kVB / 2 + j
#pragma unroll
            for (int i = 0; i < Cfg::kM; ++i) {
                const int h = i / (Cfg::kVB / 2), j = i % (Cfg::kVB / 2);
                float *dst = reinterpret_cast<float *>(ring) + (nt * kRows + 2 * t) * (HD + 4) + Cfg::kVB * (8 * h + g) + 2 * j;
                *reinterpret_cast<float2 *>(dst) = make_float2(o[nt][i][0], o[nt][i][2]);
                *reinterpret_cast<float2 *>(dst + HD + 4) = make_float2(o[nt][i][1], o[nt][i][3]);
            }
        }
        __syncthreads();
        const int slot = wk.slot(cta);
        for (int x = threadIdx.x; x < it.nrows * (HD / 4); x += kThreads) {
            const int r = x / (HD / 4), d = 4 * (x % (HD / 4));
            float mm = -kInf, mmv = -kInf, ll = 0.f;
#pragma unroll
            for (int i = 0; i < kWarps; ++i) mm = fmaxf(mm, mlm[i][r][0]), mmv = fmaxf(mmv, mlm[i][r][2]);
            const float b = finite_or_0(mm), bv = finite_or_0(mmv);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                ll += mlm[i][r][1] * ex2(mlm[i][r][0] - b);
                const float f = ex2(mlm[i][r][2] - bv);
                const float4 v = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(smem) + i * kMerge + r * (HD + 4) + d);
                acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
            }
            // O is in units of 2^(M - kLift), l in units of 2^m; a row that saw nothing has l = 0
            const float f = ll == 0.f ? 0.f : ex2(bv - b) * kUnlift / ll;
            acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
            if (whole) {
                const int row = it.row0 + r, tok = row / p.a.group, hq = head * p.a.group + row - tok * p.a.group;
                T *dst = static_cast<T *>(p.out) + (static_cast<int64_t>(it.seq.q0) + tok) * p.out_row +
                         hq * p.out_head + d;
                store_out4(dst, acc.x, acc.y, acc.z, acc.w);
            } else {
                const int64_t at = static_cast<int64_t>(slot) * NT * kRows + r;
                *reinterpret_cast<float4 *>(p.part.o + at * HD + d) = acc;
                if (d == 0) *reinterpret_cast<float2 *>(p.part.ml + 2 * at) = make_float2(mm, ll);
            }
        }
        if (threadIdx.x == 0 && wk.first == 0 && !whole)
            p.part.split[cta] = Split{pair, head, it.nrows, wk.last_cta(pl)};
        __syncthreads();
    }
}

// Joins the partial answers of the items that several CTAs share: their
// weights are l 2^(m - max m).  An item of few parts (prompts: 2 or 3) has a
// row per 16 lanes; the parts of one of many (a long context: hundreds) are
// spread over the CTA, so that the loads of all of them are in flight at once.
// Tasks (item, rows, dims) are dealt over a fixed grid; the order of the sums
// is that of the CTAs, the same every time.
constexpr int kCombThreads = 256;
constexpr int kCombPerSm = 4;

// A part's share is formed before its answers are added up: times l they could pass fp32's range.
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : __fdividef(1.0f, l); }
__device__ __forceinline__ void add(float4 &acc, const float4 &v, float share) {
    acc.x += v.x * share, acc.y += v.y * share, acc.z += v.z * share, acc.w += v.w * share;
}

template <typename T>
__global__ void __launch_bounds__(kCombThreads) kv8_combine_kernel(const AttnArgs p, int hd, int ctas, int few) {
    extern __shared__ int sm_i[];  // [ctas] tasks of the entries before this one
    __shared__ int warp_n[kCombThreads / 32];
    __shared__ float4 acc_s[kCombThreads / 32][4];
    __shared__ float2 ml_s[kCombThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, grp = tid >> 4, gl = tid & 15;
    const int chunks = hd / 64, fine = hd / 16;
    kernel_begins();
    int tasks = 0;
    for (int i0 = 0; i0 < ctas; i0 += kCombThreads) {
        const int i = i0 + tid;
        int mine = 0;
        if (i < ctas) {
            const Split sp = p.part.split[i];
            if (sp.nrows > 0) mine = sp.last_cta - i < few ? (sp.nrows + 15) / 16 : sp.nrows * fine;
        }
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int n = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += n;
        }
        if (lane == 31) warp_n[warp] = upto;
        __syncthreads();
        int before = tasks + upto - mine;
#pragma unroll
        for (int w = 0; w < kCombThreads / 32; ++w) {
            if (w < warp) before += warp_n[w];
            tasks += warp_n[w];
        }
        if (i < ctas) sm_i[i] = before;
        __syncthreads();
    }
    auto out_at = [&](const Split &sp, int r) {  // row r of the item
        const int si = sp.pair / p.a.tiles, row = (sp.pair - si * p.a.tiles) * p.a.rows + r;
        const int tok = row / p.a.group, hq = sp.head * p.a.group + row - tok * p.a.group;
        return static_cast<T *>(p.out) + (static_cast<int64_t>(load_seq(p.b, si, false).q0) + tok) * p.out_row +
               hq * p.out_head;
    };
    for (int task = blockIdx.x; task < tasks; task += gridDim.x) {
        int first = 0, end = ctas;  // the last entry with sm_i <= task: the one that has it, as empty ones follow it
        while (end - first > 1) {
            const int mid = (first + end) >> 1;
            if (sm_i[mid] <= task) first = mid;
            else end = mid;
        }
        const Split sp = p.part.split[first];
        const int sub = task - sm_i[first], n = sp.last_cta - first + 1;
        if (n <= few) {  // 16 lanes hold a row, lane gl dims 64 c + 4 gl ..
            const int r = 16 * sub + grp;
            if (r >= sp.nrows) continue;
            // lane i has part i's maximum and sum
            auto part_at = [&](int i) { return static_cast<int64_t>(2 * (first + i) + (i == 0 ? 1 : 0)) * p.a.rows + r; };
            auto load = [&](float4 (&v)[4], int i) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c < chunks) v[c] = *reinterpret_cast<const float4 *>(p.part.o + part_at(i) * hd + 64 * c + 4 * gl);
            };
            float4 v0[4];  // on its way while the shares are formed
            load(v0, 0);
            const uint32_t half = 0xffffu << (lane & 16);
            const float2 ml = gl < n ? *reinterpret_cast<const float2 *>(p.part.ml + 2 * part_at(gl)) : make_float2(-kInf, 0.f);
            float top = ml.x;
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(half, top, o));
            const float w = ml.y * ex2(ml.x - finite_or_0(top));
            float l = w;
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) l += __shfl_xor_sync(half, l, o);
            const float mine = w * inverse(l);
            float4 acc[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
            auto take = [&](const float4 (&v)[4], int i) {
                const float share = __shfl_sync(half, mine, (lane & 16) + i);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c < chunks) add(acc[c], v[c], share);
            };
            for (int i = 0;;) {
                take(v0, i);
                if (++i == n) break;
                load(v0, i);
            }
            T *dst = out_at(sp, r) + 4 * gl;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (c < chunks) store_out4(dst + 64 * c, acc[c].x, acc[c].y, acc[c].z, acc[c].w);
            continue;
        }
        // 4 lanes hold 16 dims of the row, every 64th part per 4 lanes
        const int r = sub / fine, d = 16 * (sub % fine) + 4 * (tid & 3);
        float m = -kInf, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        constexpr int kAt = 5;  // parts at a time: all of one item's on 148 SMs (two CTAs each, 64 groups here)
        for (int i0 = tid >> 2; i0 < n; i0 += kAt * (kCombThreads / 4)) {
            float2 ml[kAt];
            float4 v[kAt];
#pragma unroll
            for (int k = 0; k < kAt; ++k) {
                const int i = i0 + k * (kCombThreads / 4);
                const int64_t at = static_cast<int64_t>(2 * (first + i) + (i == 0 ? 1 : 0)) * p.a.rows + r;
                ml[k] = i < n ? *reinterpret_cast<const float2 *>(p.part.ml + 2 * at) : make_float2(-kInf, 0.f);
                v[k] = i < n ? *reinterpret_cast<const float4 *>(p.part.o + at * hd + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            float mn = m;
#pragma unroll
            for (int k = 0; k < kAt; ++k) mn = fmaxf(mn, ml[k].x);
            const float b = finite_or_0(mn), old = l * ex2(m - b);
            l = old;
#pragma unroll
            for (int k = 0; k < kAt; ++k) l += ml[k].y *= ex2(ml[k].x - b);
            m = mn;
            const float inv = inverse(l), so = old * inv;
            acc.x *= so, acc.y *= so, acc.z *= so, acc.w *= so;
#pragma unroll
            for (int k = 0; k < kAt; ++k) add(acc, v[k], ml[k].y * inv);
        }
        // join the warp's 8 groups, then the warps
        float top = m;
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float w = l * ex2(m - finite_or_0(top));
        l = w;
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const float share = w * inverse(l);
        acc.x *= share, acc.y *= share, acc.z *= share, acc.w *= share;
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            acc.x += __shfl_xor_sync(0xffffffffu, acc.x, o), acc.y += __shfl_xor_sync(0xffffffffu, acc.y, o);
            acc.z += __shfl_xor_sync(0xffffffffu, acc.z, o), acc.w += __shfl_xor_sync(0xffffffffu, acc.w, o);
        }
        if (lane < 4) {
            acc_s[warp][lane] = acc;
            if (lane == 0) ml_s[warp] = make_float2(top, l);
        }
        __syncthreads();
        if (tid < 4) {
            constexpr int kW = kCombThreads / 32;
            float all = -kInf, sum = 0.f, ws[kW];
#pragma unroll
            for (int i = 0; i < kW; ++i) all = fmaxf(all, ml_s[i].x);
#pragma unroll
            for (int i = 0; i < kW; ++i) sum += ws[i] = ml_s[i].y * ex2(ml_s[i].x - finite_or_0(all));
            const float inv = inverse(sum);
            acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < kW; ++i) add(acc, acc_s[i][tid], ws[i] * inv);
            store_out4(out_at(sp, r) + d, acc.x, acc.y, acc.z, acc.w);
        }
        __syncthreads();
    }
}

// Rows of a sequence and kv head up to which the rows kernel is taken (its further tiles read the cache again, from
// L2).  Measured against the prompt kernel on five shapes of 20 to 160 MB of cache: at 16 rows 29 to 39 us against 42
// to 78, at 32 rows 38 to 54 against 43 to 80, at 48 rows 47 to 71 against 39 to 68, at 64 rows 56 to 81 against 40 to 69.
// Tiles of 16 rows instead of 8 (head dims 64 and 128; at 256 their sums spill: 52 us against 37): at 16 rows 29 to 39 us
// against 31 to 45.
constexpr int kRowsMost = 32;
// CTAs per SM of the rows kernel: registers allow two of 128 threads.
constexpr int kRowsPerSm = 2;

cudaError_t sm_count(int *sms) {
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    return e != cudaSuccess ? e : cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
}

template <int HD, int NT, typename T>
cudaError_t launch_tiles(const AttnArgs &p, int ctas, cudaStream_t s) {
    const size_t smem = RowsCfg<HD>::kSmem;
    const cudaError_t e = cudaFuncSetAttribute(kv8_rows_kernel<HD, NT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(smem));
    return e != cudaSuccess ? e : launch_behind(kv8_rows_kernel<HD, NT, T>, dim3(ctas), kThreads, smem, s, p);
}
template <int HD, typename T>
cudaError_t launch_rows(const AttnArgs &p, int ctas, cudaStream_t s) {
    if constexpr (HD <= 128)
        if (p.a.rows == 2 * kRows) return launch_tiles<HD, 2, T>(p, ctas, s);
    return launch_tiles<HD, 1, T>(p, ctas, s);
}
template <typename T>
cudaError_t launch_combine(const AttnArgs &p, int hd, int ctas, int sms, cudaStream_t s) {
    // parts up to which an item is joined by rows: more where there are many items to fill the grid with (48 items of 6
    // to 9 parts: 36.0 us with 8, 31.2 with 16; one item of 10 parts: 9.9 with 8, 11.1 with 16; ten other shapes alike)
    const int few = static_cast<int64_t>(p.b.batch) * p.a.tiles * p.c.heads >= 32 ? 16 : 8;
    return launch_behind(kv8_combine_kernel<T>, dim3(kCombPerSm * sms), kCombThreads,
                         sizeof(int) * static_cast<size_t>(ctas), s, p, hd, ctas, few);
}
template <typename T>
cudaError_t launch_attention(const AttnArgs &p, int hd, int ctas, int sms, cudaStream_t s) {
    const cudaError_t e = p.a.rows > 2 * kRows
                              ? launch_prompt(p, hd, std::is_same<T, __half>::value, ctas, s)
                          : hd == 64  ? launch_rows<64, T>(p, ctas, s)
                          : hd == 128 ? launch_rows<128, T>(p, ctas, s)
                                      : launch_rows<256, T>(p, ctas, s);
    return e != cudaSuccess ? e : launch_combine<T>(p, hd, ctas, sms, s);
}

struct Debug {  // mg_kv8_set_debug, of the calling thread
    uint64_t wait_ns = kWaitBudgetNs;
    int stall = -1;
};
thread_local Debug debug;

struct Plan {
    int rows, unit, extra, tiles, ctas, sms;
    size_t bytes;
};
// How a call runs: set by the cache's dimensions and the batch's bounds alone, so that the workspace's size is too.
cudaError_t plan_of(int hd, int group, int max_q, Plan *pl) {
    int sms = 0;
    const cudaError_t e = sm_count(&sms);
    if (e != cudaSuccess) return e;
    const bool prompt = static_cast<int64_t>(max_q) * group > kRowsMost;
    pl->sms = sms;
    const bool two = hd <= 128 && static_cast<int64_t>(max_q) * group > kRows;  // the sums of 16 rows of 256 dims spill
    pl->rows = prompt ? prompt_rows(hd) : two ? 2 * kRows : kRows;
    pl->unit = prompt ? kPromptUnit : kUnit;
    pl->extra = prompt ? kPromptExtra : 0;
    pl->ctas = prompt ? sms : sms * kRowsPerSm;
    pl->tiles = static_cast<int>((static_cast<int64_t>(max_q) * group + pl->rows - 1) / pl->rows);
    pl->bytes = partials_bytes(pl->ctas, pl->rows, hd);
    return cudaSuccess;
}
mg_status cuda_error(const char *who, cudaError_t e) {
    char buf[160];
    snprintf(buf, sizeof buf, "%s: %s", who, cudaGetErrorString(e));
    return report_error(MG_ERR_CUDA, buf);
}
mg_status check_heads(const char *who, const mg_kv8_cache *c, const mg_kv8_batch *b, int num_heads) {
    char buf[200];
    if (num_heads <= 0 || num_heads % c->num_kv_heads != 0) {
        snprintf(buf, sizeof buf, "%s: num_heads must be a positive multiple of num_kv_heads", who);
        return report_error(MG_ERR_INVALID, buf);
    }
    if (num_heads / c->num_kv_heads > 128 ||
        static_cast<int64_t>(b->batch) * b->max_q * (num_heads / c->num_kv_heads) > (1ll << 30)) {
        snprintf(buf, sizeof buf, "%s: more than 128 heads per kv head, or batch * max_q too large", who);
        return report_error(MG_ERR_UNSUPPORTED, buf);
    }
    return MG_OK;
}
}  // namespace
}  // namespace kv8
}  // namespace mg

using namespace mg;

extern "C" mg_status mg_kv8_attention_workspace(const mg_kv8_cache *cache, const mg_kv8_batch *batch,
                                                int32_t num_heads, int64_t *bytes_out) {
    using namespace kv8;
    const char *who = "mg_kv8_attention_workspace";
    mg_status st = check_cache_batch(who, cache, batch);
    if (st == MG_OK) st = check_heads(who, cache, batch, num_heads);
    if (st != MG_OK) return st;
    if (!bytes_out) return report_error(MG_ERR_INVALID, "mg_kv8_attention_workspace: null output");
    Plan pl;
    const cudaError_t e = plan_of(cache->head_dim, num_heads / cache->num_kv_heads, batch->max_q, &pl);
    if (e != cudaSuccess) return cuda_error(who, e);
    *bytes_out = static_cast<int64_t>(pl.bytes);
    return MG_OK;
}

extern "C" mg_status mg_kv8_attention(const mg_kv8_cache *cache, const mg_kv8_batch *batch,
                                      const mg_kv8_attention_args *args, void *stream) {
    using namespace kv8;
    const char *who = "mg_kv8_attention";
    mg_status st = check_cache_batch(who, cache, batch);
    if (st != MG_OK) return st;
    if (!args || args->struct_size != static_cast<int32_t>(sizeof *args))
        return report_error(MG_ERR_INVALID, "mg_kv8_attention: null argument or struct_size mismatch");
    st = check_heads(who, cache, batch, args->num_heads);
    if (st != MG_OK) return st;
    if (args->dtype != MG_BF16 && args->dtype != MG_F16)
        return report_error(MG_ERR_UNSUPPORTED, "mg_kv8_attention: dtype must be MG_BF16 or MG_F16");
    const float scale_log2 = args->scale * 1.4426950408889634f;
    if (args->window < 0 || !(fabsf(scale_log2) <= FLT_MAX))
        return report_error(MG_ERR_INVALID, "mg_kv8_attention: need window >= 0 and a finite scale (scale * log2(e) too)");
    if (!args->q_dev || !args->out_dev) return report_error(MG_ERR_INVALID, "mg_kv8_attention: null q or out");
    if (((reinterpret_cast<uintptr_t>(args->q_dev) | reinterpret_cast<uintptr_t>(args->out_dev)) % 16) != 0 ||
        ((args->q_row_stride | args->q_head_stride | args->out_row_stride | args->out_head_stride) % 8) != 0)
        return report_error(MG_ERR_INVALID,
                            "mg_kv8_attention: q and out must be 16-byte aligned with strides in multiples of 8");
    // a part of an item may read a row that another part has answered already
    if (args->q_dev == args->out_dev) return report_error(MG_ERR_INVALID, "mg_kv8_attention: out must not be q");
    const int group = args->num_heads / cache->num_kv_heads;
    Plan pl;
    cudaError_t e = plan_of(cache->head_dim, group, batch->max_q, &pl);
    if (e != cudaSuccess) return cuda_error(who, e);
    if (!args->workspace_dev || reinterpret_cast<uintptr_t>(args->workspace_dev) % 16 != 0 ||
        args->workspace_bytes < static_cast<int64_t>(pl.bytes))
        return report_error(MG_ERR_INVALID, "mg_kv8_attention: workspace missing, unaligned or too small "
                                            "(mg_kv8_attention_workspace)");
    AttnArgs p;
    p.c = cache_of(cache);
    p.b = batch_of(batch);
    // a window that reaches every position is none (and no position less it underflows)
    const int window = args->window >= batch->max_ctx ? 0 : args->window;
    p.a = AttnShape{group, pl.rows, pl.tiles, window, pl.unit, pl.extra};
    p.part = partials_at(args->workspace_dev, pl.ctas, pl.rows);
    p.q = args->q_dev, p.out = args->out_dev;
    p.q_row = args->q_row_stride, p.q_head = args->q_head_stride;
    p.out_row = args->out_row_stride, p.out_head = args->out_head_stride;
    p.scale_log2 = scale_log2;
    p.wait_ns = debug.wait_ns;
    p.stall = debug.stall;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    e = args->dtype == MG_BF16 ? launch_attention<__nv_bfloat16>(p, cache->head_dim, pl.ctas, pl.sms, s)
                               : launch_attention<__half>(p, cache->head_dim, pl.ctas, pl.sms, s);
    return e == cudaSuccess ? MG_OK : cuda_error(who, e);
}

extern "C" mg_status mg_kv8_set_debug(uint64_t wait_budget_ns, int32_t stall) {
    using namespace kv8;
    if (stall < -1 || stall >= kHandoffs) {
        char buf[100];
        snprintf(buf, sizeof buf, "mg_kv8_set_debug: stall %d outside [-1, %d)", stall, static_cast<int>(kHandoffs));
        return report_error(MG_ERR_INVALID, buf);
    }
    debug.wait_ns = wait_budget_ns ? wait_budget_ns : kWaitBudgetNs;
    debug.stall = stall;
    return MG_OK;
}
