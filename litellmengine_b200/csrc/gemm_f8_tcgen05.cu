// y[T, N] = x[T, K] . w[N, K]^T of numbers of 8 bits under float32 scales (f8_blocks.cuh has the format), of one matrix or of a stack's matrices by
// rows sorted by expert, on the 5th-generation tensor cores (tcgen05.mma.kind::f8f6f4).
//
//   y[t, n] = sum over tiles b of 128 values of K: sx[t, b] * sw[n / 128, b] * (sum over the 128 values of cx * cw)
// Products of codes are exact and a tile's sum is the tensor core's, in float32.  The scales are float32 numbers that no product applies, so every tile of K has
// an accumulator of its own in tensor memory, which other warps take out, multiply and add up in registers while the next ones are computed.
//   * Few rows: bytes bound the product.  The weights are the left operand (128 features a tile), the rows the right one (NT of them), so that no lane is spent
//     on rows that are not there.  K is cut over a cluster's CTAs, which add their sums up in each other's shared memory in the parts' order;
//     nothing is left for another kernel and no result depends on timing.
//   * Many rows: pairs of CTAs, or CTAs of 128 rows alone.  The rows are the left operand, so that a lane is a row and its scale one number for 64 or 128 features.
//   * Gate and up: act(gate) * up leaves as rows of 8 bits, 128 features a scale.
//   * Rows sorted by expert: an item (up to a tile's rows of one expert) takes the place of a tile of rows; how many there are only the device knows.
// Waits are bounded: one that runs out sets status code 10, and the copies and products that are under way then end, which is waited for on their own barriers
// (bounded too), before the CTA does; what was not computed is neither stored nor added (routed experts' rows that were not are added up as the workspace has them:
// the status says that the result is of no use).
#include "f8_blocks.cuh"
#include "tcgen05_attention.cuh"

#include <type_traits>

#define F8_STATUS 10

__device__ __forceinline__ bool f8_wait(unsigned long long* bar, unsigned parity, int waits, volatile int* abort_flag, int32_t* status) {
    for (int i = 0; i < waits; ++i) {
        if (t5_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
    }
    *abort_flag = 1;
    if (atomicCAS(status, 0, F8_STATUS) == 0) status[1] = blockIdx.y;
    return false;
}
// What was asked for before a wait ran out: its end.
__device__ __forceinline__ void f8_land(unsigned long long* bar, unsigned parity) {
    for (int i = 0; i < T5_WAIT_LIMIT && !t5_try_wait(bar, parity); ++i) {}
}
// The uses of a ring's barriers that may be under way, of `asked` in all.
__device__ __forceinline__ void f8_land_ring(unsigned long long* bars, int ring, int asked) {
    for (int i = max(0, asked - ring); i < asked; ++i) f8_land(&bars[i % ring], (i / ring) & 1);
}
__device__ __forceinline__ void f8_tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, unsigned long long* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(t5_smem(dst)), "l"(map),
                 "r"(x), "r"(y), "r"(z), "r"(t5_smem(bar)) : "memory");
}
__device__ __forceinline__ void f8_mma_lead(unsigned lead, unsigned d_tmem, unsigned long long a_desc, unsigned long long b_desc, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
                 " @q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::
                     "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
__device__ __forceinline__ unsigned long long f8_mul2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// Instruction descriptor: e4m3 x e4m3 -> float32, M x N, both K-major.
__host__ __device__ constexpr unsigned f8_idesc(int m, int n) {
    return (1u << 4) | (static_cast<unsigned>(n >> 3) << 17) | (static_cast<unsigned>(m >> 4) << 24);
}

struct F8Args {
    const float* w_scales;                // [tiles][first 64 features, 65th, last][K4]
    const float* x_scales;                // [x_rows][K4]
    long long x_rows;
    void* y;                              // [T, N]; gated: the codes [tiles / 2][y_rows][128]
    float* y_scales;                      // gated: [y_rows][y_k4]
    long long y_rows;
    int T, N, K, ktiles, k4, y_k4, tiles, vec, waits;       // k4: room for a row's scales; tiles: of a matrix of the stack; N gated: features of the result
    int32_t* status;
    MxAct act;
    const bf16* plain;                    // a matrix [tokens, K] that the kernel takes to 8 bits itself
    F8Groups groups;
    int on_input;                         // a row's weight multiplies its gate and up values instead of the result
    const float* base;                    // picks as they are: what a token's sum starts from, or null
};
enum { F8_STORE = 0, F8_ADD = 1, F8_GATED = 2 };

// ---- few rows -------------------------------------------------------------------------------------------------------
// Warps: two that feed weights and issue, four for the sums of each of a CTA's tiles of the weight, and those that make rows of a matrix, or one that feeds rows.
#define F8_MAKERS(WT) ((WT) == 2 ? 4 : 8)
#define F8_PLAIN_ROWS(GATED) ((GATED) ? 4 : 8)              // up to which a product makes its rows of a bfloat16 matrix of whole, aligned pieces of eight values itself
#define F8_FEW_CTAS(NT, WT) ((NT) * (WT) > 64 ? 1 : 2)          // on an SM: sums of 64 rows of two tiles need the registers of both
#define F8_FEW_THREADS(PLAIN, WT) (32 * (2 + 4 * (WT) + ((PLAIN) ? F8_MAKERS(WT) : 1)))

// grid (parts of K, tiles of features, tiles of rows or items), a cluster the parts of a tile.  WS: stages of weights; G: stages whose rows come together, two
// such groups at a time.  A CTA's tile is 128 features, gated 64 + 64 gate and as many up features, of two tiles of the weight.
// Warp 0 feeds the weights, warp 1 issues, warps from 2 on take the sums, the last feeds the rows and their scales; or, PLAIN, x comes as a matrix and the last warps make
// the rows of their part of K in shared memory: one launch and no rows in memory, for steps so short that every CTA can do it while its weights come.  Measured, so and with a launch
// for the rows (us): 4,096 by 6,144, a row 6.8 and 7.5, 8 rows 7.8 and 8.1, 16 rows 9.0 and 8.4; 12,288 by 4,096 10.1 and 11.1, 10.9 and 11.5, 12.8 and 12.0; gated, a row and 4 rows, 2,048 by 2 x 1,024 4.5 and 5.3,
// 4.7 and 5.3; 1,024 by 2 x 4,096 5.0 and 5.6, 5.3 and 5.8; 2,048 by 2 x 6,144 7.6 and 8.0, 8.2 and 8.3; 4,096 by 2 x 12,288 19.2 and 19.9, 19.7 and 19.7; 2,048 by 2 x 24,576 19.2 and 19.9, 19.4 and 19.5; with the
// down product behind it the same or up to 1.1 less, but 1,024 by 2 x 2,560 and 2,560 by 2 x 9,728, up to 0.2 of 9 and 0.4 of 19 more.  8 gated rows: 2,048 by 2 x 1,024 5.7 and 5.5.
// Measured (us): a row of 4,096 by 6,144 6.8 to 7.3 (25 MB, 3.5 TB/s); 8 rows of 8 bits, 12,288 by 4,096, 10.1 (50 MB, 5.0 TB/s), 4,096 by 24,576 17.7 (101 MB, 5.7 TB/s); gated, 8 rows of
// 4,096 by 2 x 12,288 18.7 (5.4 TB/s); 48 tokens' picks, 8 of 64 experts, 1,024 by 2,048 86 (4.7 TB/s of the weights) with their sorting and adding up.  Three CTAs an SM with three
// stages for the latter, so that more of them begin while others end, came out 84 to 88 there (85 to 90 with two, rows in bfloat16) and slower for 8 large experts (49 instead of 45 us).
template <int NT, int WS, int G, bool PLAIN, int MODE, typename TO, bool GROUPED>
__global__ void __launch_bounds__(F8_FEW_THREADS(PLAIN, MODE == F8_GATED ? 2 : 1), F8_FEW_CTAS(NT, MODE == F8_GATED ? 2 : 1)) f8_few_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                                                                         const F8Args a) {
    constexpr int WT = MODE == F8_GATED ? 2 : 1, THREADS = F8_FEW_THREADS(PLAIN, WT), MAKERS = F8_MAKERS(WT), LAST = 2 + 4 * WT, FEATURES = 128 * WT;
    constexpr bool TOGETHER = MODE != F8_GATED && !PLAIN;         // a row's scale comes times its tile of weights' (gate and up rows have one each)
    // Rows of an accumulator that are asked for together.  Of 64 rows' sums half (their registers leave no room for scales ahead): 64 rows of 4,096 by 24,576 26.9 us, in pieces of 16 with
    // scales ahead 27.9; 32 rows 20.5 and 20.2, gated 27.4 and 21.8.
    constexpr int PIECE = NT == 64 && MODE != F8_GATED ? 32 : 16;
    constexpr unsigned W_BYTES = WT * F8_TILE, X_BYTES = NT * F8_K, SLOT = NT * WT;
    constexpr unsigned SLOTS = 256 / SLOT < 4 ? 256 / SLOT : 4, COLS = SLOT * SLOTS < 32 ? 32 : SLOT * SLOTS;      // accumulators in turn; two CTAs share tensor memory
    static_assert(COLS <= 256 && SLOTS >= 2, "tensor memory");
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* w_s = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
    unsigned char* x_s = w_s + WS * W_BYTES;                      // [2][G][NT][128], 128-byte swizzle like the weights
    float* sx_s = reinterpret_cast<float*>(x_s + 2 * G * X_BYTES);        // [2][G][NT]
    float* sums = reinterpret_cast<float*>(w_s);                  // [NT][FEATURES], when the stages have been read
    __shared__ __align__(8) unsigned long long full[WS], empty[WS], x_full[2], x_empty[2], acc_full[SLOTS], acc_empty[SLOTS], drained, fed;
    __shared__ unsigned tmem_base_s;
    __shared__ int abort_flag, asked_s[2];                        // asked_s: stages of weights, groups of rows that were asked for
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int part = blockIdx.x, parts = gridDim.x;
    int kb0 = part * a.ktiles / parts, kbs = (part + 1) * a.ktiles / parts - kb0;
    int row0 = blockIdx.z * NT, rows = min(NT, a.T - row0), first_tile = blockIdx.y * WT;
    const bool joins = GROUPED && MODE == F8_STORE && a.groups.ids;
    if constexpr (GROUPED) {
        pdl_wait();                                               // the items are the kernel's in front
        if (a.groups.ids) {
            // A pick is an item.  Behind its down product a token's picks are the parts of the sum instead of K's: the cluster adds them up.
            row0 = joins ? blockIdx.z * parts + part : blockIdx.z;
            const int e = a.groups.ids[row0];
            rows = 1;
            if (static_cast<unsigned>(e) < static_cast<unsigned>(a.groups.E)) first_tile += e * a.tiles;
            else if (!joins) return;                              // the whole cluster
            if (joins) kb0 = 0, kbs = static_cast<unsigned>(e) < static_cast<unsigned>(a.groups.E) ? a.ktiles : 0;
        } else {
            if (static_cast<int>(blockIdx.z) >= a.groups.counts[0]) return;
            const int4 item = a.groups.items[blockIdx.z];
            first_tile += item.x * a.tiles, row0 = item.y, rows = item.z;
        }
    }
    const int early = min(WS, kbs);
    auto weights = [&](int kb, int s) {                           // into stage s
        t5_expect_tx(&full[s], W_BYTES);
#pragma unroll
        for (int w = 0; w < WT; ++w) t5_tma_2d(w_s + s * W_BYTES + w * F8_TILE, &w_map, 0, ((first_tile + w) * a.ktiles + kb0 + kb) * 128, &full[s]);
    };
    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < WS; ++s) { t5_mbar_init(&full[s], 1); t5_mbar_init(&empty[s], 1); }
        for (int s = 0; s < 2; ++s) { t5_mbar_init(&x_full[s], PLAIN ? MAKERS : 2); t5_mbar_init(&x_empty[s], 1 + 4 * WT); }      // the products and the warps of sums
        for (int s = 0; s < static_cast<int>(SLOTS); ++s) { t5_mbar_init(&acc_full[s], 1); t5_mbar_init(&acc_empty[s], 4 * WT); }
        t5_mbar_init(&drained, 1);
        t5_mbar_init(&fed, PLAIN ? 1 : 2);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        // Weights are nobody's output: the first of them are on their way before anything else, whatever runs in front.
        for (int kb = 0; kb < early; ++kb) weights(kb, kb);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(t5_smem(&tmem_base_s)), "r"(COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    t5_fence_before();
    __syncthreads();
    t5_fence_after();
    pdl_invite();                                                 // not before: this CTA's tensor memory is taken
    const unsigned tmem = __shfl_sync(0xffffffffu, tmem_base_s, 0);

    if (warp == 0) {
        if (lane == 0) {
            int issued = early, s = early % WS;
            unsigned phase = early == WS ? 0 : 1;                 // a barrier that was never used passes for the phase before its first
            if (early < kbs) pdl_wait();                          // the rest waits for products anyway, and these for the kernel in front: no bound on that
#pragma unroll 1
            for (int kb = early; kb < kbs; ++kb) {
                if (!f8_wait(&empty[s], phase, a.waits, &abort_flag, a.status)) break;
                weights(kb, s);
                issued = kb + 1;
                if (++s == WS) s = 0, phase ^= 1;
            }
            asked_s[0] = issued;
            t5_arrive(&fed);
        }
        __syncwarp();
    } else if (warp == 1) {
        const unsigned lead = elect_one();
        const unsigned long long wd = t5_desc(w_s, 16, 1024), xd = t5_desc(x_s, 16, 1024);
        bool ok = true;
        pdl_wait();                                               // the bounded waits below are not for the kernel in front
        int s = 0, slot = 0, q = 0, g = 0;
        unsigned phase = 0, turn = 0, acc_phase = 1;
#pragma unroll 1
        for (int kb = 0; kb < kbs; ++kb) {
            if (q == 0) ok = __all_sync(0xffffffffu, f8_wait(&x_full[g], turn, a.waits, &abort_flag, a.status));
            ok = ok && __all_sync(0xffffffffu, f8_wait(&acc_empty[slot], acc_phase, a.waits, &abort_flag, a.status) &&
                                                   f8_wait(&full[s], phase, a.waits, &abort_flag, a.status));
            if (!ok) break;
            t5_fence_after();
#pragma unroll
            for (int w = 0; w < WT; ++w)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    f8_mma_lead(lead, tmem + slot * SLOT + w * NT, wd + ((s * W_BYTES + w * F8_TILE) >> 4) + 2 * k, xd + (((g * G + q) * X_BYTES) >> 4) + 2 * k,
                                f8_idesc(128, NT), k ? 1u : 0u);
            t5_commit_lead(lead, &empty[s]);
            t5_commit_lead(lead, &acc_full[slot]);
            if (++s == WS) s = 0, phase ^= 1;
            if (++slot == static_cast<int>(SLOTS)) slot = 0, acc_phase ^= 1;
            if (++q == G) {
                t5_commit_lead(lead, &x_empty[g]);
                q = 0, g ^= 1;
                if (g == 0) turn ^= 1;
            }
        }
        t5_commit_lead(lead, &drained);                           // what was issued has ended, and all of it has been told
        f8_land(&drained, 0);
    } else if (warp < LAST) {
        const int quarter = warp & 3, w = (warp - 2) >> 2, feature = quarter * 32 + lane;
        pdl_wait();
        unsigned long long acc[NT / 2];                           // two rows each
#pragma unroll
        for (int i = 0; i < NT / 2; ++i) acc[i] = 0ull;
        // A lane has the weights' scales of every 32nd tile of K; of up rows two, where these 64 lie in two blocks.
        constexpr int HELD = MODE == F8_GATED ? 2 : 1;
        float mine[HELD];
        const bool second = HELD == 2 && quarter >= 2 && feature - 64 >= f8_split(a.N, blockIdx.y * WT + w);
        int slot = 0, q = 0, g = 0;
        unsigned turn = 0, acc_phase = 0;
        bool ok = true;
#pragma unroll 1
        for (int kb = 0; kb < kbs; ++kb) {
            if (!TOGETHER && (kb & 31) == 0) {
                const float* s = a.w_scales + (first_tile + w) * 3LL * a.k4 + kb0 + kb + lane;
#pragma unroll
                for (int i = 0; i < HELD; ++i) mine[i] = kb + lane < kbs ? s[HELD == 1 || quarter < 2 ? 0 : (1 + i) * a.k4] : 0.0f;
            }
            if (q == 0) {
                ok = __all_sync(0xffffffffu, f8_wait(&x_full[g], turn, a.waits, &abort_flag, a.status));
                if (!ok) break;
            }
            const unsigned at = tmem + (static_cast<unsigned>(quarter * 32) << 16) + slot * SLOT + w * NT;
            const float* sx = sx_s + (g * G + q) * NT;
            // A piece's scales are asked for ahead of the wait for its sums, which no load passes; while one piece is multiplied and added the next is on its way.
            ulonglong2 s[2][4];
            auto scales = [&](int c) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[c & 1][i] = *reinterpret_cast<const ulonglong2*>(sx + c * PIECE + 4 * i);
            };
            if (PIECE == 16) scales(0);
            ok = __all_sync(0xffffffffu, f8_wait(&acc_full[slot], acc_phase, a.waits, &abort_flag, a.status));
            if (!ok) break;
            t5_fence_after();
            float sw = __shfl_sync(0xffffffffu, mine[0], kb & 31);
            if constexpr (HELD == 2) {
                const float other = __shfl_sync(0xffffffffu, mine[HELD - 1], kb & 31);
                if (second) sw = other;
            }
            const unsigned long long sw2 = t5_two(sw, sw);
            unsigned r[2][PIECE];
            auto ask = [&](int c) {
                if constexpr (PIECE == 32) t5_ld32(at + c * PIECE, r[c & 1]);
                else t5_ld16(at + c * PIECE, r[c & 1]);
            };
            ask(0);
#pragma unroll
            for (int c = 0; c < NT / PIECE; ++c) {
                t5_wait_ld();
                if (c + 1 < NT / PIECE) {
                    ask(c + 1);
                    if (PIECE == 16) scales(c + 1);
                } else {                                            // all of it is in registers
                    t5_fence_before();
                    __syncwarp();
                    if (lane == 0) t5_arrive(&acc_empty[slot]);
                }
#pragma unroll
                for (int i = 0; i < PIECE; i += 4) {
                    unsigned long long *to = acc + (c * PIECE + i) / 2;
                    const ulonglong2 both = PIECE == 16 ? s[c & 1][i / 4] : *reinterpret_cast<const ulonglong2*>(sx + c * PIECE + i);
                    unsigned long long lo = both.x, hi = both.y;
                    if (!TOGETHER) lo = f8_mul2(lo, sw2), hi = f8_mul2(hi, sw2);
                    to[0] = t5_fma2(t5_two(__uint_as_float(r[c & 1][i]), __uint_as_float(r[c & 1][i + 1])), lo, to[0]);
                    to[1] = t5_fma2(t5_two(__uint_as_float(r[c & 1][i + 2]), __uint_as_float(r[c & 1][i + 3])), hi, to[1]);
                }
            }
            if (++slot == static_cast<int>(SLOTS)) slot = 0, acc_phase ^= 1;
            if (++q == G) {
                __syncwarp();
                if (lane == 0) t5_arrive(&x_empty[g]);
                q = 0, g ^= 1;
                if (g == 0) turn ^= 1;
            }
        }
        if (ok) {
#pragma unroll
            for (int i = 0; i < NT; i += 2) {
                float v[2];
                t5_untwo(acc[i / 2], v[0], v[1]);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (i + j < rows) sums[(i + j) * FEATURES + w * 128 + feature] = joins && kbs && a.groups.weights ? v[j] * a.groups.weights[row0] : v[j];
            }
        } else {
            // A wait ran out.  Who asks for copies has stopped; the copies (the stages are where the sums go) and the products end; then NaNs tell
            // whoever adds the parts up that these sums are not there.  Nothing of it is in the way of a product that does not give up.
            f8_land(&fed, 0);
            f8_land_ring(full, WS, asked_s[0]);
            if (!PLAIN) f8_land_ring(x_full, 2, asked_s[1]);
            f8_land(&drained, 0);
            for (int i = 0; i < rows; ++i) sums[i * FEATURES + w * 128 + feature] = __uint_as_float(0x7fffffffu);
        }
    } else if constexpr (PLAIN) {                                 // rows beyond the last keep what stands there, nobody minds
        // A warp takes two stages of a row at a time, sixteen lanes each, and has the next group's values on their way while it makes this one's.
        static_assert(G % 2 == 0, "stages go in pairs");
        constexpr int BATCH = (F8_PLAIN_ROWS(MODE == F8_GATED) * G / 2 + MAKERS - 1) / MAKERS;       // units of a group that a warp has at most
        const int p = lane & 15, units = rows * (G / 2);
        const int left = a.K - kb0 * F8_K - (lane >> 4) * F8_K - p * 8;       // values of the row from the lane's first on
        const bf16* from[BATCH];
        pdl_wait();
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            const int u = warp - LAST + j * MAKERS;
            long long r = 0;
            if (u < units) r = GROUPED ? row0 / a.groups.top : row0 + u / (G / 2);        // a pick's token
            from[j] = a.plain + r * a.K + kb0 * F8_K + (lane >> 4) * F8_K + p * 8 + u % (G / 2) * 2 * F8_K;
        }
        uint4 raw[BATCH];
        auto fetch = [&](int grp) {
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const int u = warp - LAST + j * MAKERS, at = grp * G * F8_K;
                raw[j] = u < units && at + u % (G / 2) * 2 * F8_K < left ? *reinterpret_cast<const uint4*>(from[j] + at) : make_uint4(0u, 0u, 0u, 0u);
            }
        };
        fetch(0);
#pragma unroll 1
        for (int grp = 0; grp * G < kbs; ++grp) {
            const int g = grp & 1;
            if (!__all_sync(0xffffffffu, f8_wait(&x_empty[g], ((grp >> 1) & 1) ^ 1, a.waits, &abort_flag, a.status))) break;
            uint4 now[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) now[j] = raw[j];
            fetch(grp + 1);                                       // beyond the part: not used, and beyond the row not read
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const int u = warp - LAST + j * MAKERS, r = u / (G / 2), q = u % (G / 2) * 2 + (lane >> 4);
                if (u >= units) break;                            // for the whole warp
                const unsigned most = f8_most16(mx_most8(now[j]));
                const F8Scale s = f8_scale(most);
                // the 128-byte swizzle: 16-byte piece i of row r at i ^ (r % 8)
                *reinterpret_cast<uint2*>(x_s + (g * G + q) * X_BYTES + r * F8_K + (((p >> 1) ^ (r & 7)) << 4) + (p & 1) * 8) = f8_codes8(now[j], most, s.inverse);
                if (p == 0) sx_s[(g * G + q) * NT + r] = s.scale;
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) t5_arrive(&x_full[g]);
        }
    } else {
        int issued = 0;
        pdl_wait();
#pragma unroll 1
        for (int grp = 0; grp * G < kbs; ++grp) {
            const int g = grp & 1, first = kb0 + grp * G;
            if (!__all_sync(0xffffffffu, f8_wait(&x_empty[g], ((grp >> 1) & 1) ^ 1, a.waits, &abort_flag, a.status))) break;
            if (lane == 0) {
                t5_expect_tx(&x_full[g], G * X_BYTES);
                f8_tma_3d(x_s + g * G * X_BYTES, &x_map, 0, row0, first, &x_full[g]);
            }
            constexpr int EACH = (G * NT + 31) / 32;
            float s[EACH];
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                const int i = lane + 32 * j, kb = first + i / NT;
                s[j] = i < G * NT && kb < a.ktiles && row0 + i % NT < a.x_rows ? a.x_scales[(row0 + i % NT) * static_cast<long long>(a.k4) + kb] : 0.0f;
                if (TOGETHER && kb < a.ktiles) s[j] *= a.w_scales[first_tile * 3LL * a.k4 + kb];
            }
#pragma unroll
            for (int j = 0; j < EACH; ++j)
                if (lane + 32 * j < G * NT) sx_s[g * G * NT + lane + 32 * j] = s[j];
            __syncwarp();
            if (lane == 0) t5_arrive(&x_full[g]);
            issued = grp + 1;
        }
        if (lane == 0) {
            asked_s[1] = issued;
            t5_arrive(&fed);
        }
        __syncwarp();
    }
    t5_fence_before();
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    // What the warp's first row is added to is on its way while the parts meet.
    const int feature = blockIdx.y * 128 + 4 * lane, first_row = part + warp * parts;
    float4 old = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if constexpr (MODE == F8_ADD) {
        pdl_wait();                                               // the warps that feed weights have not
        if (a.vec && first_row < rows && feature < a.N) old = *reinterpret_cast<const float4*>(static_cast<const float*>(a.y) + static_cast<size_t>(row0 + first_row) * a.N + feature);
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");       // every part's sums are there
    {
        const unsigned base = t5_smem(sums);
        auto total = [&](int at, float4 v) {                      // what they join and the parts' sums in order, four features, all parts' loads in flight at once
            float4 f[8];
#pragma unroll
            for (int p = 0; p < 8; ++p)
                if (p < parts) {
                    unsigned addr;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(addr) : "r"(base + 4u * at), "r"(p));
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(f[p].x), "=f"(f[p].y), "=f"(f[p].z), "=f"(f[p].w) : "r"(addr));
                }
#pragma unroll
            for (int p = 0; p < 8; ++p)
                if (p < parts) v.x += f[p].x, v.y += f[p].y, v.z += f[p].z, v.w += f[p].w;
            return v;
        };
        // Whether a sum that is NaN (of four neighbouring features all are) is one of a part that gave up.
        auto missing = [&](float sum) {
            if (sum == sum) return false;
            unsigned quit = 0;
            for (int p = 0; p < parts; ++p) {
                unsigned addr, flag;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(addr) : "r"(t5_smem(&abort_flag)), "r"(p));
                asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(flag) : "r"(addr));
                quit |= flag;
            }
            return quit != 0;
        };
        if constexpr (MODE == F8_GATED) {
            // a warp a row, four features a lane, all of a block
            const int f = 4 * lane;
            const long long block = blockIdx.y;
            unsigned char* codes = static_cast<unsigned char*>(a.y);
#pragma unroll 1
            for (int r = first_row; r < rows; r += THREADS / 32 * parts) {
                const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float4 g = total(r * FEATURES + (f >> 6) * 128 + (f & 63), none), u = total(r * FEATURES + (f >> 6) * 128 + 64 + (f & 63), none);
                const bool quit = missing(g.x + u.x);
                if (GROUPED && a.on_input) {
                    const float w = a.groups.weights[row0 + r];
                    g.x *= w, g.y *= w, g.z *= w, g.w *= w, u.x *= w, u.y *= w, u.z *= w, u.w *= w;
                }
                const float v[4] = {mx_gated(g.x, u.x, a.act), mx_gated(g.y, u.y, a.act), mx_gated(g.z, u.z, a.act), mx_gated(g.w, u.w, a.act)};
                unsigned most = max(max(mx_abs_bits(v[0]), mx_abs_bits(v[1])), max(mx_abs_bits(v[2]), mx_abs_bits(v[3])));
                most = __reduce_max_sync(0xffffffffu, most);
                const F8Scale s = f8_scale(most);
                if (!__any_sync(0xffffffffu, quit)) {
                    float q[4] = {v[0] * s.inverse, v[1] * s.inverse, v[2] * s.inverse, v[3] * s.inverse};
                    f8_settle(q, v, most);
                    *reinterpret_cast<unsigned*>(codes + (block * a.y_rows + row0 + r) * F8_K + f) = mx_e4m3x4(q[0], q[1], q[2], q[3]);
                    if (lane == 0) a.y_scales[(row0 + r) * static_cast<long long>(a.y_k4) + block] = s.scale;
                }
            }
        } else {
            TO* y = static_cast<TO*>(a.y);
            const int f = feature;
#pragma unroll 2
            for (int r = first_row; f < a.N && r < rows; r += THREADS / 32 * parts) {
                const size_t out_row = joins ? blockIdx.z : row0 + r;
                float from[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (joins && a.base)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (f + i < a.N) from[i] = a.base[out_row * a.N + f + i];
                const float4 t = total(r * FEATURES + 4 * lane, make_float4(from[0], from[1], from[2], from[3]));
                if (missing(t.x)) continue;
                float ts[4] = {t.x, t.y, t.z, t.w};
                if (GROUPED && a.groups.weights && !joins) {
                    const float w = a.groups.weights[row0 + r];
#pragma unroll
                    for (int i = 0; i < 4; ++i) ts[i] *= w;
                }
                TO* to = y + out_row * a.N + f;
                if (a.vec) {                                      // N a multiple of 4, y aligned
                    if constexpr (sizeof(TO) == 4) {
                        float4 v = make_float4(ts[0], ts[1], ts[2], ts[3]);
                        if (MODE == F8_ADD) {
                            const float4 o = r == first_row ? old : *reinterpret_cast<const float4*>(to);
                            v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
                        }
                        *reinterpret_cast<float4*>(to) = v;
                    } else {
                        const __nv_bfloat162 lo = __floats2bfloat162_rn(ts[0], ts[1]), hi = __floats2bfloat162_rn(ts[2], ts[3]);
                        *reinterpret_cast<uint2*>(to) = make_uint2(*reinterpret_cast<const unsigned*>(&lo), *reinterpret_cast<const unsigned*>(&hi));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (f + i < a.N) to[i] = from_f32<TO>(MODE == F8_ADD ? ts[i] + to_f32(to[i]) : ts[i]);
                }
            }
        }
    }
    __syncwarp();
    // Nobody leaves while its sums are read.  A thread that is here has all that it read, because it has made what it stored of it, or has seen that it is
    // NaN and of a part that gave up; the stores themselves need not be out yet, which a release would wait for.
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    if (warp == 1) {
        t5_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(COLS) : "memory");
    }
}

// ---- many rows: pairs of CTAs, and CTAs alone ---------------------------------------------------------------------------------------
// The two CTAs of a cluster compute a tile of 256 rows x 256 features together (cta_group::2): each brings its own 128 rows and half of the features, and
// reads both halves.  Or (CTAS = 1) a CTA computes a tile of 128 rows alone and brings all of the features: for 33 to 128 rows, experts of few rows, and where rounds of pairs would be
// half empty.  A CTA's tensor memory holds four accumulators of 128 rows x 128 features: a tile of K's products fill two of them, one for each tile of the weight,
// while those of the tile before are taken out.  Each has barriers and four warps of its own (a row and 128 features a thread, 64 pairs of sums in registers), so that
// its way round (products, the word of them, taking out, the word that it is free) overlaps the other three's.  Taking out (tcgen05.ld) and adding (fma of two at a time)
// alternate in quarters of 32 features; the accumulator is free again with the last quarter's additions still to do.
// Shared memory is busy with the products' operands, so that a load from it or a look at a barrier takes 100 to 200 clocks: what the next tile of K needs (its scales,
// whether its accumulator is full) is asked for between additions.  Scales come by a warp's asynchronous copies, eight tiles of K at a time into a ring of two: loads of the
// threads that need them would wait together with tcgen05.ld, whose wait is for all.
// Measured: a tile of K takes 700 clocks, its products 512.  4,096 rows of 4,096 by 24,576: 380 to 410 us with the clocks that the power limit leaves (1.3 to 1.5 GHz), 2.0 to
// 2.15 PFLOP/s; 1,024 rows by 4,096 21 to 22 us; gated, 2,045 rows of 4,096 by 2 x 12,288 205 to 220 us.  Two accumulators of 256 features, taken out and added in turns, made it 1,700 clocks a
// tile of K.
// The clusters are persistent: the copies go on into the next tile while the threads write a finished one.  Tiles are numbered row tile fastest: what runs at one time
// shares few weights, and the rows stay in the second-level cache.  Of rows sorted by expert the features are fastest: an expert's rows and weights are few.
// Warp 0 feeds the weights, 2 the rows, 3 the scales; warp 1 (of the first CTA) issues; warps 4 to 11 take the sums and write them.
#define FP_STAGES(CTAS) ((CTAS) == 2 ? 4 : 3)
#define FP_THREADS 384
#define FP_BLOCK 8192             // a warp's rows on their way out: 32 of 64 features, or of 128 in 16 bits
#define FP_RING 2                 // groups of tiles of K whose scales are there
#define FP_GROUP 8
#define FP_SCALES (128 * 4 + 2 * 16)      // bytes of a tile of K's: 128 rows', three of either tile of weights
#define FP_SMALL 56               // registers of a thread that takes no sums, and of one that does: (128 * 56 + 256 * 224) = 384 * 168
#define FP_LARGE 224

__device__ __forceinline__ unsigned fp_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned fp_map_to(unsigned smem_addr, unsigned rank) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(smem_addr), "r"(rank));
    return r;
}
// A wait that ran out ends the pair's work, not one CTA's alone: the other one's flag too.
template <int CTAS> __device__ __forceinline__ bool fp_give_up(volatile int* abort_flag, int32_t* status) {
    *abort_flag = 1;
    if (CTAS == 2) {
        const unsigned other = fp_map_to(t5_smem(const_cast<int*>(abort_flag)), fp_rank() ^ 1);
        asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(other), "r"(1u) : "memory");
    }
    if (atomicCAS(status, 0, F8_STATUS) == 0) status[1] = blockIdx.x;
    return false;
}
template <int CTAS> __device__ __forceinline__ bool fp_wait(unsigned long long* bar, unsigned parity, int waits, volatile int* abort_flag, int32_t* status) {
    for (int i = 0; i < waits; ++i) {
        if (t5_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
    }
    return fp_give_up<CTAS>(abort_flag, status);
}
// Whether a barrier's phase is complete, without waiting for it; and the wait of a warp that has looked.  A look takes 100 clocks until its answer is there, so what is
// likely to be complete is asked for ahead of what can run without it; a vote over the lanes would take another 45.  All lanes come out of it together:
// what follows are instructions of whole warps.
__device__ __forceinline__ bool fp_look(unsigned long long* bar, unsigned parity) {
    unsigned ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(t5_smem(bar)), "r"(parity) : "memory");
    return ok != 0;
}
template <int CTAS> __device__ __forceinline__ bool fp_wait_warp(bool seen, unsigned long long* bar, unsigned parity, int waits, volatile int* abort_flag, int32_t* status) {
    bool ok = true;
    if (!seen) ok = fp_wait<CTAS>(bar, parity, waits, abort_flag, status);
    __syncwarp();
    return ok;
}
// One lane's word for the warp, if `ok`, without a branch that would part it from the others.  A warp that has given up tells nobody that a place is free: it may not
// have been its turn, and others still read there.
__device__ __forceinline__ void fp_tell(unsigned bar, bool ok) {
    asm volatile("{\n .reg .pred p;\n setp.eq.b32 p, %1, 0;\n @p mbarrier.arrive.shared::cluster.b64 _, [%0];\n}\n" ::"r"(bar), "r"(ok ? threadIdx.x & 31 : 1u) : "memory");
}
// Boxes into this CTA's shared memory, counted on a barrier of the pair's first CTA.
__device__ __forceinline__ void fp_tma_2d(void* dst, const CUtensorMap* map, int x, int y, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::
                     "r"(t5_smem(dst)), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void fp_tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::
                     "r"(t5_smem(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
template <int CTAS> __device__ __forceinline__ void fp_commit_lead(unsigned lead, unsigned long long* bar) {
    if constexpr (CTAS == 1) t5_commit_lead(lead, bar);
    else asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n"
                 " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}\n" ::
                     "r"(t5_smem(bar)), "h"(static_cast<unsigned short>(3)), "r"(lead) : "memory");
}
template <int CTAS> __device__ __forceinline__ void fp_mma_lead(unsigned lead, unsigned d_tmem, unsigned long long a_desc, unsigned long long b_desc, unsigned idesc, unsigned accumulate) {
    if constexpr (CTAS == 1) f8_mma_lead(lead, d_tmem, a_desc, b_desc, idesc, accumulate);
    else asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
                 " @q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::
                     "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
__device__ __forceinline__ void fp_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// The pair's warps meet: nobody signals a CTA that has left.  WHO (a text) keeps the places apart.
#define fp_meet(WHO) asm volatile("// " WHO "\nbarrier.cta.sync.aligned 0;\nbarrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory")
// Whether all of the eight warps that take sums say so.
__device__ __forceinline__ bool fp_all(bool yes) {
    unsigned r;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.and.aligned.pred q, 1, 256, p;\n selp.u32 %0, 1, 0, q;\n}\n"
                 : "=r"(r) : "r"(static_cast<unsigned>(yes)) : "memory");
    return r != 0;
}

// mx_gated (microscaling.cuh) with the fast exponential and reciprocal as they are, off by less than 8 + 1.5 |z| units of 2^-24, of eight values step by step: the products
// wait for 64 of these a thread and tile, which one after the other take 8,000 clocks.  SILU: z = g, no clamps, no shift.
template <bool SILU> __device__ __forceinline__ void fp_gated8(float (&g)[8], float (&u)[8], const MxAct& a, float* out) {
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (!SILU) {
            g[i] = g[i] > a.limit ? a.limit : g[i];
            u[i] = (u[i] > a.limit ? a.limit : u[i] < -a.limit ? -a.limit : u[i]) + a.shift;
            s[i] = g[i] * (a.alpha + a.beta * g[i] * g[i]) * -1.4426950408889634f;
        } else {
            s[i] = g[i] * -1.4426950408889634f;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = t5_ex2(s[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = 1.0f + s[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("rcp.approx.ftz.f32 %0, %0;\n" : "+f"(s[i]));
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = g[i] * s[i] * u[i];
}
// What a tile of the launch is.
struct FpTile {
    int row0, rows;                       // of the pair: first, and how many there are from it on (more than 256 where it goes on)
    int features;                         // number of the 256 features of a matrix
    int tile;                             // number of the first of the two tiles of the weight
};
template <bool GROUPED, int CTAS> __device__ __forceinline__ FpTile fp_tile(const F8Args& a, int t, int row_tiles) {
    if constexpr (GROUPED) {
        const int per = a.tiles / 2, i = t / per, f = t - i * per;
        const int4 item = a.groups.items[i];
        return {item.y, item.z, f, item.x * a.tiles + 2 * f};
    } else {
        const int f = t / row_tiles, r = t - f * row_tiles;
        return {r * 128 * CTAS, a.T - r * 128 * CTAS, f, 2 * f};
    }
}

// SPLIT: gated, and the up features of a tile may lie in two blocks.
template <int MODE, typename TO, bool GROUPED, bool SPLIT, int CTAS>
__global__ void __launch_bounds__(FP_THREADS, 1) f8_pair_kernel(const __grid_constant__ CUtensorMap w_map,
                                                                                         const __grid_constant__ CUtensorMap x_map,
                                                                                         const __grid_constant__ CUtensorMap y_map, const F8Args a, int row_tiles,
                                                                                         int all_tiles) {
    constexpr int STAGES = FP_STAGES(CTAS), W_BYTES = 2 / CTAS * F8_TILE;       // of a stage of weights in this CTA
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* w_s = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
    unsigned char* x_s = w_s + STAGES * W_BYTES;               // [STAGES][128 rows][128]
    unsigned char* out_s = x_s + STAGES * F8_TILE;             // a block for each of the eight warps
    float* most_s = reinterpret_cast<float*>(out_s);              // gated: [2][2][128]
    unsigned char* scales_s = out_s + 8 * FP_BLOCK;               // [RING]
    __shared__ __align__(8) unsigned long long full[STAGES], empty[STAGES], acc_full[4], acc_empty[4], s_full[FP_RING], s_empty[FP_RING], drained;
    __shared__ unsigned tmem_base_s;
    __shared__ int abort_flag, asked_s[2];                        // asked_s: boxes of weights, of rows that were asked for
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const unsigned rank = __shfl_sync(0xffffffffu, fp_rank(), 0);
    const int cluster = blockIdx.x / CTAS, clusters = gridDim.x / CTAS, ktiles = a.ktiles;
    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) { t5_mbar_init(&full[s], 2); t5_mbar_init(&empty[s], 1); }      // weights and rows
        for (int s = 0; s < 4; ++s) { t5_mbar_init(&acc_full[s], 1); t5_mbar_init(&acc_empty[s], 4 * CTAS); }      // 4 warps of each CTA
        for (int s = 0; s < FP_RING; ++s) { t5_mbar_init(&s_full[s], 32); t5_mbar_init(&s_empty[s], 8); }
        t5_mbar_init(&drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (CTAS == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(t5_smem(&tmem_base_s)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(t5_smem(&tmem_base_s)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
        }
    }
    t5_fence_before();
    __syncthreads();
    fp_cluster_sync();                                            // the other CTA's barriers exist before anyone signals them
    t5_fence_after();
    pdl_invite();                                                 // not before: tensor memory is taken
    const unsigned tmem = __shfl_sync(0xffffffffu, tmem_base_s, 0);
    if (GROUPED || warp != 0) pdl_wait();                         // weights are nobody's output, the items are
    const int tiles = GROUPED ? a.groups.counts[0] * (a.tiles / 2) : all_tiles;

    // This thread's box (or two of weights: 64 features of either tile, so that an accumulator is a tile) for tile at and tile of K kb, into stage s.
    const unsigned first = fp_map_to(t5_smem(full), 0);           // the first CTA's barriers
    auto ask = [&](const FpTile& at, int kb, int s) {
        if (rank == 0) t5_expect_tx(&full[s], warp == 0 ? 2 * F8_TILE : CTAS * F8_TILE);       // of both CTAs
        if constexpr (CTAS == 1) {
            if (warp == 0)
                for (int w = 0; w < 2; ++w) t5_tma_2d(w_s + s * W_BYTES + w * F8_TILE, &w_map, 0, ((at.tile + w) * ktiles + kb) * 128, &full[s]);
            else f8_tma_3d(x_s + s * F8_TILE, &x_map, 0, at.row0, kb, &full[s]);
            return;
        }
        const unsigned bar = first + s * 8;
        if (warp == 0) {
            const int line = (at.tile * ktiles + kb) * 128 + static_cast<int>(rank) * 64;
            fp_tma_2d(w_s + s * F8_TILE, &w_map, 0, line, bar);
            fp_tma_2d(w_s + s * F8_TILE + F8_TILE / 2, &w_map, 0, line + ktiles * 128, bar);
        } else fp_tma_3d(x_s + s * F8_TILE, &x_map, 0, at.row0 + static_cast<int>(rank) * 128, kb, bar);
    };
    int asked = 0;                                                // boxes, in the thread that asks

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(FP_SMALL));
        if (warp == 0 || warp == 2) {
            if (lane == 0) {
                int s = 0;
                unsigned phase = 1;                               // a barrier that was never used passes for the phase before its first
                bool ok = true;
                int ahead = !GROUPED && warp == 0 ? STAGES : -1;       // boxes of weights that do not wait for the kernel in front
                for (int t = cluster; ok && t < tiles; t += clusters) {
                    const FpTile at = fp_tile<GROUPED, CTAS>(a, t, row_tiles);
#pragma unroll 1
                    for (int kb = 0; kb < ktiles; ++kb) {
                        if (ahead >= 0 && ahead-- == 0) pdl_wait();       // the bounded waits below are not for that kernel
                        if (!fp_wait<CTAS>(&empty[s], phase, a.waits, &abort_flag, a.status)) {
                            asked = (t - cluster) / clusters * ktiles + kb;
                            ok = false;
                            break;
                        }
                        ask(at, kb, s);
                        if (++s == STAGES) s = 0, phase ^= 1;
                    }
                }
                if (ok) asked = tiles > cluster ? (tiles - cluster + clusters - 1) / clusters * ktiles : 0;
                asked_s[warp >> 1] = asked;
                // The products tell both CTAs that they have read a stage, and none may leave before it has been told (of products that stop, the last commit tells).
                if (warp == 0 && ok)
                    for (int i = max(0, asked - STAGES); i < asked; ++i)
                        for (int j = 0; j < T5_WAIT_LIMIT && !t5_try_wait(&empty[i % STAGES], (i / STAGES) & 1) && !*static_cast<volatile int*>(&abort_flag); ++j) {}
            }
            __syncwarp();
        } else if (warp == 1 && rank == 0) {
            const unsigned lead = elect_one();
            const unsigned long long wd = t5_desc(w_s, 16, 1024), xd = t5_desc(x_s, 16, 1024);
            const unsigned idesc = f8_idesc(128 * CTAS, 128);
            int s = 0;
            unsigned phase = 0, buf = 0, acc_phase = 1;
            bool ok = true, seen = false;
            for (int t = cluster; ok && t < tiles; t += clusters) {
#pragma unroll 1
                for (int kb = 0; kb < ktiles; ++kb) {
                    ok = fp_wait_warp<CTAS>(seen, &full[s], phase, a.waits, &abort_flag, a.status) && ok;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        ok = fp_wait_warp<CTAS>(false, &acc_empty[2 * buf + h], acc_phase, a.waits, &abort_flag, a.status) && ok;
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        t5_fence_after();
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            fp_mma_lead<CTAS>(lead, tmem + buf * 256 + h * 128, xd + s * (F8_TILE >> 4) + 2 * k, wd + ((s * W_BYTES + h * (W_BYTES / 2)) >> 4) + 2 * k, idesc, k ? 1u : 0u);
                        if (h == 1) fp_commit_lead<CTAS>(lead, &empty[s]);
                        fp_commit_lead<CTAS>(lead, &acc_full[2 * buf + h]);
                    }
                    if (!ok) break;
                    if (++s == STAGES) s = 0, phase ^= 1;
                    seen = fp_look(&full[s], phase);
                    buf ^= 1;
                    if (buf == 0) acc_phase ^= 1;
                }
            }
        } else if (warp == 3) {
            // A tile of K's scales: four rows a lane, and of the weights' the first six lanes', copied without a register between.
            int slot = 0;
            unsigned phase = 1;
            bool ok = true;
            for (int t = cluster; ok && t < tiles; t += clusters) {
                const FpTile at = fp_tile<GROUPED, CTAS>(a, t, row_tiles);
                const int r0 = at.row0 + static_cast<int>(rank) * 128 + lane;
                const float* cw = a.w_scales + (at.tile * 3LL + min(lane, 5)) * a.k4;
                const float* cx[4];
                int bytes[4];                                     // beyond the last row: zeros
#pragma unroll
                for (int i = 0; i < 4; ++i) bytes[i] = r0 + 32 * i < a.x_rows ? 4 : 0, cx[i] = a.x_scales + (bytes[i] ? (r0 + 32 * i) * static_cast<long long>(a.k4) : 0);
#pragma unroll 1
                for (int kb0 = 0; kb0 < ktiles; kb0 += FP_GROUP) {
                    ok = __all_sync(0xffffffffu, fp_wait<CTAS>(&s_empty[slot], phase, a.waits, &abort_flag, a.status));
                    if (!ok) break;
                    unsigned to = t5_smem(scales_s) + slot * (FP_GROUP * FP_SCALES);
#pragma unroll 1
                    for (int kb = kb0; kb < min(kb0 + FP_GROUP, ktiles); ++kb, to += FP_SCALES) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(to + (lane + 32 * i) * 4), "l"(cx[i] + (bytes[i] ? kb : 0)), "r"(bytes[i]) : "memory");
                        if (lane < 6) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(to + 512 + (lane / 3 * 4 + lane % 3) * 4), "l"(cw + kb) : "memory");
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(t5_smem(&s_full[slot])) : "memory");
                    if (++slot == FP_RING) slot = 0, phase ^= 1;
                }
            }
            asm volatile("cp.async.wait_all;\n" ::: "memory");
        }
        // The two kinds of warps meet at the end from code of their own: what stands behind a place where they come together again is not held to the few registers
        // that these have left.
        __syncwarp();
        t5_fence_before();
        fp_meet("feeding");
        if (*static_cast<volatile int*>(&abort_flag)) {
            // A wait ran out, both CTAs know it, and what is under way ends before they go away.  A barrier fills when all who bring its bytes have asked: those
            // who stopped earlier ask for what the others have asked for already, at most a ring's worth, into places that the products have left
            // (whoever asked first has waited for that).  Then the first CTA's barriers tell when all of it is there, and one more commit when the products are.
            if ((warp == 0 || warp == 2) && lane == 0) {
                int most = 0;
                for (int who = 0; who < 2; ++who)
                    for (unsigned r = 0; r < CTAS; ++r) {
                        int n;
                        asm volatile("ld.shared::cluster.s32 %0, [%1];\n" : "=r"(n) : "r"(fp_map_to(t5_smem(&asked_s[who]), r)) : "memory");
                        most = max(most, n);
                    }
                for (; asked < most; ++asked) ask(fp_tile<GROUPED, CTAS>(a, cluster + asked / ktiles * clusters, row_tiles), asked % ktiles, asked % STAGES);
                if (rank == 0) f8_land_ring(full, STAGES, most);
            } else if (warp == 1) {
                if (rank == 0) fp_commit_lead<CTAS>(elect_one(), &drained);     // the lane that issued: elect gives the same one for the same lanes
                f8_land(&drained, 0);
            }
            __syncwarp();
            fp_meet("feeding");
        }
        if (warp == 1) {
            t5_fence_after();
            if constexpr (CTAS == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
            else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(FP_LARGE));
        const int quarter = warp & 3, half = (warp - 4) >> 2, row = quarter * 32 + lane;
        const unsigned acc_empty_first = fp_map_to(t5_smem(&acc_empty[0]), 0), s_empty_own = fp_map_to(t5_smem(&s_empty[0]), rank);
        unsigned char* block = out_s + (warp - 4) * FP_BLOCK;
        const unsigned from = tmem + (static_cast<unsigned>(quarter * 32) << 16) + half * 128;
        unsigned buf = 0, acc_phase = 0, slot = 0, s_phase = 0, turn = 0;
        for (int t = cluster; t < tiles; t += clusters) {
            const FpTile at = fp_tile<GROUPED, CTAS>(a, t, row_tiles);
            unsigned long long acc[64];                           // two features each
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = 0ull;
            const int split = SPLIT ? f8_split(a.N, 2 * at.features + half) : 64;
            float sx;
            float4 sw;
            auto scales = [&](int kb) {
                const unsigned char* p = scales_s + (slot * FP_GROUP + kb % FP_GROUP) * FP_SCALES;
                sx = *reinterpret_cast<const float*>(p + row * 4);
                sw = *reinterpret_cast<const float4*>(p + 512 + half * 16);
            };
            // One that gives up goes on with what there is, and stores nothing.
            bool ok = fp_wait_warp<CTAS>(false, &s_full[slot], s_phase, a.waits, &abort_flag, a.status);
            scales(0);
            ok = fp_wait_warp<CTAS>(false, &acc_full[2 * buf + half], acc_phase, a.waits, &abort_flag, a.status) && ok;
            t5_fence_after();
            unsigned r[2][32];
            t5_ld32(from + buf * 256, r[0]);
#pragma unroll 1
            for (int kb = 0; kb < ktiles; ++kb) {
                // The wait for numbers waits for all that a thread has asked for.  So what the next tile of K needs (its scales, whether its accumulator is full) is asked
                // for together with them, with additions in between.
                const bool last = kb + 1 == ktiles, group_ends = kb % FP_GROUP == FP_GROUP - 1 || last;
                const float s0 = sx * sw.x, s1 = MODE == F8_GATED ? sx * sw.y : s0, s2 = SPLIT ? sx * sw.z : s1;
                const unsigned long long first_64 = t5_two(s0, s0), other_64 = t5_two(s1, s1);
                auto add = [&](int c) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int f = (c - 2) * 32 + 2 * i;       // of the up features
                        const unsigned long long s = c < 2 ? first_64 : SPLIT ? t5_two(f < split ? s1 : s2, f + 1 < split ? s1 : s2) : other_64;
                        acc[c * 16 + i] = t5_fma2(t5_two(__uint_as_float(r[c & 1][2 * i]), __uint_as_float(r[c & 1][2 * i + 1])), s, acc[c * 16 + i]);
                    }
                };
                const unsigned now = from + buf * 256;
                t5_wait_ld();
                t5_ld32(now + 32, r[1]);
                bool seen_s = true;
                if (group_ends) {
                    __syncwarp();
                    fp_tell(s_empty_own + slot * 8, ok);
                    if (++slot == FP_RING) slot = 0, s_phase ^= 1;
                    if (!last) seen_s = fp_look(&s_full[slot], s_phase);
                }
                add(0);
                t5_wait_ld();
                t5_ld32(now + 64, r[0]);
                if (!last) {
                    if (group_ends) ok = fp_wait_warp<CTAS>(seen_s, &s_full[slot], s_phase, a.waits, &abort_flag, a.status) && ok;
                    scales(kb + 1);
                }
                add(1);
                t5_wait_ld();
                t5_ld32(now + 96, r[1]);
                unsigned long long* const next = &acc_full[2 * (buf ^ 1) + half];
                const unsigned next_phase = buf ? acc_phase ^ 1 : acc_phase;
                const bool seen = last || fp_look(next, next_phase);
                add(2);
                t5_wait_ld();
                // All of it is in registers: the accumulator is free again, with a quarter of the additions still to do.
                t5_fence_before();
                __syncwarp();
                fp_tell(acc_empty_first + (2 * buf + half) * 8, ok);
                buf ^= 1;
                acc_phase = next_phase;
                if (!last) {
                    ok = fp_wait_warp<CTAS>(seen, next, next_phase, a.waits, &abort_flag, a.status) && ok;
                    t5_fence_after();
                    t5_ld32(from + buf * 256, r[0]);
                }
                add(3);
            }
            ok = __all_sync(0xffffffffu, ok);
            if constexpr (MODE == F8_GATED) ok = fp_all(ok);      // the two halves of a row meet below: all go on or leave together
            if (!ok) break;                                       // what has not been computed is not stored
            const int valid = min(at.rows - static_cast<int>(rank) * 128 - quarter * 32, 32);        // of the warp's rows
            const long long row0 = at.row0 + static_cast<int>(rank) * 128 + quarter * 32;
            if constexpr (MODE == F8_GATED) {
                float w = 1.0f;
                if (GROUPED && a.on_input && lane < valid) w = a.groups.weights[row0 + lane];
                float v[64];
                unsigned most = 0;
                auto gated = [&](auto silu) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float g[8], u[8];
#pragma unroll
                        for (int j = 0; j < 4; ++j) t5_untwo(acc[i * 4 + j], g[2 * j], g[2 * j + 1]), t5_untwo(acc[32 + i * 4 + j], u[2 * j], u[2 * j + 1]);
                        if (GROUPED)
#pragma unroll
                            for (int j = 0; j < 8; ++j) g[j] *= w, u[j] *= w;
                        fp_gated8<decltype(silu)::value>(g, u, a.act, v + 8 * i);
                    }
                };
                if (a.act.beta == 0.0f && a.act.shift == 0.0f) gated(std::true_type());       // without clamps too (mx_act)
                else gated(std::false_type());
#pragma unroll
                for (int i = 0; i < 64; ++i) most = max(most, mx_abs_bits(v[i]));
                // the other 64 features of the row are another thread's; two places in turn, so that the next tile's need not wait for these to be read
                most_s[(turn * 2 + half) * 128 + row] = __uint_as_float(most);
                asm volatile("bar.sync 1, 256;\n" ::: "memory");
                most = max(most, __float_as_uint(most_s[(turn * 2 + (half ^ 1)) * 128 + row]));
                turn ^= 1;
                const F8Scale s = f8_scale(most);
                if (lane < valid) {
                    const long long to = at.features * a.y_rows + row0 + lane;
                    unsigned char* codes = static_cast<unsigned char*>(a.y) + to * F8_K + half * 64;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        unsigned c[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {             // not settled (f8_blocks.cuh): 2,045 rows of 4,096 by 2 x 12,288 217 to 223 us with it, 4,096 of 1,024 by 2 x 4,096 46 to 51
                            const float* q = v + 16 * i + 4 * j;
                            c[j] = mx_e4m3x4(q[0] * s.inverse, q[1] * s.inverse, q[2] * s.inverse, q[3] * s.inverse);
                        }
                        *reinterpret_cast<uint4*>(codes + i * 16) = make_uint4(c[0], c[1], c[2], c[3]);
                    }
                    if (half == 0) a.y_scales[(row0 + lane) * a.y_k4 + at.features] = s.scale;
                }
            } else {
                // 32 neighbouring features of each of the warp's rows make a block in shared memory, in pieces of 16 bytes that the row number scatters over the banks (the
                // copy engine's swizzle).  The copy engine takes blocks out, adds, and leaves out what is beyond the matrix; rows of an expert that end
                // within these 32, and rows that it cannot address, leave by the lanes.
                constexpr int LINE = 32 * sizeof(TO), PIECES = LINE / 16, BLOCKS = FP_BLOCK / (32 * LINE);       // bytes of a row, its pieces, blocks that there is room for
                float w = 1.0f;
                if (GROUPED && a.groups.weights && lane < valid) w = a.groups.weights[row0 + lane];
                TO* y = static_cast<TO*>(a.y) + row0 * a.N;
                const bool copies = a.vec && (!GROUPED || valid == 32);
                auto place = [&](int r, int piece) { return r * LINE + ((PIECES == 8 ? piece ^ (r & 7) : piece ^ ((r >> 1) & 3)) << 4); };
#pragma unroll
                for (int c0 = 0; c0 < 4; c0 += BLOCKS) {
                    const int first_col = at.features * 256 + half * 128 + c0 * 32, blocks = min((a.N - first_col + 31) / 32, BLOCKS);
                    if (blocks <= 0 || valid <= 0) break;
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");       // the blocks have been read
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < BLOCKS; ++c)
#pragma unroll
                        for (int p = 0; p < PIECES; ++p) {
                            unsigned q[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float lo, hi;
                                if constexpr (sizeof(TO) == 4) {
                                    t5_untwo(acc[(c0 + c) * 16 + p * 2 + i / 2], lo, hi);
                                    q[i] = __float_as_uint((i & 1 ? hi : lo) * (GROUPED ? w : 1.0f));
                                } else {
                                    t5_untwo(acc[(c0 + c) * 16 + p * 4 + i], lo, hi);
                                    q[i] = GROUPED ? t5_pack(lo * w, hi * w) : t5_pack(lo, hi);
                                }
                            }
                            *reinterpret_cast<uint4*>(block + c * (32 * LINE) + place(lane, p)) = make_uint4(q[0], q[1], q[2], q[3]);
                        }
                    if (copies) {
                        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                        __syncwarp();
                        if (lane == 0) {
#pragma unroll
                            for (int c = 0; c < BLOCKS; ++c)
                                if (c < blocks) {
                                    if (MODE == F8_ADD)
                                        asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.bulk_group [%0, {%2, %3}], [%1];\n" ::"l"(&y_map),
                                                     "r"(t5_smem(block + c * (32 * LINE))), "r"(first_col + c * 32), "r"(static_cast<int>(row0)) : "memory");
                                    else
                                        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];\n" ::"l"(&y_map),
                                                     "r"(t5_smem(block + c * (32 * LINE))), "r"(first_col + c * 32), "r"(static_cast<int>(row0)) : "memory");
                                }
                            asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
                        }
                        __syncwarp();
                        continue;
                    }
                    __syncwarp();
#pragma unroll 1
                    for (int c = 0; c < blocks; ++c) {
                        const unsigned char* from_s = block + c * (32 * LINE);
                        if (a.vec) {                              // rows of whole, aligned pieces of 16 bytes
                            constexpr int PIECE = 16 / sizeof(TO);
                            const int p = lane % PIECES, col = first_col + c * 32 + p * PIECE;
#pragma unroll
                            for (int i = 0; i < PIECES; ++i) {
                                const int r = i * (32 / PIECES) + lane / PIECES;
                                if (r >= valid || col >= a.N) continue;
                                uint4 v = *reinterpret_cast<const uint4*>(from_s + place(r, p));
                                uint4* to = reinterpret_cast<uint4*>(y + static_cast<size_t>(r) * a.N + col);
                                if constexpr (MODE == F8_ADD) {
                                    const float4 o = *reinterpret_cast<const float4*>(to);
                                    v.x = __float_as_uint(__uint_as_float(v.x) + o.x), v.y = __float_as_uint(__uint_as_float(v.y) + o.y);
                                    v.z = __float_as_uint(__uint_as_float(v.z) + o.z), v.w = __float_as_uint(__uint_as_float(v.w) + o.w);
                                }
                                *to = v;
                            }
                        } else {
                            const int col = first_col + c * 32 + lane;
                            if (col < a.N)
#pragma unroll 4
                                for (int r = 0; r < valid; ++r) {
                                    TO v = *reinterpret_cast<const TO*>(from_s + place(r, lane * static_cast<int>(sizeof(TO)) / 16) + lane * sizeof(TO) % 16);
                                    TO* to = y + static_cast<size_t>(r) * a.N + col;
                                    if constexpr (MODE == F8_ADD) v += *to;
                                    *to = v;
                                }
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");       // the result is there before this grid is over
        __syncwarp();
        t5_fence_before();
        fp_meet("sums");
        if (*static_cast<volatile int*>(&abort_flag)) fp_meet("sums");
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
#define F8_DEVICES 64
static int f8_device() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < F8_DEVICES ? dev : -1;
}
static int f8_sms(int dev) {
    static int sms[F8_DEVICES] = {0};
    if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms[dev] = 0;
    return sms[dev];
}
// Lets a kernel have its shared memory, once a device (`had`: a flag for each).
template <typename K> static int f8_allow(K kern, size_t smem, int dev, bool* had) {
    if (had[dev]) return LLM_OK;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    had[dev] = e == cudaSuccess;
    return static_cast<int>(e);
}
static bool f8_encoder() {
    CUtensorMap any;
    if (g_t5_state == 0) (void)t5_encode_2d(&any, nullptr, 64, 64, 64, 64);       // finds the driver's entry point
    return g_t5_state > 0;
}
// Codes of weights: lines of 128 bytes.
static bool f8_weight_map(CUtensorMap* map, const void* w, long long lines, int box_lines) {
    if (!f8_encoder() || lines >= (1LL << 31)) return false;
    const cuuint64_t dims[2] = {F8_K, static_cast<cuuint64_t>(lines)}, strides[1] = {F8_K};
    const cuuint32_t box[2] = {F8_K, static_cast<cuuint32_t>(box_lines)}, es[2] = {1u, 1u};
    return g_t5_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(w), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Codes of rows [ktiles][rows][128] in boxes of `box_tiles` x `box_rows` x 128.
static bool f8_rows_map(CUtensorMap* map, const void* x, long long rows, int ktiles, int box_rows, int box_tiles) {
    if (!f8_encoder() || rows >= (1LL << 31)) return false;
    const cuuint64_t dims[3] = {F8_K, static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(ktiles)}, strides[2] = {F8_K, static_cast<cuuint64_t>(rows) * F8_K};
    const cuuint32_t box[3] = {F8_K, static_cast<cuuint32_t>(box_rows), static_cast<cuuint32_t>(box_tiles)}, es[3] = {1u, 1u, 1u};
    return g_t5_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(x), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Into how many parts K is cut: the most, up to 8 (a cluster), with which all clusters run at once.  One or two CTAs an SM, less an eighth, because clusters do not
// fill a group of SMs to the last slot.
static int f8_parts(long long tiles, int ktiles, int sms, int ctas) {
    const int slots = ctas * sms * 7 / 8;
    int best = 1;
    while (best < 8 && (best + 1) * tiles <= slots && ktiles / (best + 1) >= 2) ++best;
    return best;
}
// A weight as the host knows it: what its products need of it, the copy engine's maps included, put together once (llm_f8_describe).
struct F8Weight {
    CUtensorMap whole, halves;            // its codes in boxes of a tile, of half a tile
    const void* codes;
    const float* scales;
    int E, N, K, tiles, gated, ready;     // N: of a matrix; gated: of its gate; tiles: of 128 rows of a matrix
};
struct F8Call {
    const F8Weight* w;
    const void* x;                        // rows of 8 bits
    int row_tiles;                        // tiles of rows, or room for items
};
template <int NT, int WS, int G, bool PLAIN, int MODE, typename TO, bool GROUPED> static int f8_few(const F8Call& c, const F8Args& a, cudaStream_t s) {
    constexpr int WT = MODE == F8_GATED ? 2 : 1;
    CUtensorMap x_map = {};
    if (!PLAIN && !f8_rows_map(&x_map, c.x, a.x_rows, a.ktiles, NT, G)) return LLM_REFUSED_SIZE;
    constexpr size_t smem = static_cast<size_t>(WS) * WT * F8_TILE + 2 * G * NT * (F8_K + sizeof(float)) + 1024;
    static_assert(NT * 128 * sizeof(float) <= WS * F8_TILE, "the sums fit the weights' stages");
    static_assert(smem * F8_FEW_CTAS(NT, WT) <= 226 * 1024, "an SM's shared memory");
    auto kern = f8_few_kernel<NT, WS, G, PLAIN, MODE, TO, GROUPED>;
    static bool had[F8_DEVICES];
    const int dev = f8_device();
    if (dev < 0) return LLM_REFUSED_SIZE;
    if (const int rc = f8_allow(kern, smem, dev, had)) return rc;
    const int tiles = (MODE == F8_GATED ? a.tiles / 2 : (a.N + 127) / 128), sms = f8_sms(dev);
    if (tiles > 65535 || c.row_tiles > 65535 || sms <= 0) return LLM_REFUSED_SIZE;
    const bool joins = GROUPED && MODE == F8_STORE && a.groups.ids;
    const int parts = joins ? a.groups.top : f8_parts(static_cast<long long>(tiles) * c.row_tiles, a.ktiles, sms, F8_FEW_CTAS(NT, WT));
    launch_pdl_cluster(kern, dim3(parts, tiles, c.row_tiles), dim3(F8_FEW_THREADS(PLAIN, WT)), smem, s, parts, c.w->whole, x_map, a);
    return launch_status();
}
template <int MODE, typename TO, bool GROUPED, bool SPLIT, int CTAS> static int f8_pair(const F8Call& c, F8Args a, cudaStream_t s) {
    CUtensorMap x_map, y_map = {};
    const int dev = f8_device();
    if (dev < 0 || f8_sms(dev) < 2) return LLM_REFUSED_SIZE;
    if (!f8_rows_map(&x_map, c.x, a.x_rows, a.ktiles, 128, 1)) return LLM_REFUSED_SIZE;
    if (MODE != F8_GATED) {                                       // [T, N] in boxes of 32 rows of 32 features
        a.vec = a.vec && a.N * sizeof(TO) % 16 == 0;
        const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.N), static_cast<cuuint64_t>(a.T)}, strides[1] = {static_cast<cuuint64_t>(a.N) * sizeof(TO)};
        const cuuint32_t box[2] = {32, 32}, es[2] = {1u, 1u};
        if (a.vec && g_t5_encode(&y_map, sizeof(TO) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.y, dims, strides, box, es,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, sizeof(TO) == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return LLM_REFUSED_SIZE;
    }
    constexpr size_t smem = static_cast<size_t>(FP_STAGES(CTAS)) * (2 / CTAS + 1) * F8_TILE + 8 * FP_BLOCK + FP_RING * FP_GROUP * FP_SCALES + 1024;
    static_assert(smem <= 227 * 1024 - 256, "shared memory of an SM");
    static_assert(128 * FP_SMALL + 256 * FP_LARGE <= FP_THREADS * 168, "registers of the launch");
    auto kern = f8_pair_kernel<MODE, TO, GROUPED, SPLIT, CTAS>;
    static bool had[F8_DEVICES];
    if (const int rc = f8_allow(kern, smem, dev, had)) return rc;
    const long long all = static_cast<long long>(c.row_tiles) * (a.tiles / 2);
    const int slots = f8_sms(dev) / CTAS;
    if (all > (1LL << 30)) return LLM_REFUSED_SIZE;
    const int clusters = all < slots ? static_cast<int>(all) : slots;
    launch_pdl_cluster(kern, dim3(CTAS * clusters), dim3(FP_THREADS), smem, s, CTAS, CTAS == 2 ? c.w->halves : c.w->whole, x_map, y_map, a, c.row_tiles, static_cast<int>(all));
    return launch_status();
}

// How a product of T rows by `tiles` of 128 of the weight's rows runs: the rows of a tile.  Up to 32 rows one tile of rows reads the weight once.  Tiles of 64 rows go on as long
// as every tile of rows and weight has an SM to itself; K is cut where SMs are left, which the others do not do.  Of these, CTAs of 128 rows alone take 6/5 of the time that pairs of
// 256 rows take for a tile of 256 features, but twice as many run at once: whoever needs less time for all.  Measured, rows of 8 bits, by tiles of 64, 128 and 256 (us): 64 rows of 4,096 by
// 24,576 26.7, 24.1, 33.4; 65 by 6,144 15.1, 20.8, 17.5; 128 by 24,576 49, 26.4, 37.0; 197 by 6,144 25.8, 21.4, 18.6; 256 by 4,096 15.2, 21.3, 18.5; 256 rows of 12,288 by 4,096 35.6, 53.4, 43.5; 384 of
// 4,096 by 24,576 114, 50.0, 58.5; 512 160, 73.5, 65.4; 1,024 by 4,096 (128 and 256) 23.8, 22.0; 2,048 43.7, 39.7; 65 rows of 2,048 by 12,288 15.1, 12.5, 12.0; 384 29.5, 14.0, 20.8; 197 rows of 1,358 by
// 2,501 7.4, 12.2, 11.6; 512 12.6, 12.3, 11.8; gated, 128 rows of 4,096 by 2 x 12,288 54.9, 25.0, 35.8; 256 86.5, 44.8, 38.0; 384 of 1,358 by 2 x 1,450 13.7, 12.0, 12.4.
static int f8_tile_rows(int T, int tiles, int sms) {
    if (T <= 32) return T <= 16 ? 16 : 32;
    if (static_cast<long long>((T + 63) / 64) * tiles <= sms) return 64;
    const long long wide = (tiles + 1) / 2;                       // tiles of 256 features
    const long long alone = ((T + 127) / 128 * wide + sms - 1) / sms, paired = ((T + 255) / 256 * wide + sms / 2 - 1) / (sms / 2);       // rounds
    return 6 * alone < 5 * paired ? 128 : 256;
}

template <int MODE, typename TO, bool GROUPED> static int f8_way(F8Call c, const F8Args& a, int per, cudaStream_t s) {         // per: rows of an item
    if (!GROUPED) {
        const int dev = f8_device();
        if (dev < 0) return LLM_REFUSED_SIZE;
        per = f8_tile_rows(a.T, (MODE == F8_GATED ? 2 : 1) * ((a.N + 127) / 128), f8_sms(dev));
        c.row_tiles = (a.T + per - 1) / per;
    }
    if (per == 256) return MODE == F8_GATED && a.N % 64 ? f8_pair<MODE, TO, GROUPED, MODE == F8_GATED, 2>(c, a, s) : f8_pair<MODE, TO, GROUPED, false, 2>(c, a, s);
    if (per == 128) return MODE == F8_GATED && a.N % 64 ? f8_pair<MODE, TO, GROUPED, MODE == F8_GATED, 1>(c, a, s) : f8_pair<MODE, TO, GROUPED, false, 1>(c, a, s);
    if constexpr (MODE == F8_GATED) {
        if (per == 16) return a.plain ? f8_few<16, 3, 2, true, MODE, TO, GROUPED>(c, a, s) : f8_few<16, 3, 2, false, MODE, TO, GROUPED>(c, a, s);
        if constexpr (!GROUPED) return per == 32 ? f8_few<32, 3, 1, false, MODE, TO, GROUPED>(c, a, s) : f8_few<64, 5, 2, false, MODE, TO, GROUPED>(c, a, s);
    } else {
        if constexpr (!GROUPED)
            if (a.plain) return f8_few<16, 5, 4, true, MODE, TO, false>(c, a, s);
        if (per == 16) return f8_few<16, 5, 4, false, MODE, TO, GROUPED>(c, a, s);
        if constexpr (!GROUPED) return per == 32 ? f8_few<32, 5, 2, false, MODE, TO, GROUPED>(c, a, s) : f8_few<64, 4, 2, false, MODE, TO, GROUPED>(c, a, s);
    }
    return LLM_REFUSED_SIZE;                                      // items have 16, 128 or 256 rows
}

extern "C" int llm_f8_weight_size() { return static_cast<int>(sizeof(F8Weight)); }
// room: llm_f8_weight_size() bytes on the host, 64-byte aligned; codes, scales: of a stack of E matrices of N rows (gated: N gate and N up rows).
extern "C" int llm_f8_describe(void* room, const void* codes, const void* scales, int E, int N, int K, int gated) {
    if (reinterpret_cast<uintptr_t>(room) % 64 || !aligned16(codes) || !aligned16(scales)) return LLM_REFUSED_ALIGN;
    if (E <= 0 || N <= 0 || N > (1 << 22) || K <= 0 || K > (1 << 20)) return LLM_REFUSED_SIZE;
    F8Weight w = {};
    w.codes = codes, w.scales = static_cast<const float*>(scales);
    w.E = E, w.N = N, w.K = K, w.gated = gated, w.tiles = gated ? 2 * ((N + 127) / 128) : (N + 255) / 256 * 2;
    const long long lines = static_cast<long long>(E) * w.tiles * f8_tiles(K) * 128;
    if (!f8_weight_map(&w.whole, codes, lines, 128) || !f8_weight_map(&w.halves, codes, lines, 64)) return LLM_REFUSED_SIZE;
    w.ready = 1;
    *static_cast<F8Weight*>(room) = w;
    return LLM_OK;
}

static bool f8_takes_plain(const void* plain, int dtype, int T, int K, bool gated) { return T <= F8_PLAIN_ROWS(gated) && dtype == LLM_DT_BF16 && K % 8 == 0 && aligned16(plain); }
static int f8_args(F8Args* a, const F8Weight* w, int gated, const void* rows, long long padded, int T, int waits, int32_t* status) {
    if (!w || !w->ready || w->gated != gated || status == nullptr || T > (1 << 24)) return LLM_REFUSED_SIZE;
    if (!aligned16(rows)) return LLM_REFUSED_ALIGN;
    if (rows && padded < T) return LLM_REFUSED_SIZE;
    *a = {};
    a->w_scales = w->scales;
    a->N = w->N, a->K = w->K, a->ktiles = f8_tiles(w->K), a->k4 = f8_k4(w->K), a->y_k4 = f8_k4(w->N), a->tiles = w->tiles;
    a->x_scales = rows ? f8_row_scales(const_cast<void*>(rows), padded, a->ktiles) : nullptr, a->x_rows = padded;
    a->T = T, a->waits = waits, a->status = status;
    return LLM_OK;
}
// The rows of a product's x: those that are there; made of the matrix `plain` where there is room for them; or none, and the product makes them.
static int f8_operand(F8Args* a, void* rows, long long padded, const void* plain, int dtype, bool gated, uintptr_t stream) {
    if (!plain) return rows ? LLM_OK : LLM_REFUSED_ALIGN;
    if (rows) return llm_f8_rows(plain, dtype, rows, padded, a->T, a->K, nullptr, 1, stream);
    if (!f8_takes_plain(plain, dtype, a->T, a->K, gated)) return LLM_REFUSED_ALIGN;
    a->plain = static_cast<const bf16*>(plain);
    return LLM_OK;
}

// rows: of 8 bits [T, K], `padded` of them, or room for them (null: none, for up to F8_PLAIN_ROWS of a bfloat16 matrix of whole, aligned pieces of eight values) and
// `plain` a matrix [T, K] of `dtype`; y: [T, N] float32 or bfloat16; add: y (float32) holds a summand already.
extern "C" int llm_linear_f8(const void* weight, void* rows, long long padded, const void* plain, int dtype, void* y, int out_dtype, int add, int T, int waits,
                             int32_t* status, uintptr_t stream) {
    if (T <= 0) return LLM_OK;
    if (out_dtype != LLM_DT_F32 && (out_dtype != LLM_DT_BF16 || add)) return LLM_REFUSED_DTYPE;
    const F8Weight* w = static_cast<const F8Weight*>(weight);
    F8Args a;
    if (const int rc = f8_args(&a, w, 0, rows, padded, T, waits, status)) return rc;
    if (const int rc = f8_operand(&a, rows, padded, plain, dtype, false, stream)) return rc;
    a.y = y;
    a.vec = a.N % 4 == 0 && aligned16(y);
    const F8Call c = {w, rows, 0};
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (add) return f8_way<F8_ADD, float, false>(c, a, 0, s);
    return out_dtype == LLM_DT_F32 ? f8_way<F8_STORE, float, false>(c, a, 0, s) : f8_way<F8_STORE, bf16, false>(c, a, 0, s);
}

// weight gated; made: act(x gate^T) * (x up^T) as rows of 8 bits [T, N], `made_padded` of them.
extern "C" int llm_linear_f8_silu_mul(const void* weight, void* rows, long long padded, const void* plain, int dtype, void* made, long long made_padded, int T, int act,
                                      float limit, int waits, int32_t* status, uintptr_t stream) {
    if (T <= 0) return LLM_OK;
    const F8Weight* w = static_cast<const F8Weight*>(weight);
    F8Args a;
    if (const int rc = f8_args(&a, w, 1, rows, padded, T, waits, status)) return rc;
    if (!mx_act(act, limit, &a.act) || made_padded < T) return LLM_REFUSED_SIZE;
    if (!aligned16(made)) return LLM_REFUSED_ALIGN;
    if (const int rc = f8_operand(&a, rows, padded, plain, dtype, true, stream)) return rc;
    a.y = made, a.y_rows = made_padded;
    a.y_scales = f8_row_scales(made, made_padded, f8_tiles(a.N));
    return f8_way<F8_GATED, float, false>({w, rows, 0}, a, 0, reinterpret_cast<cudaStream_t>(stream));
}

// Tokens whose picks stay as they are: two launches instead of five, and nothing to sort or add up.  An expert that several of them pick is read once for each, from the second
// time on out of the second-level cache.  Measured, as they are and sorted (us), 1, 2, 4, 5 and 8 tokens: 64 experts, 8 a token, 1,024 by 2,048 15.7 and 22.2, 21.6 and 30.1, 35.5 and 40.5,
// 51.9 and 48.3, 66.4 and 52.5; 8 experts, 2 a token, 2,048 by 4,096 18.5 and 21.2, 23.1 and 28.6, 28.7 and 32.3, 43.7 and 36.6, 47.7 and 41.7.  Up to eight picks: a cluster adds them up.
#define F8_UNSORTED_TOKENS 4
static bool f8_unsorted(int T, int top, bool plain) { return plain && T <= F8_UNSORTED_TOKENS && top <= 8; }
// Routed experts: picks sorted by expert, gate and up, down, each token's rows added up.  x [T, K] of `dtype`; ids, weights [T, top]; out and base as for llm_f8_add_up.
// work: room for, each from a multiple of 256 bytes on, the sorting's results (llm_moe_f8_work has the sizes), rows of x (none where the picks stay as they are: the product makes them), the
// middle's rows, the experts' results in float32 (none where the picks stay as they are).
// Rows of an item, by how many picks an expert has on average.  Measured, with 16, 128 and 256 rows (us): 64 experts, 8 a token, 1,024 by 2,048, 6 picks an expert 85, 99, 130; 12: 101, 106,
// 143; 24: 129, 114, 153; 64: 240, 122, 163; 128 (128 and 256 rows): 156, 175; 256: 246, 269; 375: 334, 343; 512: 434, 440; 1,024: 789, 762.  8 experts, 2 a token, 2,048 by 4,096, 12: 49, 55, 73; 24: 59, 55,
// 75; 40: 82, 58, 77; 64: 102, 61, 81; 256: 128, 125; 512: 183, 191; 750: 264, 267; 1,024: 346, 321; 2,048: 641, 605; 1,450 by 1,358, 12: 29, 38, 47; 24: 32, 37, 46; 40: 33, 38; 64: 49, 39, 48; 512: 91, 91; 1,024:
// 135, 133; 512 by 1,024, 24: 20, 23; 64: 23, 26; 256: 54, 30, 31.  4 experts, 1 a token, 4,096 by 2,048, 512: 96, 106; 1,024: 172, 158.  The rule looks at picks alone: with 17 to 64 of them, small matrices would
// take 10 to 15 % less by items of 16 rows, large ones take 7 to 50 % less as it is.  Items of 32 rows come out between 16 and 128, those of 64 behind.
static int f8_item_rows(long long picks, int E) { return picks <= 16LL * E ? 16 : picks <= 768LL * E ? 128 : 256; }
static long long f8_up(long long n) { return (n + 255) / 256 * 256; }
struct F8Work {
    int per, room;
    long long counts, places, weights, x, middle, y, all;
};
static F8Work f8_work(int T, int top, int E, int W, int ff, bool plain) {
    const long long picks = static_cast<long long>(T) * top;
    F8Work k = {};
    k.per = f8_unsorted(T, top, plain) ? 16 : f8_item_rows(picks, E);
    k.room = static_cast<int>((E < picks ? E : picks) + picks / k.per);
    const long long padded = f8_padded_rows(picks);
    auto rows_bytes = [&](int n) { return padded * (f8_tiles(n) * F8_K + f8_k4(n) * 4LL); };
    k.counts = f8_up(16LL * k.room);
    k.places = k.counts + 256, k.weights = k.places + f8_up(4 * picks);
    k.x = k.weights + f8_up(4 * picks);
    k.middle = k.x + (f8_unsorted(T, top, plain) ? 0 : f8_up(rows_bytes(W)));
    k.y = k.middle + f8_up(rows_bytes(ff));
    k.all = k.y + (f8_unsorted(T, top, plain) ? 0 : picks * W * 4);
    return k;
}
static bool f8_plain_experts(const void* x, int dtype, int W) { return dtype == LLM_DT_BF16 && W % 8 == 0 && aligned16(x); }
extern "C" long long llm_moe_f8_work(const void* x, int dtype, int T, int top, int E, int W, int ff) {
    return f8_work(T, top, E, W, ff, f8_plain_experts(x, dtype, W)).all;
}
extern "C" int llm_f8_sort(const int32_t*, const float*, int, int, int, int32_t*, void*, int32_t*, float*, uintptr_t);
extern "C" int llm_f8_add_up(const float*, const int32_t*, const float*, void*, int, int, int, int, uintptr_t);
extern "C" int llm_moe_f8(const void* gate_up, const void* down, const void* x, int dtype, const int32_t* ids, const float* weights, int T, int top, void* work,
                          const float* base, void* out, int out_dtype, int act, float limit, int on_input, int waits, int32_t* status, uintptr_t stream) {
    if (T <= 0) return LLM_OK;
    if (top <= 0 || static_cast<long long>(T) * top > (1 << 24)) return LLM_REFUSED_SIZE;
    if (out_dtype != LLM_DT_F32 && out_dtype != LLM_DT_BF16) return LLM_REFUSED_DTYPE;
    if (reinterpret_cast<uintptr_t>(work) % 256) return LLM_REFUSED_ALIGN;
    const F8Weight *g = static_cast<const F8Weight*>(gate_up), *d = static_cast<const F8Weight*>(down);
    if (!g || !d || g->E != d->E || g->E > F8_MOST_EXPERTS || g->N != d->K || g->K != d->N) return LLM_REFUSED_SIZE;
    const int picks = T * top, W = g->K, ff = g->N;
    const bool plain = f8_plain_experts(x, dtype, W), unsorted = f8_unsorted(T, top, plain);
    const F8Work k = f8_work(T, top, g->E, W, ff, plain);
    unsigned char* at = static_cast<unsigned char*>(work);
    int32_t *counts = reinterpret_cast<int32_t*>(at + k.counts), *places = reinterpret_cast<int32_t*>(at + k.places);
    float* row_weights = reinterpret_cast<float*>(at + k.weights);
    const long long padded = f8_padded_rows(picks);
    void* x_rows = unsorted ? nullptr : at + k.x;
    if (!unsorted) {
        if (const int rc = llm_f8_sort(ids, weights, picks, g->E, k.per, counts, at, places, row_weights, stream)) return rc;
        if (const int rc = llm_f8_rows(x, dtype, x_rows, padded, T, W, places, top, stream)) return rc;
    }
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    F8Args a;
    if (const int rc = f8_args(&a, g, 1, x_rows, padded, picks, waits, status)) return rc;
    if (!mx_act(act, limit, &a.act)) return LLM_REFUSED_SIZE;
    a.plain = unsorted ? static_cast<const bf16*>(x) : nullptr;
    a.y = at + k.middle, a.y_rows = padded, a.y_scales = f8_row_scales(at + k.middle, padded, f8_tiles(ff));
    const F8Groups groups = {unsorted ? ids : nullptr, top, g->E, counts, reinterpret_cast<const int4*>(at), unsorted ? weights : row_weights};
    a.groups = groups;
    a.on_input = on_input;
    if (const int rc = f8_way<F8_GATED, float, true>({g, x_rows, unsorted ? picks : k.room}, a, k.per, s)) return rc;
    if (const int rc = f8_args(&a, d, 0, at + k.middle, padded, picks, waits, status)) return rc;
    a.y = unsorted ? out : at + k.y;
    a.vec = W % 4 == 0 && aligned16(a.y);
    a.groups = groups;
    if (on_input) a.groups.weights = nullptr;
    a.base = base;
    const F8Call c = {d, at + k.middle, unsorted ? T : k.room};
    if (unsorted && out_dtype == LLM_DT_BF16) return f8_few<16, 5, 4, false, F8_STORE, bf16, true>(c, a, s);
    // Rows stay float32 until a token's are added up, whatever the result's type: picks as they are have their sum rounded once too.
    if (const int rc = f8_way<F8_STORE, float, true>(c, a, k.per, s)) return rc;
    return unsorted ? LLM_OK : llm_f8_add_up(reinterpret_cast<const float*>(at + k.y), places, base, out, out_dtype, T, W, top, stream);
}
// Kernels that llm_moe_f8 launches.
extern "C" int llm_moe_f8_launches(const void* x, int dtype, int T, int top, int W) { return f8_unsorted(T, top, f8_plain_experts(x, dtype, W)) ? 2 : 5; }
