// y[T, N] = x[T, K] . w[N, K]^T of microscaled operands: rows of 8 bits, weights of 4 (microscaling.cuh has the formats), for any
// number of rows, on the block-scaled products of the 5th-generation tensor cores (tcgen05.mma.kind::mxf8f6f4.block_scale).
//
//   y[t, n] = sum over blocks b of sx[t, b] * sw[n, b] * (sum over the 32 values of b of x * w)
// The products of e4m3 and e2m1 values and powers of two are exact; the sums are kept in float32.
//
// The weights are the left operand (128 features a tile), the tokens the right one (NT of them), so that no lane is spent on tokens
// that are not there.  A stage is 128 values of K: a box of the weight's tile (8 KB; the copy engine spreads its 4-bit codes over
// 16 KB, sixteen of them and eight bytes of nothing, as the products read them, and counts the 8 KB on its barrier), a box of the rows, and
// the pieces of both operands' scales, which the tensor core copies to its own memory in front of the stage's four products.
// Roles of single CTAs: warp 0 feeds the weights and their scales, warp 1 issues, warps 2 to 5 take the sums, warp 6 feeds the rows and theirs; all of them write
// the result.  Of a pair's CTA: warp 0 feeds the weights, 10 the rows and 11 the scales, warp 1 of the first CTA issues, 2 to 5 and 6 to 9 write the result
// in turns.  Waits are bounded: one that runs out sets status code 9, and the copies and products that are under way then end, which is waited for
// on their own barriers (bounded too), before the CTA does; sums that are not there are not stored, nor added to a stream.
//   * Few rows: bytes bound the product.  K is cut over a cluster's CTAs, which add their sums up in each other's shared memory in the
//     parts' order; nothing is left for another kernel and no result depends on timing.  The first weights are on their way before the
//     CTA waits for the kernel in front.
//   * Gate and up: a tile is 64 gate features and the 64 up features beside them; act(gate) * up leaves as rows of 8 bits.
#include "microscaling.cuh"
#include "tcgen05_attention.cuh"

#define MG_ROWS 128               // features of a tile (gated: 64 of both)
#define MG_MAKERS 9               // warps that make rows of a matrix
#define MG_THREADS(PLAIN) (32 * (2 + ((PLAIN) ? MG_MAKERS : 5)))
#define MG_W_BYTES (MG_ROWS * MX_K)       // of a stage's weights in shared memory
#define MG_W_READ (MG_W_BYTES / 2)        // the same as the copy engine counts them: what it reads
#define MG_STATUS 9

__device__ __forceinline__ bool mg_wait(unsigned long long* bar, unsigned parity, int waits, volatile int* abort_flag, int32_t* status) {
    for (int i = 0; i < waits; ++i) {
        if (t5_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
    }
    *abort_flag = 1;
    if (atomicCAS(status, 0, MG_STATUS) == 0) status[1] = blockIdx.y;
    return false;
}
// What was asked for before a wait ran out: its end.
__device__ __forceinline__ void mg_land(unsigned long long* bar, unsigned parity) {
    for (int i = 0; i < T5_WAIT_LIMIT && !t5_try_wait(bar, parity); ++i) {}
}
// The uses of a ring's barriers that may be under way, of `asked` in all.
__device__ __forceinline__ void mg_land_ring(unsigned long long* bars, int ring, int asked) {
    for (int i = max(0, asked - ring); i < asked; ++i) mg_land(&bars[i % ring], (i / ring) & 1);
}
__device__ __forceinline__ void mg_tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, unsigned long long* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(t5_smem(dst)), "l"(map),
                 "r"(x), "r"(y), "r"(z), "r"(t5_smem(bar)) : "memory");
}
// A piece of scales to tensor memory: 32 lanes of 16 bytes, repeated in every quarter of the lanes.
__device__ __forceinline__ void mg_scales_lead(unsigned lead, unsigned tmem, unsigned long long desc) {
    asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n @q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n}\n" ::"r"(tmem), "l"(desc), "r"(lead) : "memory");
}
__device__ __forceinline__ void mg_mma_lead(unsigned lead, unsigned d_tmem, unsigned long long a_desc, unsigned long long b_desc, unsigned idesc,
                                            unsigned a_scales, unsigned b_scales, unsigned accumulate) {
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %6, 0;\n setp.ne.b32 q, %7, 0;\n"
                 " @q tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::
                     "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate), "r"(lead) : "memory");
}
// 32 lanes of 16 bytes without a swizzle, groups of eight lanes 128 bytes apart.
__device__ __forceinline__ unsigned long long mg_scale_desc(const void* smem) {
    return static_cast<unsigned long long>((t5_smem(smem) & 0x3FFFF) >> 4) | (static_cast<unsigned long long>(128 >> 4) << 32) | (1ull << 46);
}
// Instruction descriptor: A e2m1, B e4m3, both K-major, scales powers of two; `block`: which of the four scales of a word, for both.
__host__ __device__ constexpr unsigned mg_idesc(int m, int n, unsigned block) {
    return (block << 4) | (5u << 7) | (0u << 10) | (static_cast<unsigned>(n >> 3) << 17) | (1u << 23) | (static_cast<unsigned>(m >> 4) << 24) | (block << 29);
}

struct MgArgs {
    const unsigned char *w_scales, *x_scales;
    void* y;                              // [T, N]; gated: the codes [T, out_kpad]
    unsigned char* y_scales;              // gated
    int T, N, ktiles, out_kpad, vec, waits;
    int32_t* status;
    MxAct act;
    const void* plain;                    // a bfloat16 matrix [T, K] that the kernel takes to 8 bits itself
    int K;
};
enum { MG_STORE = 0, MG_ADD = 1, MG_GATED = 2 };

// grid (parts of K, tiles of features, tiles of tokens), a cluster the parts of a tile.  WS: stages of weights; G: stages whose rows and scales
// come together, two such groups at a time.
// PLAIN: x comes as a matrix, and the warps that will take the sums make the rows of 8 bits of their part of K in shared memory first: one launch
// and no rows in memory, for steps so short that every CTA can do it while its weights come.
template <int NT, int WS, int G, bool PLAIN, int MODE, typename TO>
__global__ void __launch_bounds__(MG_THREADS(PLAIN), 2) linear_mx_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                                                                               const __grid_constant__ CUtensorMap ws_map,
                                                                               const __grid_constant__ CUtensorMap xs_map, const MgArgs a) {
    constexpr int THREADS = MG_THREADS(PLAIN);
    constexpr unsigned X_BYTES = NT * MX_K, S_BYTES = G * MX_PIECE, GROUP_BYTES = G * X_BYTES + 2 * S_BYTES;
    constexpr unsigned S_COL0 = NT < 32 ? 32 : NT, COLS = 128;
    static_assert(S_COL0 + 2 * G * 8 <= COLS, "tensor memory");
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* w_s = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
    unsigned char* g_s = w_s + WS * MG_W_BYTES;                   // [2][G rows' boxes [NT][128], 128-byte swizzle like the weights; weights' pieces, rows' pieces]
    float* sums = reinterpret_cast<float*>(w_s);                  // [NT][128], when the stages have been read
    // a group's weights' scales and its rows have barriers of their own: each is waited for by itself where the other was never asked for
    __shared__ __align__(8) unsigned long long full[WS], empty[WS], gw_full[2], gx_full[2], g_empty[2], acc_full, drained, fed;
    __shared__ unsigned tmem_base_s;
    __shared__ int abort_flag, asked_s[2];                        // asked_s: stages of weights, groups of rows that were asked for
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int part = blockIdx.x, parts = gridDim.x, tile = blockIdx.y, tok0 = blockIdx.z * NT;
    const int kb0 = part * a.ktiles / parts, kbs = (part + 1) * a.ktiles / parts - kb0, early = min(min(WS, 2 * G), kbs);
    const int toks = min(NT, a.T - tok0);
    auto weights = [&](int kb, int s) {                           // into stage s; with the first of a group all of its scales
        const int at = tile * a.ktiles + kb0 + kb;
        if (kb % G == 0) {                                        // what stands behind the part's last stage is read and not used
            const int g = (kb / G) & 1;
            t5_expect_tx(&gw_full[g], S_BYTES);
            t5_tma_2d(g_s + g * GROUP_BYTES + G * X_BYTES, &ws_map, 0, at, &gw_full[g]);
        }
        t5_expect_tx(&full[s], MG_W_READ);
        t5_tma_2d(w_s + s * MG_W_BYTES, &w_map, 0, at * MG_ROWS, &full[s]);
    };
    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < WS; ++s) { t5_mbar_init(&full[s], 1); t5_mbar_init(&empty[s], 1); }
        for (int s = 0; s < 2; ++s) { t5_mbar_init(&gw_full[s], 1); t5_mbar_init(&gx_full[s], PLAIN ? MG_MAKERS : 1); t5_mbar_init(&g_empty[s], 1); }
        t5_mbar_init(&acc_full, 1);
        t5_mbar_init(&drained, 1);
        t5_mbar_init(&fed, PLAIN ? 1 : 2);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        // Weights and their scales are nobody's output: the first of them are on their way before anything else, whatever runs in front.
        for (int kb = 0; kb < early; ++kb) weights(kb, kb);
    }
    if (warp == 6 && lane == 0 && !PLAIN) {
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&x_map) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&xs_map) : "memory");
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
                const int g = kb / G;
                if (kb % G == 0 && !mg_wait(&g_empty[g & 1], ((g >> 1) & 1) ^ 1, a.waits, &abort_flag, a.status)) break;
                if (!mg_wait(&empty[s], phase, a.waits, &abort_flag, a.status)) break;
                weights(kb, s);
                issued = kb + 1;
                if (++s == WS) s = 0, phase ^= 1;
            }
            asked_s[0] = issued;
            t5_arrive(&fed);
        }
        __syncwarp();
    } else if (warp == 6 && !PLAIN) {
        if (lane == 0) {
            int issued = 0;
            pdl_wait();
#pragma unroll 1
            for (int g = 0; g * G < kbs; ++g) {
                unsigned char* to = g_s + (g & 1) * GROUP_BYTES;
                if (!mg_wait(&g_empty[g & 1], ((g >> 1) & 1) ^ 1, a.waits, &abort_flag, a.status)) break;
                t5_expect_tx(&gx_full[g & 1], G * X_BYTES + S_BYTES);
                mg_tma_3d(to, &x_map, 0, tok0, kb0 + g * G, &gx_full[g & 1]);
                t5_tma_2d(to + G * X_BYTES + S_BYTES, &xs_map, 0, (tok0 / 128) * a.ktiles + kb0 + g * G, &gx_full[g & 1]);
                issued = g + 1;
            }
            asked_s[1] = issued;
            t5_arrive(&fed);
        }
        __syncwarp();
    } else if (warp == 1) {
        const unsigned lead = elect_one();
        const unsigned long long wd = t5_desc(w_s, 16, 1024), xd = t5_desc(g_s, 16, 1024), sd = mg_scale_desc(g_s + G * X_BYTES);
        const unsigned off = tok0 % 128 / 32;                     // the tile's first token in its piece of scales
        bool ok = true;
        pdl_wait();                                               // the bounded waits below are not for the kernel in front
        int s = 0;
        unsigned phase = 0;
#pragma unroll 1
        for (int k0 = 0; ok && k0 < kbs; k0 += G) {
            const int g = (k0 / G) & 1;
            const unsigned turn = (k0 / G >> 1) & 1;
            ok = __all_sync(0xffffffffu, mg_wait(&gw_full[g], turn, a.waits, &abort_flag, a.status) && mg_wait(&gx_full[g], turn, a.waits, &abort_flag, a.status));
            if (!ok) break;
            // [weights, rows] of each stage; the products that read the group before last have run
            const unsigned sc0 = tmem + S_COL0 + g * (G * 8);
#pragma unroll
            for (int q = 0; q < G; ++q)
#pragma unroll
                for (int p = 0; p < 2; ++p) mg_scales_lead(lead, sc0 + 8 * q + 4 * p, sd + ((g * GROUP_BYTES + p * S_BYTES + q * MX_PIECE) >> 4));
#pragma unroll 1
            for (int q = 0; q < min(G, kbs - k0); ++q) {
                ok = __all_sync(0xffffffffu, mg_wait(&full[s], phase, a.waits, &abort_flag, a.status));
                if (!ok) break;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mg_mma_lead(lead, tmem, wd + s * (MG_W_BYTES >> 4) + 2 * k, xd + ((g * GROUP_BYTES + q * X_BYTES) >> 4) + 2 * k, mg_idesc(MG_ROWS, NT, k),
                                sc0 + 8 * q, sc0 + 8 * q + 4 + off, (k0 | q | k) ? 1u : 0u);
                t5_commit_lead(lead, &empty[s]);
                if (++s == WS) s = 0, phase ^= 1;
            }
            if (ok) t5_commit_lead(lead, &g_empty[g]);
        }
        t5_commit_lead(lead, ok ? &acc_full : &drained);          // drained: what was issued has ended, and that was not all
    } else {
        pdl_wait();
        if constexpr (PLAIN) {                                    // warps 2 to 10; rows beyond T keep what stands there, nobody minds
            // A warp takes two stages of a row at a time, sixteen lanes each, and has the next group's values on their way while it makes this one's.
            static_assert(G % 2 == 0, "stages go in pairs");
            constexpr int BATCH = (NT * G / 2 + MG_MAKERS - 1) / MG_MAKERS;       // units of a group that a warp has at most
            const int p = lane & 15, units = a.T * (G / 2);
            const bf16* x = static_cast<const bf16*>(a.plain) + kb0 * MX_K + (lane >> 4) * MX_K + p * 8;
            const int left = a.K - kb0 * MX_K - (lane >> 4) * MX_K - p * 8;       // values of the row from the lane's first on
            uint4 raw[BATCH];
            auto fetch = [&](int g) {
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    const int u = warp - 2 + j * MG_MAKERS, at = (g * G + u % (G / 2) * 2) * MX_K;
                    raw[j] = u < units && at < left ? *reinterpret_cast<const uint4*>(x + static_cast<size_t>(u / (G / 2)) * a.K + at) : make_uint4(0u, 0u, 0u, 0u);
                }
            };
            fetch(0);
#pragma unroll 1
            for (int g = 0; g * G < kbs; ++g) {
                unsigned char* to = g_s + (g & 1) * GROUP_BYTES;
                if (!__all_sync(0xffffffffu, mg_wait(&g_empty[g & 1], ((g >> 1) & 1) ^ 1, a.waits, &abort_flag, a.status))) break;
                uint4 now[BATCH];
#pragma unroll
                for (int j = 0; j < BATCH; ++j) now[j] = raw[j];
                fetch(g + 1);                                     // beyond the part: not used, and beyond the row not read
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    const int u = warp - 2 + j * MG_MAKERS, r = u / (G / 2), q = u % (G / 2) * 2 + (lane >> 4);
                    if (u >= units) break;                        // for the whole warp
                    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&now[j]);
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 f = __bfloat1622float2(h[i]);
                        v[2 * i] = f.x, v[2 * i + 1] = f.y;
                    }
                    unsigned word;
                    const uint2 c = mx_encode8<MX_E4M3>(v, word);
                    // the 128-byte swizzle: 16-byte piece i of row r at i ^ (r % 8)
                    *reinterpret_cast<uint2*>(to + q * X_BYTES + r * MX_K + (((p >> 1) ^ (r & 7)) << 4) + (p & 1) * 8) = c;
                    if (p == 0) *reinterpret_cast<unsigned*>(to + G * X_BYTES + S_BYTES + q * MX_PIECE + (r & 31) * 16 + (r >> 5) * 4) = word;
                }
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) t5_arrive(&gx_full[g & 1]);
            }
        }
        if (warp < 6) {
            const int quarter = warp & 3, row = quarter * 32 + lane;
            const bool ok = __all_sync(0xffffffffu, mg_wait(&acc_full, 0, a.waits, &abort_flag, a.status));
            t5_fence_after();
            if (ok) {
#pragma unroll 1
                for (int c = 0; c < NT / 16; ++c) {
                    unsigned r[16];
                    t5_ld16(tmem + (static_cast<unsigned>(quarter * 32) << 16) + 16 * c, r);
                    t5_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (16 * c + i < toks) sums[(16 * c + i) * MG_ROWS + row] = __uint_as_float(r[i]);
                }
            } else {
                // A wait ran out.  Who asks for copies has stopped; the copies (the stages are where the sums go) and the products end; then NaNs tell
                // whoever adds the parts up that these sums are not there.  Nothing of it is in the way of a product that does not give up.
                mg_land(&fed, 0);
                mg_land_ring(full, WS, asked_s[0]);
                mg_land_ring(gw_full, 2, (asked_s[0] + G - 1) / G);
                if (!PLAIN) mg_land_ring(gx_full, 2, asked_s[1]);
                for (int i = 0; i < T5_WAIT_LIMIT && !t5_try_wait(&drained, 0) && !t5_try_wait(&acc_full, 0); ++i) {}
                for (int i = 0; i < toks; ++i) sums[i * MG_ROWS + row] = __uint_as_float(0x7fffffffu);
            }
        }
    }
    t5_fence_before();
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    // What the warp's first token is added to is on its way while the parts meet (an 8B-shape decode step of 32 requests 2.24 ms, 2.27 without).
    const int feature = tile * MG_ROWS + 4 * lane, first_tok = part + warp * parts;
    float4 old = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if constexpr (MODE == MG_ADD) {
        pdl_wait();                                               // the warps that feed weights have not
        if (a.vec && first_tok < toks && feature < a.N) old = *reinterpret_cast<const float4*>(static_cast<const float*>(a.y) + static_cast<size_t>(tok0 + first_tok) * a.N + feature);
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");       // every part's sums are there
    {
        const unsigned base = t5_smem(sums);
        auto total = [&](int at) {                                // the parts' sums in order, four features, all parts' loads in flight at once
            float4 f[8];
#pragma unroll
            for (int p = 0; p < 8; ++p)
                if (p < parts) {
                    unsigned addr;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(addr) : "r"(base + 4u * at), "r"(p));
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(f[p].x), "=f"(f[p].y), "=f"(f[p].z), "=f"(f[p].w) : "r"(addr));
                }
            float4 v = f[0];
#pragma unroll
            for (int p = 1; p < 8; ++p)
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
        if constexpr (MODE == MG_GATED) {
            // sixteen lanes a token, four features a lane, eight lanes a block
            const int f = 4 * (tid & 15), step = THREADS / 16 * parts;
            unsigned char* codes = static_cast<unsigned char*>(a.y);
#pragma unroll 1
            for (int t0 = 0; t0 < toks; t0 += step) {
                const int tok = t0 + part + (tid >> 4) * parts;
                const bool there = tok < toks;
                const float4 g = total((there ? tok : 0) * MG_ROWS + f), u = total((there ? tok : 0) * MG_ROWS + 64 + f);
                unsigned scale;
                const unsigned made = mx_gated_codes<true>(g, u, a.act, scale);
                if (there && !missing(g.x + u.x)) {               // for all of a block's lanes
                    const size_t t = tok0 + tok;
                    *reinterpret_cast<unsigned*>(codes + t * a.out_kpad + tile * 64 + f) = made;
                    if ((tid & 7) == 0) a.y_scales[mx_scale_at(t, (tile * 64 + f) / MX_BLOCK, a.out_kpad / MX_K)] = static_cast<unsigned char>(scale);
                }
            }
        } else {
            TO* y = static_cast<TO*>(a.y);
            const int f = feature;
#pragma unroll 2
            for (int tok = first_tok; f < a.N && tok < toks; tok += THREADS / 32 * parts) {
                const float4 t = total(tok * MG_ROWS + 4 * lane);
                if (missing(t.x)) continue;
                float ts[4] = {t.x, t.y, t.z, t.w};
                TO* to = y + static_cast<size_t>(tok0 + tok) * a.N + f;
                if (a.vec) {                                      // N a multiple of 4, y aligned
                    if constexpr (sizeof(TO) == 4) {
                        float4 v = t;
                        if (MODE == MG_ADD) {
                            const float4 o = tok == first_tok ? old : *reinterpret_cast<const float4*>(to);
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
                        if (f + i < a.N) to[i] = from_f32<TO>(MODE == MG_ADD ? ts[i] + to_f32(to[i]) : ts[i]);
                }
            }
        }
    }
    __syncwarp();
    // Nobody leaves while its sums are read.  A thread that is here has all that it read, because it has made what it stored of it, or has seen that it is
    // NaN and of a part that gave up; the stores themselves need not be out yet, which a release would wait for (one row x 4,096 by 6,144 5.5 us, 5.8 with it; an 8B-shape
    // decode step of 4 requests 1.82 ms, 1.87).
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    if (warp == 1) {
        t5_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(COLS) : "memory");
    }
}

// ---- many rows: pairs of CTAs ---------------------------------------------------------------------------------------
// The two CTAs of a cluster compute a tile of 256 features x NT tokens together (cta_group::2): each brings its own 128 features and half
// of the tokens, and reads both halves.  The clusters are persistent and hold two accumulators, so that a tile's result is written under the
// next one's products; 192 tokens at most leave room for both and for two groups of scales in tensor memory.  Tiles are numbered token tile
// fastest: what runs at one time shares few weights, and the rows stay in the second-level cache.
#define MP_NT 192                 // most tokens of a tile; a launch takes as many as waste least (mp_width)
#define MP_STAGES 6
#define MP_THREADS 384            // weights, products, 4 + 4 warps for the results, rows, scales
#define MP_X_BYTES (MP_NT / 2 * MX_K)
#define MP_QUAD 4                                                 // stages whose scales come together, two such groups at a time
#define MP_S_BYTES (MP_QUAD * 3 * MX_PIECE)                       // own weights' scales, then both pieces of the rows'
#define MP_S_COLS (MP_QUAD * 12)
#define MP_TURN 8192                                              // a block of sums on their way out

__device__ __forceinline__ unsigned mp_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned mp_map_to(unsigned smem_addr, unsigned rank) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(smem_addr), "r"(rank));
    return r;
}
// A wait that ran out ends the pair's work, not one CTA's alone: the other one's flag too.
__device__ __forceinline__ bool mp_give_up(volatile int* abort_flag, int32_t* status) {
    *abort_flag = 1;
    const unsigned other = mp_map_to(t5_smem(const_cast<int*>(abort_flag)), mp_rank() ^ 1);
    asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(other), "r"(1u) : "memory");
    if (atomicCAS(status, 0, MG_STATUS) == 0) status[1] = blockIdx.x;
    return false;
}
__device__ __forceinline__ bool mp_wait(unsigned long long* bar, unsigned parity, int waits, volatile int* abort_flag, int32_t* status) {
    for (int i = 0; i < waits; ++i) {
        if (t5_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
    }
    return mp_give_up(abort_flag, status);
}
__device__ __forceinline__ bool mp_wait_cluster(unsigned long long* bar, unsigned parity, int waits, volatile int* abort_flag, int32_t* status) {
    for (int i = 0; i < waits; ++i) {
        unsigned ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(ok) : "r"(t5_smem(bar)), "r"(parity) : "memory");
        if (ok) return true;
        if (*abort_flag) return false;
    }
    return mp_give_up(abort_flag, status);
}
// Boxes into this CTA's shared memory, counted on a barrier of the pair's first CTA.
__device__ __forceinline__ void mp_tma_2d(void* dst, const CUtensorMap* map, int x, int y, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::
                     "r"(t5_smem(dst)), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void mp_tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::
                     "r"(t5_smem(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void mp_commit_lead(unsigned lead, unsigned long long* bar) {
    asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n"
                 " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}\n" ::
                     "r"(t5_smem(bar)), "h"(static_cast<unsigned short>(3)), "r"(lead) : "memory");
}
__device__ __forceinline__ void mp_scales_lead(unsigned lead, unsigned tmem, unsigned long long desc) {
    asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n @q tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n}\n" ::"r"(tmem), "l"(desc), "r"(lead) : "memory");
}
__device__ __forceinline__ void mp_mma_lead(unsigned lead, unsigned d_tmem, unsigned long long a_desc, unsigned long long b_desc, unsigned idesc,
                                            unsigned a_scales, unsigned b_scales, unsigned accumulate) {
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %6, 0;\n setp.ne.b32 q, %7, 0;\n"
                 " @q tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::
                     "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate), "r"(lead) : "memory");
}
// Whether all of the four warps at this barrier say so.
__device__ __forceinline__ bool mp_all(bool yes, int bar) {
    unsigned r;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.and.aligned.pred q, %2, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
                 : "=r"(r) : "r"(static_cast<unsigned>(yes)), "r"(bar) : "memory");
    return r != 0;
}
__device__ __forceinline__ void mp_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

template <int MODE, typename TO>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MP_THREADS, 1) linear_mx_pair_kernel(
    const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap ws_map,
    const __grid_constant__ CUtensorMap xs_map, const __grid_constant__ CUtensorMap y_map, const MgArgs a, int nt, int token_tiles, int tiles) {
    constexpr int CHUNK = MP_TURN / (MG_ROWS * sizeof(TO));       // tokens of a block
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* w_s = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
    unsigned char* x_s = w_s + MP_STAGES * MG_W_BYTES;            // [STAGES][96 tokens][128]
    unsigned char* s_s = x_s + MP_STAGES * MP_X_BYTES;            // [2][the weights' QUAD pieces, the rows' two times QUAD]
    float* turns_s = reinterpret_cast<float*>(s_s + 2 * MP_S_BYTES);      // two blocks for each half of the result's warps
    __shared__ __align__(8) unsigned long long full[MP_STAGES], empty[MP_STAGES], s_full[2], s_empty[2], acc_full[2], acc_empty[2], drained;
    __shared__ unsigned tmem_base_s;
    __shared__ int abort_flag, asked_s[3];                        // asked_s: boxes of weights, of rows and groups of scales that were asked for
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const unsigned rank = __shfl_sync(0xffffffffu, mp_rank(), 0);
    const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1, ktiles = a.ktiles;
    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < MP_STAGES; ++s) { t5_mbar_init(&full[s], 2); t5_mbar_init(&empty[s], 1); }      // weights and rows
        for (int s = 0; s < 2; ++s) {
            t5_mbar_init(&s_full[s], 1);
            t5_mbar_init(&s_empty[s], 1);
            t5_mbar_init(&acc_full[s], 1);
            t5_mbar_init(&acc_empty[s], 16);                      // 8 warps of 2 CTAs
        }
        t5_mbar_init(&drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(t5_smem(&tmem_base_s)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    }
    t5_fence_before();
    __syncthreads();
    mp_cluster_sync();                                            // the other CTA's barriers exist before anyone signals them
    t5_fence_after();
    pdl_invite();                                                 // not before: tensor memory is taken
    const unsigned tmem = __shfl_sync(0xffffffffu, tmem_base_s, 0);
    if (warp != 0) pdl_wait();                                    // weights are nobody's output

    // One box of this thread's (of weights, rows or scales) for tile t and from stage kb on, into place s of its ring.
    const bool feeds_scales = warp == 11;
    unsigned long long* const own = feeds_scales ? s_full : full;
    const unsigned first = mp_map_to(t5_smem(own), 0);            // the first CTA's barriers
    const int ring = feeds_scales ? 2 : MP_STAGES, step = feeds_scales ? MP_QUAD : 1;
    const unsigned bytes = 2 * (feeds_scales ? MP_S_BYTES : warp == 0 ? MG_W_READ : nt / 2 * MX_K);      // of both CTAs
    auto ask = [&](int tok0, int at, int kb, int s) {
        if (rank == 0) t5_expect_tx(&own[s], bytes);
        const unsigned bar = first + s * 8;
        if (warp == 0) mp_tma_2d(w_s + s * MG_W_BYTES, &w_map, 0, (at + kb) * MG_ROWS, bar);
        else if (warp == 10) mp_tma_3d(x_s + s * MP_X_BYTES, &x_map, 0, tok0 + static_cast<int>(rank) * (nt / 2), kb, bar);
        else {                                                    // what stands behind the last tile of K is read and not used
            mp_tma_2d(s_s + s * MP_S_BYTES, &ws_map, 0, at + kb, bar);
            mp_tma_3d(s_s + s * MP_S_BYTES + MP_QUAD * MX_PIECE, &xs_map, 0, kb, tok0 / 128, bar);
        }
    };
    const int steps = (ktiles + step - 1) / step;                 // of a tile
    int asked = 0;                                                // boxes, or groups of scales, in the thread that asks

    if (warp == 0 || warp >= 10) {
        // Three threads feed: the weights (warp 0), the rows (10) and the scales (11).  Asking for a box takes a thread 80 clocks and a
        // turn of the loop 150 more; one thread for all of a stage took 650, its four products 400.
        if (lane == 0) {
            unsigned long long* free = feeds_scales ? s_empty : empty;
            int s = 0;
            unsigned phase = 1;                                   // a barrier that was never used passes for the phase before its first
            bool ok = true;
            int ahead = warp == 0 ? MP_STAGES : -1;               // boxes of weights that do not wait for the kernel in front
            for (int t = cluster; ok && t < tiles; t += clusters) {
                const int tok0 = (t % token_tiles) * nt, at = ((t / token_tiles) * 2 + static_cast<int>(rank)) * ktiles;
#pragma unroll 1
                for (int kb = 0; kb < ktiles; kb += step) {
                    if (ahead >= 0 && ahead-- == 0) pdl_wait();   // the bounded waits below are not for that kernel
                    if (!mp_wait(&free[s], phase, a.waits, &abort_flag, a.status)) {
                        asked = (t - cluster) / clusters * steps + kb / step;
                        ok = false;
                        break;
                    }
                    ask(tok0, at, kb, s);
                    if (++s == ring) s = 0, phase ^= 1;
                }
            }
            if (ok) asked = (tiles - cluster + clusters - 1) / clusters * steps;
            asked_s[warp == 0 ? 0 : warp - 9] = asked;
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            const unsigned lead = elect_one();
            const unsigned long long wd = t5_desc(w_s, 16, 1024), xd = t5_desc(x_s, 16, 1024), sd = mg_scale_desc(s_s);
            const unsigned idesc = mg_idesc(2 * MG_ROWS, nt, 0);
            int s = 0, n = 0, quad = 0;
            unsigned phase = 0;
            bool ok = true;
            for (int t = cluster; ok && t < tiles; t += clusters, ++n) {
                const int buf = n & 1;
                const unsigned off = ((t % token_tiles) * nt % 128) / 32;        // the tile's first token in its piece of scales
                if (n >= 2) ok = __all_sync(0xffffffffu, mp_wait_cluster(&acc_empty[buf], ((n >> 1) - 1) & 1, a.waits, &abort_flag, a.status));
                t5_fence_after();
#pragma unroll 1
                for (int k0 = 0; ok && k0 < ktiles; k0 += MP_QUAD, ++quad) {
                    const int qs = quad & 1;
                    ok = __all_sync(0xffffffffu, mp_wait(&s_full[qs], (quad >> 1) & 1, a.waits, &abort_flag, a.status));
                    if (!ok) break;
                    // [weights, rows' first piece, rows' second] of each stage; products that read the group before last have run
                    const unsigned sc0 = tmem + 2 * MP_NT + qs * MP_S_COLS;
#pragma unroll
                    for (int q = 0; q < MP_QUAD; ++q)
#pragma unroll
                        for (int p = 0; p < 3; ++p) mp_scales_lead(lead, sc0 + 12 * q + 4 * p, sd + ((qs * MP_S_BYTES + (p * MP_QUAD + q) * MX_PIECE) >> 4));
#pragma unroll 1
                    for (int q = 0; q < min(MP_QUAD, ktiles - k0); ++q) {
                        ok = __all_sync(0xffffffffu, mp_wait(&full[s], phase, a.waits, &abort_flag, a.status));
                        if (!ok) break;
                        const unsigned sc = sc0 + 12 * q;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mp_mma_lead(lead, tmem + buf * MP_NT, wd + s * (MG_W_BYTES >> 4) + 2 * k, xd + s * (MP_X_BYTES >> 4) + 2 * k,
                                        idesc | (static_cast<unsigned>(k) << 4) | (static_cast<unsigned>(k) << 29), sc, sc + 4 + off, (k0 | q | k) ? 1u : 0u);
                        mp_commit_lead(lead, &empty[s]);
                        if (++s == MP_STAGES) s = 0, phase ^= 1;
                    }
                    if (ok) mp_commit_lead(lead, &s_empty[qs]);
                }
                if (ok) mp_commit_lead(lead, &acc_full[buf]);
            }
        }
    } else {                                                      
        // warps 2 to 5 and 6 to 9: two halves that take a tile's blocks of tokens in turn
        const int quarter = warp & 3, half = (warp - 2) >> 2, e = (tid - 64) & 127;
        float* turn = turns_s + half * (2 * MP_TURN / 4);
        const unsigned acc_empty_first = mp_map_to(t5_smem(&acc_empty[0]), 0);
        int n = 0, turns = 0;
        for (int t = cluster; t < tiles; t += clusters, ++n) {
            const int buf = n & 1, tok0 = (t % token_tiles) * nt, wt = (t / token_tiles) * 2 + static_cast<int>(rank);
            const int toks = min(nt, a.T - tok0);
            bool ok = __all_sync(0xffffffffu, mp_wait(&acc_full[buf], (n >> 1) & 1, a.waits, &abort_flag, a.status));
            ok = mp_all(ok, 1 + half);                            // the four warps meet below: they go on or leave together
            if (!ok) break;                                       // what has not been computed is not stored
            t5_fence_after();
            const unsigned acc = tmem + (static_cast<unsigned>(quarter * 32) << 16) + buf * MP_NT;
            if constexpr (MODE == MG_GATED) {
                // 16 tokens at a time through shared memory; then sixteen lanes a token, four features a lane, eight lanes a block
                const int f = 4 * (e & 15);
                unsigned char* codes = static_cast<unsigned char*>(a.y);
#pragma unroll 1
                for (int c = 16 * half; c < toks; c += 32, ++turns) {
                    unsigned r[16];
                    t5_ld16(acc + c, r);
                    t5_wait_ld();
                    float* to = turn + (turns & 1) * (MP_TURN / 4);
#pragma unroll
                    for (int i = 0; i < 16; ++i) to[i * MG_ROWS + quarter * 32 + lane] = __uint_as_float(r[i]);
                    asm volatile("bar.sync %0, 128;\n" ::"r"(1 + half) : "memory");      // with two blocks in turn the next writes wait for this one's reads
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int tok = (e >> 4) + 8 * i;
                        const float4 g = *reinterpret_cast<const float4*>(to + tok * MG_ROWS + f), u = *reinterpret_cast<const float4*>(to + tok * MG_ROWS + 64 + f);
                        unsigned scale;
                        const unsigned made = mx_gated_codes<false>(g, u, a.act, scale);
                        if (c + tok < toks) {
                            const size_t row = tok0 + c + tok;
                            *reinterpret_cast<unsigned*>(codes + row * a.out_kpad + wt * 64 + f) = made;
                            if ((e & 7) == 0) a.y_scales[mx_scale_at(row, (wt * 64 + f) / MX_BLOCK, a.out_kpad / MX_K)] = static_cast<unsigned char>(scale);
                        }
                    }
                }
            } else if (a.vec) {
                // 8 KB at a time through shared memory and out by the copy engine, which also adds and leaves out what is beyond
                // the matrix.  By it and by stores straight from the lanes (a token's 32 features), us, float32 / bfloat16 / added: 4,096 x 1,024 by 6,144
                // 37.5, 39.8 / 31.6, 39.4 / 49.6, 69.6; 700 x 4,096 by 4,096 14.5, 14.9 / 13.9, 15.1 / 15.3, 18.8; 2,048 x 4,096 by 4,096 32.0, 32.4 / 29.9,
                // 30.8 / 35.4, 36.6; 4,096 x 4,096 by 6,144 82.7, 86.2 / 77.0, 78.0 / 90.9, 89.6, and by 24,576, under the power cap, 318, 347 / 316,
                // 318 / 375, 362: only long additions are a little faster from the lanes.
#pragma unroll 1
                for (int c = CHUNK * half; c < toks; c += 2 * CHUNK, ++turns) {
                    unsigned r[CHUNK];
                    if constexpr (CHUNK == 32) t5_ld32(acc + c, r);
                    else t5_ld16(acc + c, r);
                    TO* to = reinterpret_cast<TO*>(turn) + (turns & 1) * (CHUNK * MG_ROWS) + quarter * 32 + lane;
                    if (e == 0) asm volatile("cp.async.bulk.wait_group.read 1;\n" ::: "memory");       // the block before last has been read
                    t5_wait_ld();
                    asm volatile("bar.sync %0, 128;\n" ::"r"(1 + half) : "memory");
#pragma unroll
                    for (int i = 0; i < CHUNK; ++i) to[i * MG_ROWS] = from_f32<TO>(__uint_as_float(r[i]));
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    asm volatile("bar.sync %0, 128;\n" ::"r"(1 + half) : "memory");
                    if (e == 0 && wt * MG_ROWS < a.N) {
                        const unsigned from = t5_smem(to - (quarter * 32 + lane));
                        if (MODE == MG_ADD)
                            asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.bulk_group [%0, {%2, %3}], [%1];\n" ::"l"(&y_map), "r"(from),
                                         "r"(wt * MG_ROWS), "r"(tok0 + c) : "memory");
                        else
                            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];\n" ::"l"(&y_map), "r"(from),
                                         "r"(wt * MG_ROWS), "r"(tok0 + c) : "memory");
                    }
                    if (e == 0) asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
                }
            } else {
                // rows that the copy engine cannot address: a lane is a feature, a token's 32 features leave side by side
                const int f = wt * MG_ROWS + quarter * 32 + lane;
                TO* y = static_cast<TO*>(a.y) + static_cast<size_t>(tok0) * a.N + f;
#pragma unroll 1
                for (int c = 16 * half; c < toks; c += 32) {
                    unsigned r[16];
                    t5_ld16(acc + c, r);
                    float old[16];
                    if (MODE == MG_ADD)
#pragma unroll
                        for (int i = 0; i < 16; ++i) old[i] = f < a.N && c + i < toks ? to_f32(y[static_cast<size_t>(c + i) * a.N]) : 0.0f;
                    t5_wait_ld();
                    if (f < a.N)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (c + i < toks)
                                y[static_cast<size_t>(c + i) * a.N] = from_f32<TO>(MODE == MG_ADD ? old[i] + __uint_as_float(r[i]) : __uint_as_float(r[i]));
                }
            }
            t5_fence_before();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(acc_empty_first + buf * 8) : "memory");
        }
        if (e == 0) asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");       // the result is there before this grid is over
    }
    t5_fence_before();
    __syncthreads();
    mp_cluster_sync();                                            // nobody signals a CTA that has left
    if (abort_flag) {
        // A wait ran out, both CTAs know it, and what is under way ends before they go away.  A barrier fills when all who bring its bytes have asked: those
        // who stopped earlier ask for what the others have asked for already, at most a ring's worth, into places that the products have left
        // (whoever asked first has waited for that).  Then the first CTA's barriers tell when all of it is there, and one more commit when the products are.
        if ((warp == 0 || warp >= 10) && lane == 0) {
            int most = 0;
            for (int who = feeds_scales ? 2 : 0; who < (feeds_scales ? 3 : 2); ++who)
                for (unsigned r = 0; r < 2; ++r) {
                    int n;
                    asm volatile("ld.shared::cluster.s32 %0, [%1];\n" : "=r"(n) : "r"(mp_map_to(t5_smem(&asked_s[who]), r)) : "memory");
                    most = max(most, n);
                }
            for (; asked < most; ++asked) {
                const int t = cluster + asked / steps * clusters;
                ask((t % token_tiles) * nt, ((t / token_tiles) * 2 + static_cast<int>(rank)) * ktiles, asked % steps * step, asked % ring);
            }
            if (rank == 0) mg_land_ring(own, ring, most);
        } else if (warp == 1) {
            if (rank == 0) mp_commit_lead(elect_one(), &drained);         // the lane that issued: elect gives the same one for the same lanes
            mg_land(&drained, 0);
        }
        __syncwarp();
        __syncthreads();
        mp_cluster_sync();
    }
    if (warp == 1) {
        t5_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
#define MG_DEVICES 64
static int mg_device() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < MG_DEVICES ? dev : -1;
}
static int mg_sms(int dev) {
    static int sms[MG_DEVICES] = {0};
    if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms[dev] = 0;
    return sms[dev];
}
// Lets a kernel have its shared memory, once a device (`had`: a flag for each).
template <typename K> static int mg_allow(K kern, size_t smem, int dev, bool* had) {
    if (had[dev]) return LLM_OK;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    had[dev] = e == cudaSuccess;
    return static_cast<int>(e);
}

// 4-bit codes, tiles of 128 rows of 64 bytes, spread by the copy engine.
static bool mg_weight_map(CUtensorMap* map, const void* w, long long rows) {
    CUtensorMap any;
    if (g_t5_state == 0) (void)t5_encode_2d(&any, w, 64, 64, 64, 64);        // finds the driver's entry point
    if (g_t5_state < 0 || rows >= (1LL << 31)) return false;
    const cuuint64_t dims[2] = {MX_K, static_cast<cuuint64_t>(rows)}, strides[1] = {MX_K / 2};
    const cuuint32_t box[2] = {MX_K, MG_ROWS}, es[2] = {1u, 1u};
    return g_t5_encode(map, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, 2, const_cast<void*>(w), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// 8-bit rows [rows, kpad] as [ktiles][rows][128] in boxes of `box_tiles` x `box_rows` x 128 values.
static bool mg_rows_map(CUtensorMap* map, const void* x, int rows, int ktiles, int box_rows, int box_tiles) {
    const cuuint64_t dims[3] = {MX_K, static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(ktiles)}, strides[2] = {static_cast<cuuint64_t>(ktiles) * MX_K, MX_K};
    const cuuint32_t box[3] = {MX_K, static_cast<cuuint32_t>(box_rows), static_cast<cuuint32_t>(box_tiles)}, es[3] = {1u, 1u, 1u};
    return g_t5_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(x), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Pieces of scales as lines of 128 words: [tiles of rows][ktiles] in boxes of `lines` lines, of `box_tiles` neighbouring tiles of rows (three
// dimensions) or of one.
static bool mg_scales_map(CUtensorMap* map, const void* scales, int row_tiles, int ktiles, int lines, int box_tiles) {
    const cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(ktiles), static_cast<cuuint64_t>(row_tiles)};
    const cuuint64_t strides[2] = {MX_PIECE, static_cast<cuuint64_t>(ktiles) * MX_PIECE};
    const cuuint32_t box[3] = {128, static_cast<cuuint32_t>(lines), static_cast<cuuint32_t>(box_tiles)}, es[3] = {1u, 1u, 1u};
    const cuuint64_t line_dims[2] = {128, static_cast<cuuint64_t>(ktiles) * static_cast<cuuint64_t>(row_tiles)};
    if (line_dims[1] >= (1ULL << 31)) return false;
    return g_t5_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, box_tiles ? 3 : 2, const_cast<void*>(scales), box_tiles ? dims : line_dims, strides, box, es,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Into how many parts K is cut: the most, up to 8 (a cluster), with which all clusters run at once.  Two CTAs an SM, less an eighth, because
// clusters do not fill a group of SMs to the last slot: one row x 4,096 by 6,144 in 4 parts 5.9 us, 5 (240 CTAs) 5.7, 6 (288) 9.5; 8 rows x
// 2,048 by 12,288 in one 6.9, two (192) 5.9, three (288) 9.7; 8 rows by 2 x 12,288 (192 tiles) in one 13.3, two 18.0.
static int mg_slots(int sms) { return 2 * sms * 7 / 8; }
static int mg_parts(long long tiles, int ktiles, int slots) {
    int best = 1;
    while (best < 8 && (best + 1) * tiles <= slots && ktiles / (best + 1) >= 2) ++best;
    return best;
}

// How many tokens a pair's tile has: 192, or 128 where the rounds of all tiles take less with them.  A tile of K = 4,096 takes 10.1 us with 192,
// 8.2 with 128, 7.4 with 64 (its weights' way to shared memory then takes longest): nt + 174.  Multiples of 64, because the products take the scales
// of a tile's rows from an even column of tensor memory only.
#define MP_BESIDE 174
static int mp_width(int T, int tiles, int sms, long long* cost) {
    int best = 0;
    for (int nt = MP_NT; nt >= 128; nt -= 64) {
        const long long all = static_cast<long long>((T + nt - 1) / nt) * ((tiles + 1) / 2), c = (all + sms / 2 - 1) / (sms / 2) * (nt + MP_BESIDE);
        if (!best || c < *cost) best = nt, *cost = c;
    }
    return best;
}

// Whether more rows than 64 go to pairs of CTAs, or to tiles of 64 rows each of which reads the weights again but whose K may be cut.  By
// the time that both take, in hundredths of a microsecond beside what they share: a wave of single CTAs 36 a tile of K and 25 a part, a round of
// pairs with 192 tokens 28.  Rows x K by N, us, single / pair: 100 x 4,096 by 4,096 8.5, 13.4; 256 11.3, 13.7; 320 16.3, 13.7; 700 29, 14.3; 160 x
// 4,096 by 6,144 15.8, 13.5; 256 x 12,288 by 4,096 23.7, 29.7; 320 39.5, 29.8; 700 x 1,024 by 1,024 6.2, 7.1; 1,024 x 1,024 by 2,048 7.8, 7.7;
// 128 x 2,048 by 12,288 11.2, 10.0; gated 128 x 4,096 by 2 x 12,288 36.5, 27.1 (64 rows: 21.5).
static bool mg_pairs_pay(int T, int tiles, int ktiles, int sms) {
    if (T <= 64) return false;
    const long long single = static_cast<long long>((T + 63) / 64) * tiles;
    const int parts = mg_parts(single, ktiles, mg_slots(sms));
    const long long waves = (single * parts + 2 * sms - 1) / (2 * sms);
    long long pairs = 0;
    (void)mp_width(T, tiles, sms, &pairs);
    return (T + 63) / 64 > 65535 || 36 * waves * ((ktiles + parts - 1) / parts) + 25 * parts > 28 * pairs * ktiles / (MP_NT + MP_BESIDE);
}

template <int NT, int WS, int G, bool PLAIN, int MODE, typename TO>
static int mg_launch(const void* w, int tiles, const void* x, MgArgs a, cudaStream_t s) {
    CUtensorMap w_map, ws_map, x_map = {}, xs_map = {};
    const int padded = static_cast<int>(mx_padded_rows(a.T)), stored = (tiles + 1) / 2 * 2;
    if (!mg_weight_map(&w_map, w, static_cast<long long>(stored) * a.ktiles * MG_ROWS) || !mg_scales_map(&ws_map, a.w_scales, stored, a.ktiles, G, 0)) return LLM_REFUSED_SIZE;
    if (!PLAIN && (!mg_rows_map(&x_map, x, padded, a.ktiles, NT, G) || !mg_scales_map(&xs_map, a.x_scales, (padded + 127) / 128, a.ktiles, G, 0))) return LLM_REFUSED_SIZE;
    constexpr size_t smem = static_cast<size_t>(WS) * MG_W_BYTES + 2 * G * (NT * MX_K + 2 * MX_PIECE) + 1024;
    static_assert(128 % NT == 0, "a tile's scales are in one piece");
    static_assert(NT * 4 <= WS * MX_K, "the sums fit the weights' stages");
    static_assert(smem <= 113 * 1024, "half of an SM's shared memory");
    auto kern = linear_mx_kernel<NT, WS, G, PLAIN, MODE, TO>;
    static bool had[MG_DEVICES];
    const int dev = mg_device();
    if (dev < 0) return LLM_REFUSED_SIZE;
    if (const int rc = mg_allow(kern, smem, dev, had)) return rc;
    const int tok_tiles = (a.T + NT - 1) / NT, sms = mg_sms(dev);
    if (tiles > 65535 || tok_tiles > 65535 || sms <= 0) return LLM_REFUSED_SIZE;
    const int parts = mg_parts(static_cast<long long>(tiles) * tok_tiles, a.ktiles, mg_slots(sms));
    launch_pdl_cluster(kern, dim3(parts, tiles, tok_tiles), dim3(MG_THREADS(PLAIN)), smem, s, parts, w_map, x_map, ws_map, xs_map, a);
    return launch_status();
}
template <int MODE, typename TO>
static int mp_launch(const void* w, int tiles, const void* x, MgArgs a, cudaStream_t s) {
    CUtensorMap w_map, x_map, ws_map, xs_map, y_map = {};
    const int padded = static_cast<int>(mx_padded_rows(a.T)), stored = (tiles + 1) / 2 * 2, dev = mg_device();
    if (dev < 0 || mg_sms(dev) < 2) return LLM_REFUSED_SIZE;
    long long cost = 0;
    const int nt = mp_width(a.T, tiles, mg_sms(dev), &cost);
    if (!mg_weight_map(&w_map, w, static_cast<long long>(stored) * a.ktiles * MG_ROWS) || !mg_rows_map(&x_map, x, padded, a.ktiles, nt / 2, 1) ||
        !mg_scales_map(&ws_map, a.w_scales, stored, a.ktiles, MP_QUAD, 0) || !mg_scales_map(&xs_map, a.x_scales, padded / 128, a.ktiles, MP_QUAD, 2))
        return LLM_REFUSED_SIZE;
    if (MODE != MG_GATED) {                                       // [T, N] in boxes of 8 KB, 128 values wide
        a.vec = a.vec && a.N * sizeof(TO) % 16 == 0;
        const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.N), static_cast<cuuint64_t>(a.T)}, strides[1] = {static_cast<cuuint64_t>(a.N) * sizeof(TO)};
        const cuuint32_t box[2] = {MG_ROWS, MP_TURN / (MG_ROWS * sizeof(TO))}, es[2] = {1u, 1u};
        if (a.vec && g_t5_encode(&y_map, sizeof(TO) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.y, dims, strides, box, es,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return LLM_REFUSED_SIZE;
    }
    constexpr size_t smem = static_cast<size_t>(MP_STAGES) * (MG_W_BYTES + MP_X_BYTES) + 2 * MP_S_BYTES + 4 * MP_TURN + 1024;
    static_assert(smem <= 227 * 1024 - 256, "shared memory of an SM");
    static_assert(2 * MP_NT + 2 * MP_S_COLS <= 512, "tensor memory");
    auto kern = linear_mx_pair_kernel<MODE, TO>;
    static bool had[MG_DEVICES];
    if (const int rc = mg_allow(kern, smem, dev, had)) return rc;
    const long long token_tiles = (a.T + nt - 1) / nt, all = token_tiles * (stored / 2);
    const int slots = mg_sms(dev) / 2;
    if (all > (1LL << 30)) return LLM_REFUSED_SIZE;
    const int clusters = all < slots ? static_cast<int>(all) : slots;
    launch_pdl(kern, dim3(2 * clusters), dim3(MP_THREADS), smem, s, w_map, x_map, ws_map, xs_map, y_map, a, nt, static_cast<int>(token_tiles), static_cast<int>(all));
    return launch_status();
}
template <int MODE, typename TO> static int mg_rows(const void* w, int tiles, const void* x, const MgArgs& a, cudaStream_t s) {
    if (a.T <= 16) return a.plain ? mg_launch<16, 5, 4, true, MODE, TO>(w, tiles, x, a, s) : mg_launch<16, 5, 4, false, MODE, TO>(w, tiles, x, a, s);
    if (a.T <= 32) return mg_launch<32, 4, 4, false, MODE, TO>(w, tiles, x, a, s);
    const int dev = mg_device(), sms = dev < 0 ? 0 : mg_sms(dev);
    if (sms < 2) return LLM_REFUSED_SIZE;
    return mg_pairs_pay(a.T, tiles, a.ktiles, sms) ? mp_launch<MODE, TO>(w, tiles, x, a, s) : mg_launch<64, 4, 2, false, MODE, TO>(w, tiles, x, a, s);
}

// Rows up to which a product takes a bfloat16 matrix of whole, aligned pieces of eight values to 8 bits itself.
#define MG_PLAIN_ROWS 16
extern "C" int llm_linear_mx_takes(const void* plain, int dtype, int T, int K) { return T <= MG_PLAIN_ROWS && dtype == LLM_DT_BF16 && K % 8 == 0 && aligned16(plain); }

// Checks a product's operands and, where there is room for rows beside a matrix `plain`, makes them.
static int mg_operands(MgArgs* a, void* rows, const void* plain, int dtype, const void* w, const void* w_scales, int T, int N, int K, int waits,
                       int32_t* status, uintptr_t stream) {
    if (N <= 0 || N > (1 << 24) || K <= 0 || K > (1 << 20) || T > (1 << 24)) return LLM_REFUSED_SIZE;
    if (!aligned16(w) || !aligned16(w_scales) || !aligned16(rows) || (reinterpret_cast<uintptr_t>(w) & 31) || status == nullptr) return LLM_REFUSED_ALIGN;
    if (plain && dtype != LLM_DT_F32 && dtype != LLM_DT_BF16) return LLM_REFUSED_DTYPE;
    const bool itself = plain && rows == nullptr;
    if (itself ? !llm_linear_mx_takes(plain, dtype, T, K) : rows == nullptr) return LLM_REFUSED_ALIGN;
    *a = {};
    a->w_scales = static_cast<const unsigned char*>(w_scales);
    a->T = T, a->N = N, a->K = K, a->ktiles = mx_tiles(K), a->waits = waits, a->status = status;
    if (itself) {
        a->plain = plain;
        return LLM_OK;
    }
    a->x_scales = mx_row_scales(rows, T, K);
    return plain ? llm_mx_rows(plain, dtype, rows, T, K, stream) : LLM_OK;
}

// rows: of 8 bits [T, K], or room for them (null: none, where llm_linear_mx_takes) and `plain` a matrix [T, K] of `dtype`; w: a weight of 4 bits
// [N, K]; y: [T, N] float32 or bfloat16; add: y (float32) holds a summand already.
extern "C" int llm_linear_mx(void* rows, const void* plain, int dtype, const void* w, const void* w_scales, void* y, int out_dtype, int add, int T, int N,
                             int K, int waits, int32_t* status, uintptr_t stream) {
    if (T <= 0) return LLM_OK;
    if ((out_dtype != LLM_DT_F32 && out_dtype != LLM_DT_BF16) || (add && out_dtype != LLM_DT_F32)) return LLM_REFUSED_DTYPE;
    MgArgs a;
    if (const int rc = mg_operands(&a, rows, plain, dtype, w, w_scales, T, N, K, waits, status, stream)) return rc;
    a.y = y;
    a.vec = N % 4 == 0 && aligned16(y);
    const int tiles = (N + MG_ROWS - 1) / MG_ROWS;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (add) return mg_rows<MG_ADD, float>(w, tiles, rows, a, s);
    if (out_dtype == LLM_DT_F32) return mg_rows<MG_STORE, float>(w, tiles, rows, a, s);
    return mg_rows<MG_STORE, bf16>(w, tiles, rows, a, s);
}

// w: a gated weight of 4 bits (N gate and N up rows); made: act(x gate^T) * (x up^T) as rows of 8 bits [T, N].
extern "C" int llm_linear_mx_silu_mul(void* rows, const void* plain, int dtype, const void* w, const void* w_scales, void* made, int T, int N, int K,
                                      int act, float limit, int waits, int32_t* status, uintptr_t stream) {
    if (T <= 0) return LLM_OK;
    MxAct form;
    if (!mx_act(act, limit, &form)) return LLM_REFUSED_SIZE;
    if (!aligned16(made)) return LLM_REFUSED_ALIGN;
    MgArgs a;
    if (const int rc = mg_operands(&a, rows, plain, dtype, w, w_scales, T, N, K, waits, status, stream)) return rc;
    const int tiles = 2 * ((N + 127) / 128);                      // as the weight has them
    a.y = made;
    a.y_scales = mx_row_scales(made, T, N);
    a.out_kpad = tiles * 64;
    a.act = form;
    return mg_rows<MG_GATED, float>(w, tiles, rows, a, reinterpret_cast<cudaStream_t>(stream));
}

// How a product of T rows of 8 bits runs: tokens of a pair's tile, or minus those of a single CTA's.
extern "C" int llm_linear_mx_way(int T, int N, int K, int is_gated, int sms) {
    const int tiles = is_gated ? 2 * ((N + 127) / 128) : (N + MG_ROWS - 1) / MG_ROWS;
    long long cost = 0;
    return mg_pairs_pay(T, tiles, mx_tiles(K), sms) ? mp_width(T, tiles, sms, &cost) : T <= 16 ? -16 : T <= 32 ? -32 : -64;
}
