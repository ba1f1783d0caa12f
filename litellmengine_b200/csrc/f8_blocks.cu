// What makes rows and weights of 8 bits under float32 scales (f8_blocks.cuh has the format), what reads them back, and what stands around products
// of rows that are sorted by expert:
//   rows      from a matrix; a row may go to several places, one for each expert that its token has picked
//   weights   from a matrix or a stack of them, gate and up rows 64 by 64 beside each other
//   values    of either, as float32 or bfloat16
//   sorting   (token, choice) pairs by expert, and the experts' rows cut into tiles
//   adding up a token's rows, in the order of its choices
// Everything is bound by memory: each value is read once and each code written once.
//
// No pointer here is __restrict__: a load of what is const and restricted counts as one of constant memory, and may move in front of the wait for the kernel that
// writes it (the sorting's picks did, where several kernels of a step were under way).
#include "f8_blocks.cuh"

#define F8_THREADS 256

// ---- rows from a matrix ---------------------------------------------------------------------------------------------
// Sixteen lanes a block of a row, eight values a lane (16 or 32 bytes); a warp takes U times two blocks, all asked for before the first is used.
// Measured: 4,096 rows of 12,288 in bfloat16 31.2 us (151 MB, 4.8 TB/s), of 4,096 11.5 us, 24 rows of 12,288 1.5 us; in float32 49 us (252 MB, 5.1 TB/s), 18.4, 2.0.
template <typename T> struct F8Raw { typedef uint4 type; };
template <> struct F8Raw<float> { struct type { float v[8]; }; };
__device__ __forceinline__ unsigned f8_most(const uint4& r) { return mx_most8(r); }
__device__ __forceinline__ unsigned f8_most(const F8Raw<float>::type& r) { return mx_most8(r.v); }
__device__ __forceinline__ uint2 f8_codes(const uint4& r, unsigned most, float inverse) { return f8_codes8(r, most, inverse); }
__device__ __forceinline__ uint2 f8_codes(const F8Raw<float>::type& r, unsigned most, float inverse) { return f8_codes8(r.v, most, inverse); }
// vec 8: rows of whole, aligned pieces of eight values; 2: of pairs; 1: any.
template <int VEC> __device__ __forceinline__ void f8_load(const bf16* row, int col, int n, uint4& r) {
    r = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (VEC == 8) {
        if (col < n) mx_raw8(row + col, r);
    } else if constexpr (VEC == 2) {
        unsigned h[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + 2 * i < n) h[i] = *reinterpret_cast<const unsigned*>(row + col + 2 * i);
        r = make_uint4(h[0], h[1], h[2], h[3]);
    } else {
        unsigned short h[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < n) h[i] = __bfloat16_as_ushort(row[col + i]);
        r = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
}
template <int VEC> __device__ __forceinline__ void f8_load(const float* row, int col, int n, F8Raw<float>::type& r) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = 0.0f;
    if constexpr (VEC == 8) {
        if (col < n) load8(row + col, r.v);
    } else if constexpr (VEC == 2) {
#pragma unroll
        for (int i = 0; i < 8; i += 2)
            if (col + i < n) {
                const float2 f = *reinterpret_cast<const float2*>(row + col + i);
                r.v[i] = f.x, r.v[i + 1] = f.y;
            }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < n) r.v[i] = row[col + i];
    }
}

template <int U, int VEC, typename T>
__global__ void __launch_bounds__(F8_THREADS) f8_rows_kernel(const T* x, unsigned char* codes, float* scales, unsigned items,
                                                             unsigned per_row, int K, int ktiles, int k4, long long padded, const int32_t* places, int top) {
    pdl_begin();
    const unsigned w = blockIdx.x * (F8_THREADS / 32) + (threadIdx.x >> 5);
    if (w >= items) return;                                       // whole warps
    const unsigned row = w / per_row;
    const int lane = threadIdx.x & 31, first = (w - row * per_row) * (2 * U) + (lane >> 4);       // of the lane's tiles of K
    typename F8Raw<T>::type raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) f8_load<VEC>(x + static_cast<size_t>(row) * K, (first + 2 * u) * F8_K + (lane & 15) * 8, K, raw[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int kb = first + 2 * u;
        const unsigned most = f8_most16(f8_most(raw[u]));
        const F8Scale s = f8_scale(most);
        const uint2 c = f8_codes(raw[u], most, s.inverse);
        if (kb >= ktiles) continue;
        for (int k = 0; k < top; ++k) {
            const long long to = places ? static_cast<long long>(places[static_cast<size_t>(row) * top + k]) : static_cast<long long>(row);
            if (to < 0) continue;                                 // a pick without an expert
            *reinterpret_cast<uint2*>(codes + (kb * padded + to) * F8_K + (lane & 15) * 8) = c;
            if ((lane & 15) == 0) scales[to * k4 + kb] = s.scale;
        }
    }
}

extern "C" int llm_f8_rows(const void* x, int dtype, void* rows, long long padded, int T, int K, const int32_t* places, int top, uintptr_t stream) {
    if (T <= 0) return LLM_OK;
    if (K <= 0 || K > (1 << 20) || T > (1 << 24) || top <= 0 || padded < T) return LLM_REFUSED_SIZE;
    if (!aligned16(rows)) return LLM_REFUSED_ALIGN;
    const int ktiles = f8_tiles(K), vec = mx_vec(K, x, dtype == LLM_DT_F32 ? 4 : 2);
    // four tiles of K a lane where that leaves every SM with enough warps
    const bool many = static_cast<long long>(T) * ktiles >= 32 * 1024;
    const unsigned u = many ? 4 : 1, per_row = (ktiles + 2 * u - 1) / (2 * u);
    const long long items = static_cast<long long>(T) * per_row;
    if (items >= (1LL << 31)) return LLM_REFUSED_SIZE;
    const dim3 grid(static_cast<unsigned>((items + F8_THREADS / 32 - 1) / (F8_THREADS / 32)));
    unsigned char* codes = static_cast<unsigned char*>(rows);
    float* scales = f8_row_scales(rows, padded, ktiles);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
#define LAUNCH(U, VEC, T_)                                                                                                                       \
    launch_pdl((f8_rows_kernel<U, VEC, T_>), grid, dim3(F8_THREADS), 0, s, static_cast<const T_*>(x), codes, scales, static_cast<unsigned>(items), per_row, K, \
               ktiles, f8_k4(K), padded, places, places ? top : 1)
#define LAUNCH_T(T_)                                        \
    if (many) { if (vec == 8) LAUNCH(4, 8, T_); else if (vec == 2) LAUNCH(4, 2, T_); else LAUNCH(4, 1, T_); } \
    else { if (vec == 8) LAUNCH(1, 8, T_); else if (vec == 2) LAUNCH(1, 2, T_); else LAUNCH(1, 1, T_); }
    if (dtype == LLM_DT_BF16) { LAUNCH_T(bf16) }
    else if (dtype == LLM_DT_F32) { LAUNCH_T(float) }
    else return LLM_REFUSED_DTYPE;
#undef LAUNCH_T
#undef LAUNCH
    return launch_status();
}

// ---- weights --------------------------------------------------------------------------------------------------------
// A CTA a block of 128 x 128: sixteen lanes a row, two rows a warp and trip, eight trips that are asked for together.  It does not invite the kernel behind
// it: products fetch weights before they wait for what is in front of them.  12,288 x 4,096 in bfloat16 26.4 us (151 MB, 5.7 TB/s), in float32 46.3 (252 MB, 5.4 TB/s); 1,003 x 1,358 in float32 4.6
// us, 88 CTAs and bound by latency.
template <int VEC, typename T>
__global__ void __launch_bounds__(F8_THREADS) f8_weight_kernel(const T* w, unsigned char* codes, float* scales, int rows, int K,
                                                               int tiles, int ktiles, int k4, int gate_rows, long long row_stride, long long matrix_stride) {
    __shared__ unsigned most_s[F8_THREADS / 32];
    pdl_wait();
    const int kb = blockIdx.x, block = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T* from = w + blockIdx.z * matrix_stride + static_cast<long long>(block) * 128 * row_stride;
    const int col = kb * F8_K + (lane & 15) * 8, there = rows - block * 128;
    const long long stack = static_cast<long long>(blockIdx.z) * tiles;
    codes += stack * ktiles * F8_TILE + kb * F8_TILE + (lane & 15) * 8;
    scales += stack * 3 * k4 + kb;
    if (gate_rows && there <= 0) {                                // one CTA more: the rows of whole tiles that gate and up do not have
        for (int f = gate_rows + warp * 2 + (lane >> 4); f < tiles * 64; f += F8_THREADS / 16)
            for (int up = 0; up < 2; ++up) *reinterpret_cast<uint2*>(codes + static_cast<long long>(f >> 6) * ktiles * F8_TILE + (up * 64 + (f & 63)) * F8_K) = make_uint2(0u, 0u);
        const int empty = (gate_rows + 63) / 64 + threadIdx.x;    // tiles of nothing else
        if (empty < tiles)
            for (int i = 0; i < 3; ++i) scales[(empty * 3LL + i) * k4] = F8_LEAST;
        return;
    }
    typename F8Raw<T>::type raw[8];
    unsigned most = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int r = u * 16 + warp * 2 + (lane >> 4);
        f8_load<VEC>(from + r * row_stride, col, r < there ? K : 0, raw[u]);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) most = max(most, f8_most(raw[u]));
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) most_s[warp] = most;
    __syncthreads();
    most = 0;
#pragma unroll
    for (int i = 0; i < F8_THREADS / 32; ++i) most = max(most, most_s[i]);
    const F8Scale s = f8_scale(most);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int r = block * 128 + u * 16 + warp * 2 + (lane >> 4), up = gate_rows && r >= gate_rows, f = up ? r - gate_rows : r;
        const int tile = gate_rows ? f >> 6 : r >> 7, at = gate_rows ? up * 64 + (f & 63) : r & 127;
        if (!gate_rows || r < rows)
            *reinterpret_cast<uint2*>(codes + static_cast<long long>(tile) * ktiles * F8_TILE + at * F8_K) = f8_codes(raw[u], most, s.inverse);
    }
    if (!gate_rows) {
        if (threadIdx.x < 3) scales[(block * 3LL + threadIdx.x) * k4] = s.scale;
    } else if (threadIdx.x < 4) {                                 // the tiles whose gate rows, first up row or last up row lie in this block
        const int first = block * 128, i = first / 64 + threadIdx.x, j = (first - gate_rows) / 64 - 1 + static_cast<int>(threadIdx.x);
        if (i * 64 < gate_rows && i * 64 / 128 == block) scales[i * 3LL * k4] = s.scale;
        if (j >= 0 && j * 64 < gate_rows) {
            if ((gate_rows + j * 64) / 128 == block) scales[(j * 3LL + 1) * k4] = s.scale;
            if ((gate_rows + min(j * 64 + 63, gate_rows - 1)) / 128 == block) scales[(j * 3LL + 2) * k4] = s.scale;
        }
    }
}

// N: rows of a matrix (gated: of gate); tiles: of 128 rows as the weight has them, an even number.
extern "C" int llm_f8_weight(const void* w, int dtype, void* codes, void* scales, int E, int N, int K, int tiles, int gated, long long row_stride,
                             long long matrix_stride, uintptr_t stream) {
    if (E <= 0 || E > 65535 || N <= 0 || N > (1 << 22) || K <= 0 || K > (1 << 20) || tiles != (gated ? 2 * ((N + 127) / 128) : (N + 255) / 256 * 2)) return LLM_REFUSED_SIZE;
    if (tiles > 65535 || row_stride < 0 || matrix_stride < 0) return LLM_REFUSED_SIZE;
    if (!aligned16(codes) || !aligned16(scales)) return LLM_REFUSED_ALIGN;
    const int esz = dtype == LLM_DT_F32 ? 4 : 2, strides = static_cast<int>((row_stride | matrix_stride) & 7);
    int vec = mx_vec(K, w, esz);                                  // of rows that lie strides apart
    if (strides) vec = strides % 2 ? 1 : vec < 2 ? 1 : 2;
    const int rows = gated ? 2 * N : N, blocks = gated ? (rows + 127) / 128 + (N % 128 ? 1 : 0) : tiles;
    if (blocks > 65535) return LLM_REFUSED_SIZE;
    const dim3 grid(f8_tiles(K), blocks, E);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
#define LAUNCH(VEC, T_)                                                                                                                              \
    launch_pdl((f8_weight_kernel<VEC, T_>), grid, dim3(F8_THREADS), 0, s, static_cast<const T_*>(w), static_cast<unsigned char*>(codes), \
               static_cast<float*>(scales), rows, K, tiles, f8_tiles(K), f8_k4(K), gated ? N : 0, row_stride, matrix_stride)
    if (dtype == LLM_DT_BF16) { if (vec == 8) LAUNCH(8, bf16); else if (vec == 2) LAUNCH(2, bf16); else LAUNCH(1, bf16); }
    else if (dtype == LLM_DT_F32) { if (vec == 8) LAUNCH(8, float); else if (vec == 2) LAUNCH(2, float); else LAUNCH(1, float); }
    else return LLM_REFUSED_DTYPE;
#undef LAUNCH
    return launch_status();
}

// ---- values ---------------------------------------------------------------------------------------------------------
// U rows a thread, asked for together.  Sixteen lanes a tile's row and eight codes a lane; where rows are not whole, aligned pieces of eight values a warp a tile's row, a lane
// pairs of neighbouring codes (or single ones) 64 (32) apart, so that what a warp stores lies side by side.
// 12,288 x 4,096 into bfloat16 29.5 us (151 MB, 5.1 TB/s; sixteen codes a lane 30.7); 1,003 x 1,358 4.8 us (sixteen codes a lane 11.3), 1,003 x 1,357 5.0 us (23.7).
template <int U, int VEC, typename T>
__global__ void __launch_bounds__(F8_THREADS) f8_values_kernel(const unsigned char* codes, const float* scales, T* out, int rows,
                                                               int N, int K, int ktiles, int k4, int tiles, long long padded, int kind) {
    // kind 0: rows, 1: a weight, 2: a gated one (N: its gate rows); tiles: of 128 rows
    constexpr int LANES = VEC == 8 ? 16 : 32, ROWS = F8_THREADS / LANES;
    pdl_begin();
    const int kb = blockIdx.x % ktiles, piece = threadIdx.x % LANES, col = kb * F8_K + piece * VEC;
    const long long first = static_cast<long long>(blockIdx.x / ktiles) * (U * ROWS) + threadIdx.x / LANES;
    uint2 c[U];
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long r = first + u * ROWS;
        c[u] = make_uint2(0u, 0u);
        s[u] = 0.0f;
        if (r >= rows) continue;
        const unsigned char* from;
        if (kind == 0) {
            from = codes + (kb * padded + r) * F8_K;
            s[u] = scales[r * k4 + kb];
        } else {
            const int per = kind == 2 ? 2 * N : N;                // rows of a matrix of the stack
            const long long e = r / per;
            const int at = static_cast<int>(r - e * per), up = kind == 2 && at >= N, i = up ? at - N : at;
            const long long tile = e * tiles + (kind == 2 ? (i >> 6) : (i >> 7));
            const int in = kind == 2 ? up * 64 + (i & 63) : i & 127, which = !up ? 0 : (i & 63) < f8_split(N, i >> 6) ? 1 : 2;
            from = codes + ((tile * ktiles + kb) * 128 + in) * F8_K;
            s[u] = scales[(tile * 3 + which) * k4 + kb];
        }
        if constexpr (VEC == 8) {
            c[u] = *reinterpret_cast<const uint2*>(from + piece * 8);
        } else if constexpr (VEC == 2) {
            const unsigned lo = *reinterpret_cast<const unsigned short*>(from + piece * 2), hi = *reinterpret_cast<const unsigned short*>(from + 64 + piece * 2);
            c[u].x = lo | hi << 16;
        } else {
            unsigned b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = from[32 * i + piece];
            c[u].x = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long r = first + u * ROWS;
        if (r >= rows) continue;
        T* to = out + r * K + col;
        float v[8];
        mx_from_e4m3x4(c[u].x, v);
        if constexpr (VEC == 8) mx_from_e4m3x4(c[u].y, v + 4);
#pragma unroll
        for (int i = 0; i < (VEC == 8 ? 8 : 4); ++i) v[i] *= s[u];
        if constexpr (VEC == 8) {
            if (col < K) store8(to, v);
        } else if constexpr (VEC == 2) {
            if (col < K) mx_store2(to, v[0], v[1]);
            if (col + 64 < K) mx_store2(to + 64, v[2], v[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (col + 32 * i < K) to[32 * i] = from_f32<T>(v[i]);
        }
    }
}

extern "C" int llm_f8_values(const void* codes, const void* scales, void* out, int dtype, int rows, int N, int K, int tiles, long long padded, int kind, uintptr_t stream) {
    if (rows <= 0) return LLM_OK;
    if (K <= 0 || K > (1 << 20) || kind < 0 || kind > 2 || (kind && N <= 0)) return LLM_REFUSED_SIZE;
    constexpr int U = 4;
    const int ktiles = f8_tiles(K), vec = mx_vec(K, out, dtype == LLM_DT_F32 ? 4 : 2), per = U * F8_THREADS / (vec == 8 ? 16 : 32);       // rows a CTA
    const long long blocks = (static_cast<long long>(rows) + per - 1) / per * ktiles;
    if (blocks >= (1LL << 31)) return LLM_REFUSED_SIZE;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
#define LAUNCH(VEC, T_)                                                                                                                              \
    launch_pdl((f8_values_kernel<U, VEC, T_>), dim3(static_cast<unsigned>(blocks)), dim3(F8_THREADS), 0, s, static_cast<const unsigned char*>(codes), \
               static_cast<const float*>(scales), static_cast<T_*>(out), rows, N, K, ktiles, f8_k4(K), tiles, padded, kind)
    if (dtype == LLM_DT_BF16) { if (vec == 8) LAUNCH(8, bf16); else if (vec == 2) LAUNCH(2, bf16); else LAUNCH(1, bf16); }
    else if (dtype == LLM_DT_F32) { if (vec == 8) LAUNCH(8, float); else if (vec == 2) LAUNCH(2, float); else LAUNCH(1, float); }
    else return LLM_REFUSED_DTYPE;
#undef LAUNCH
    return launch_status();
}

// ---- rows sorted by expert ------------------------------------------------------------------------------------------
// A cluster (of one CTA for few picks) counts the picks of each expert, lays the experts' rows one after another, cuts them into items of up to `per` rows, and
// gives every pick its row: places[pick] (-1 where the pick is no expert), weights[row].  A CTA takes neighbouring picks and adds up the counts of those
// before it out of their shared memory: 32,768 picks of 64 experts 52 us by one CTA, 9 to 12 by eight.  Which of an expert's rows a pick gets is not fixed; no result depends on it,
// a row's products being its own.
#define F8_SORT_CTAS 8
#define F8_SORT_PICKS 4           // picks of a thread that stay in registers

__global__ void __launch_bounds__(1024) f8_sort_kernel(const int32_t* ids, const float* weights, int picks, int E, int per,
                                                       int32_t* counts, int4* items, int32_t* places, float* row_weights) {
    extern __shared__ int counted_s[];                            // [E] this CTA's picks, [E] the next row of an expert
    __shared__ int2 warps_s[32];
    int* next_s = counted_s + E;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5, rank = blockIdx.x, ctas = gridDim.x;
    const int mine = (picks + ctas - 1) / ctas, from = rank * mine, to = min(from + mine, picks);
    for (int e = tid; e < E; e += blockDim.x) counted_s[e] = 0;
    pdl_begin();
    __syncthreads();
    int held[F8_SORT_PICKS];
    auto expert = [&](int p) {
        const int e = p < to ? ids[p] : -1;
        return e < E ? e : -1;
    };
    auto count = [&](int e) {                                     // one addition for the lanes with the same expert
        const unsigned same = __match_any_sync(0xffffffffu, e);
        if (e >= 0 && lane == __ffs(same) - 1) atomicAdd(&counted_s[e], __popc(same));
    };
    auto place = [&](int p, int e) {
        const unsigned same = __match_any_sync(0xffffffffu, e);
        const int first = __ffs(same) - 1;
        int r = 0;
        if (e >= 0 && lane == first) r = atomicAdd(&next_s[e], __popc(same));
        r = __shfl_sync(0xffffffffu, r, first) + __popc(same & ((1u << lane) - 1));
        if (p >= to) return;
        if (e >= 0) {
            row_weights[r] = weights[p];
        }
        places[p] = e >= 0 ? r : -1;
    };
#pragma unroll
    for (int i = 0; i < F8_SORT_PICKS; ++i) held[i] = expert(from + i * blockDim.x + tid);
#pragma unroll
    for (int i = 0; i < F8_SORT_PICKS; ++i) count(held[i]);
    for (int p = from + F8_SORT_PICKS * blockDim.x; p < to; p += blockDim.x) count(expert(p + tid));
    if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    else __syncthreads();
    int2 base = make_int2(0, 0);                                  // rows and items of the experts before this round's
    for (int e0 = 0; e0 < E; e0 += blockDim.x) {
        const int e = e0 + tid;
        int n = 0, before = 0;                                    // an expert's picks, and those of the CTAs before this one
        if (e < E) {
            if (ctas == 1) n = counted_s[e];
            else
#pragma unroll
                for (int c = 0; c < F8_SORT_CTAS; ++c) {
                    unsigned at;
                    int k;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(static_cast<unsigned>(__cvta_generic_to_shared(&counted_s[e]))), "r"(c));
                    asm volatile("ld.shared::cluster.s32 %0, [%1];\n" : "=r"(k) : "r"(at) : "memory");
                    n += k;
                    if (c < rank) before += k;
                }
        }
        int2 sum = make_int2(n, (n + per - 1) / per);
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int a = __shfl_up_sync(0xffffffffu, sum.x, o), b = __shfl_up_sync(0xffffffffu, sum.y, o);
            if (lane >= o) sum.x += a, sum.y += b;
        }
        if (lane == 31) warps_s[warp] = sum;
        __syncthreads();
        int2 total = base;
        for (int w = 0; w < warps; ++w) {
            if (w == warp) sum.x += total.x, sum.y += total.y;
            total.x += warps_s[w].x, total.y += warps_s[w].y;
        }
        if (e < E) {
            const int row = sum.x - n;
            int item = sum.y - (n + per - 1) / per;
            next_s[e] = row + before;
            if (rank == 0)
                for (int at = 0; at < n; at += per) items[item++] = make_int4(e, row + at, min(per, n - at), 0);
        }
        base = total;
        __syncthreads();
    }
    if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");        // the others' counts have been read
    if (tid == 0 && rank == 0) counts[0] = base.y, counts[1] = base.x;
#pragma unroll
    for (int i = 0; i < F8_SORT_PICKS; ++i) place(from + i * blockDim.x + tid, held[i]);
    for (int p = from + F8_SORT_PICKS * blockDim.x; p < to; p += blockDim.x) place(p + tid, expert(p + tid));
    if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");          // nobody leaves before
}

extern "C" int llm_f8_sort(const int32_t* ids, const float* weights, int picks, int E, int per, int32_t* counts, void* items, int32_t* places, float* row_weights,
                           uintptr_t stream) {
    if (picks <= 0) return LLM_OK;
    if (E <= 0 || E > F8_MOST_EXPERTS || per <= 0) return LLM_REFUSED_SIZE;
    if (!aligned16(items)) return LLM_REFUSED_ALIGN;
    const int ctas = picks > 2048 ? F8_SORT_CTAS : 1, most = ctas == 1 && picks > E ? picks : E, threads = ctas > 1 || most >= 1024 ? 1024 : (most + 31) / 32 * 32;
    launch_pdl_cluster(f8_sort_kernel, dim3(ctas), dim3(threads), 2 * E * sizeof(int), reinterpret_cast<cudaStream_t>(stream), ctas, ids, weights, picks, E, per, counts,
                       static_cast<int4*>(items), places, row_weights);
    return launch_status();
}

// out[token] = base[token] + the token's rows of y in the order of its choices, in 32 bits; rounded to the result's type once.
// 4,096 tokens of eight rows of 2,048: 45 us (285 MB, 6.3 TB/s), into float32 47.
template <typename TO>
__global__ void __launch_bounds__(128) f8_add_up_kernel(const float* y, const int32_t* places, TO* out, int N, int top, int vec,
                                                        const float* base) {
    pdl_begin();
    const size_t t = blockIdx.x;
    if (vec) {
        const int i = (blockIdx.y * 128 + threadIdx.x) * 8;
        if (i >= N) return;
        float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (base) load8(base + t * N + i, sum);
        for (int k0 = 0; k0 < top; k0 += 8) {                     // eight rows' places, then eight rows, in flight together
            int r[8];
            float v[8][8];
#pragma unroll
            for (int k = 0; k < 8; ++k) r[k] = k0 + k < top ? places[t * top + k0 + k] : -1;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (r[k] >= 0) load8(y + static_cast<size_t>(r[k]) * N + i, v[k]);
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int c = 0; c < 8; ++c) sum[c] += r[k] >= 0 ? v[k][c] : 0.0f;
        }
        store8(out + t * N + i, sum);
    } else {
        for (int i = blockIdx.y * 128 + threadIdx.x; i < N; i += gridDim.y * 128) {
            float sum = base ? base[t * N + i] : 0.0f;
            for (int k = 0; k < top; ++k) {
                const int r = places[t * top + k];
                if (r >= 0) sum += y[static_cast<size_t>(r) * N + i];
            }
            out[t * N + i] = from_f32<TO>(sum);
        }
    }
}

// y [rows, N] in float32, out [T, N] of `dtype`; base (float32 [T, N]) may be null.
extern "C" int llm_f8_add_up(const float* y, const int32_t* places, const float* base, void* out, int dtype, int T, int N, int top, uintptr_t stream) {
    if (T <= 0) return LLM_OK;
    if (N <= 0 || N > (1 << 24) || top <= 0) return LLM_REFUSED_SIZE;
    const int vec = N % 8 == 0 && aligned16(y) && aligned16(out) && aligned16(base);
    const dim3 grid(T, (N + 1023) / 1024);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == LLM_DT_F32)
        launch_pdl((f8_add_up_kernel<float>), grid, dim3(128), 0, s, y, places, static_cast<float*>(out), N, top, vec, base);
    else if (dtype == LLM_DT_BF16)
        launch_pdl((f8_add_up_kernel<bf16>), grid, dim3(128), 0, s, y, places, static_cast<bf16*>(out), N, top, vec, base);
    else
        return LLM_REFUSED_DTYPE;
    return launch_status();
}
