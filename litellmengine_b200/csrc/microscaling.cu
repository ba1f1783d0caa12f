// What makes microscaled rows and weights (microscaling.cuh has the format), and what reads them back:
//   rows of 8 bits   from a matrix; from rmsnorm(x + delta) * w, the sum kept as the new residual stream; from act(gate) * up
//   weights of 4     from a matrix, gate and up rows of a fused matrix 64 by 64 beside each other
//   values           of either, as float32 or bfloat16
// Everything is bound by memory: each value is read once and each code written once.  A lane holds eight neighbouring values
// (16 or 32 bytes a load), a block's largest magnitude takes two exchanges between lanes, and the codes are the converter's.
#include "microscaling.cuh"

#define MX_THREADS 256

// ---- rows of 8 bits from a matrix: a thread takes eight values ----------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(MX_THREADS) mx_rows_kernel(const T* __restrict__ x, unsigned char* __restrict__ codes,
                                                             unsigned char* __restrict__ scales, long long pieces, int K, int kpad, int vec) {
    pdl_begin();
    const long long at = blockIdx.x * static_cast<long long>(MX_THREADS) + threadIdx.x;
    const bool there = at < pieces;                               // pieces of a row are a multiple of 16: lanes of a block go together
    const int per_row = kpad / 8;
    const long long row = there ? at / per_row : 0;
    const int col = static_cast<int>(there ? at - row * per_row : 0) * 8;
    float v[8];
    mx_load8(x + row * K, col, K, vec, v);
    mx_store_row8(v, there, row, col, kpad, codes, scales);
}

// ---- rows of 8 bits from act(gate) * up, sums and activation in 32 bits --------------------------------------------
template <typename T>
__global__ void __launch_bounds__(MX_THREADS) mx_act_kernel(const T* __restrict__ gu, unsigned char* __restrict__ codes,
                                                            unsigned char* __restrict__ scales, long long pieces, int inter, int kpad, int vec,
                                                            int parts, long long part_stride, const MxAct act) {
    pdl_begin();
    const long long at = blockIdx.x * static_cast<long long>(MX_THREADS) + threadIdx.x;
    const bool there = at < pieces;
    const int per_row = kpad / 8;
    const long long row = there ? at / per_row : 0;
    const int col = static_cast<int>(there ? at - row * per_row : 0) * 8;
    const T* g = gu + row * 2 * inter;
    float a[8], b[8];
    mx_load8(g, col, inter, vec, a);
    mx_load8(g + inter, col, inter, vec, b);
    for (int p = 1; p < parts; ++p) {                             // a product left as its k-splits
        float c[8];
        mx_load8(g + p * part_stride, col, inter, vec, c);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] += c[i];
        mx_load8(g + p * part_stride + inter, col, inter, vec, c);
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] += c[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = col + i < inter ? mx_gated(a[i], b[i], act) : 0.0f;
    mx_store_row8(a, there, row, col, kpad, codes, scales);
}

// ---- rows of 8 bits from rmsnorm(x + delta) * w ---------------------------------------------------------------------
// One block a row (sum_out may be x: a thread writes what it has read); the row stays in registers between the sum of squares and the codes, CH pieces of eight values a thread.
template <typename TX, typename TD, int CH>
__global__ void __launch_bounds__(1024) mx_norm_kernel(const TX* x, const TD* __restrict__ delta, const float* __restrict__ w,
                                                       TX* sum_out, unsigned char* __restrict__ codes,
                                                       unsigned char* __restrict__ scales, const int32_t* __restrict__ rows, int hidden, int kpad,
                                                       float eps, int vec, int parts, long long part_stride) {
    __shared__ float scratch[32];
    if (vec)                                                      // the weights are the model's: on their way before the wait
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * blockDim.x + threadIdx.x) * 8;
            if (col < hidden) asm volatile("prefetch.global.L1 [%0];\n" ::"l"(w + col));
        }
    pdl_begin();
    const size_t src = rows ? static_cast<size_t>(rows[blockIdx.x]) : blockIdx.x;
    const TX* xr = x + src * hidden;
    float v[CH][8], ss = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * blockDim.x + threadIdx.x) * 8;
        mx_load8(xr, col, hidden, vec, v[c]);
        if (delta) {
#pragma unroll 4
            for (int p = 0; p < parts; ++p) {                     // the sublayer's product may come as its k-splits
                float d[8];
                mx_load8(delta + src * hidden + p * part_stride, col, hidden, vec, d);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] += d[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += v[c][i] * v[c][i];
        if (sum_out) mx_put8(sum_out + src * hidden, col, hidden, vec, v[c]);
    }
    ss = warp_sum(ss);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = ss;
    __syncthreads();
    ss = warp_sum((threadIdx.x & 31) < ((blockDim.x + 31) >> 5) ? scratch[threadIdx.x & 31] : 0.0f);
    const float inv = 1.0f / sqrtf(ss / static_cast<float>(hidden) + eps);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * blockDim.x + threadIdx.x) * 8;
        float g[8];
        mx_load8(w, col, hidden, vec, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] = v[c][i] * inv * g[i];
        mx_store_row8(v[c], col < kpad, blockIdx.x, col, kpad, codes, scales);
    }
}

// ---- weights of 4 bits ----------------------------------------------------------------------------------------------
// A thread takes eight values of a row of the tiles.  It does not invite the kernel behind it: products fetch weights before they
// wait for what is in front of them.
template <typename T>
__global__ void __launch_bounds__(MX_THREADS) mx_weight_kernel(const T* __restrict__ w, unsigned char* __restrict__ tiles,
                                                               unsigned char* __restrict__ scales, long long pieces, int N, int K, int ktiles,
                                                               int gated_rows, int vec) {
    pdl_wait();
    const long long at = blockIdx.x * static_cast<long long>(MX_THREADS) + threadIdx.x;
    const bool there = at < pieces;
    const int per_row = ktiles * (MX_K / 8);
    const long long row = there ? at / per_row : 0;               // of the tiles
    const int col = static_cast<int>(there ? at - row * per_row : 0) * 8;
    long long src = row;                                          // of the matrix; gated: [gate; up] of N rows each
    bool real = row < N;
    if (gated_rows) {
        const long long f = (row >> 7) * 64 + (row & 63);
        real = f < N;
        src = (row & 64) ? N + f : f;
    }
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (real) mx_load8(w + src * K, col, K, vec, v);
    unsigned word;
    const uint2 c = mx_encode8<MX_E2M1>(v, word);
    if (!there) return;
    const long long tile = (row >> 7) * ktiles + (col >> 7);
    *reinterpret_cast<unsigned*>(tiles + (tile * 128 + (row & 127)) * 64 + (col & 127) / 2) = c.x;
    if ((col & (MX_K - 1)) == 0) *reinterpret_cast<unsigned*>(scales + mx_scale_at(row, col / MX_BLOCK, ktiles)) = word;
}

// ---- the values that codes stand for --------------------------------------------------------------------------------
template <int FMT, typename T>
__global__ void __launch_bounds__(MX_THREADS) mx_values_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                               T* __restrict__ out, long long pieces, int N, int K, int ktiles, int gated_rows,
                                                               int vec) {
    pdl_begin();
    const long long at = blockIdx.x * static_cast<long long>(MX_THREADS) + threadIdx.x;
    if (at >= pieces) return;
    const int per_row = (K + 7) / 8;
    const long long dst = at / per_row;                           // row of the matrix
    const int col = static_cast<int>(at - dst * per_row) * 8;
    float v[8];
    long long row = dst;                                          // row of the codes
    if (FMT == MX_E2M1) {
        if (gated_rows) {
            const long long f = dst < N ? dst : dst - N;
            row = (f >> 6) * 128 + (dst < N ? 0 : 64) + (f & 63);
        }
        const long long tile = (row >> 7) * ktiles + (col >> 7);
        mx_from_e2m1x8(*reinterpret_cast<const unsigned*>(codes + (tile * 128 + (row & 127)) * 64 + (col & 127) / 2), v);
    } else {
        const uint2 c = *reinterpret_cast<const uint2*>(codes + row * static_cast<long long>(ktiles) * MX_K + col);
        mx_from_e4m3x4(c.x, v);
        mx_from_e4m3x4(c.y, v + 4);
    }
    const float s = mx_value(scales[mx_scale_at(row, col / MX_BLOCK, ktiles)]);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= s;
    mx_put8(out + dst * K, col, K, vec, v);
}

// ---- host side ------------------------------------------------------------------------------------------------------
#define MX_MOST_K (1 << 20)
static inline bool mx_grid(long long pieces, unsigned* blocks) {
    const long long b = (pieces + MX_THREADS - 1) / MX_THREADS;
    *blocks = static_cast<unsigned>(b);
    return b > 0 && b <= 0x7fffffffLL;
}

// x: [T, K] -> rows of 8 bits: codes [padded rows][ktiles * 128], then scales.
extern "C" int llm_mx_rows(const void* x, int dtype, void* rows, int T, int K, uintptr_t stream) {
    if (T <= 0) return LLM_OK;
    if (K <= 0 || K > MX_MOST_K) return LLM_REFUSED_SIZE;
    if (!aligned16(rows)) return LLM_REFUSED_ALIGN;
    const int kpad = mx_tiles(K) * MX_K, vec = K % 8 == 0 && aligned16(x);
    const long long pieces = static_cast<long long>(T) * (kpad / 8);
    unsigned blocks;
    if (!mx_grid(pieces, &blocks)) return LLM_REFUSED_SIZE;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    unsigned char *c = static_cast<unsigned char*>(rows), *sc = mx_row_scales(rows, T, K);
    if (dtype == LLM_DT_F32) launch_pdl(mx_rows_kernel<float>, dim3(blocks), dim3(MX_THREADS), 0, s, static_cast<const float*>(x), c, sc, pieces, K, kpad, vec);
    else if (dtype == LLM_DT_BF16) launch_pdl(mx_rows_kernel<bf16>, dim3(blocks), dim3(MX_THREADS), 0, s, static_cast<const bf16*>(x), c, sc, pieces, K, kpad, vec);
    else return LLM_REFUSED_DTYPE;
    return launch_status();
}

// gu: [parts][T, 2 * inter] = [gate | up], parts `part_stride` values apart (more than one: float32).
extern "C" int llm_mx_silu_and_mul(const void* gu, int dtype, int parts, long long part_stride, void* rows, int T, int inter, int act, float limit,
                                   uintptr_t stream) {
    if (T <= 0) return LLM_OK;
    MxAct form;
    if (inter <= 0 || inter > MX_MOST_K || parts < 1 || !mx_act(act, limit, &form)) return LLM_REFUSED_SIZE;
    if (!aligned16(rows)) return LLM_REFUSED_ALIGN;
    const int kpad = mx_tiles(inter) * MX_K, vec = inter % 8 == 0 && part_stride % 8 == 0 && aligned16(gu);
    const long long pieces = static_cast<long long>(T) * (kpad / 8);
    unsigned blocks;
    if (!mx_grid(pieces, &blocks)) return LLM_REFUSED_SIZE;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    unsigned char *c = static_cast<unsigned char*>(rows), *sc = mx_row_scales(rows, T, inter);
    if (dtype == LLM_DT_F32)
        launch_pdl(mx_act_kernel<float>, dim3(blocks), dim3(MX_THREADS), 0, s, static_cast<const float*>(gu), c, sc, pieces, inter, kpad, vec, parts, part_stride, form);
    else if (dtype == LLM_DT_BF16)
        launch_pdl(mx_act_kernel<bf16>, dim3(blocks), dim3(MX_THREADS), 0, s, static_cast<const bf16*>(gu), c, sc, pieces, inter, kpad, vec, parts, part_stride, form);
    else return LLM_REFUSED_DTYPE;
    return launch_status();
}

template <typename TX, typename TD>
static int mx_norm_launch(const void* x, const void* delta, const float* w, void* sum_out, void* codes, void* scales, const int32_t* rows, int n,
                          int hidden, float eps, int parts, long long part_stride, cudaStream_t s) {
    const int kpad = mx_tiles(hidden) * MX_K;
    const int vec = hidden % 8 == 0 && part_stride % 8 == 0 && aligned16(x) && aligned16(w) && aligned16(delta) && aligned16(sum_out);
#define GO(CH)                                                                                                                            \
    launch_pdl(mx_norm_kernel<TX, TD, CH>, dim3(n), dim3((kpad / 8 + CH * 32 - 1) / (CH * 32) * 32), 0, s, static_cast<const TX*>(x),      \
               static_cast<const TD*>(delta), w, static_cast<TX*>(sum_out), static_cast<unsigned char*>(codes),                           \
               static_cast<unsigned char*>(scales), rows, hidden, kpad, eps, vec, parts, part_stride)
    if (kpad <= 8192) GO(1);
    else if (kpad <= 16384) GO(2);
    else if (kpad <= 32768) GO(4);
    else return LLM_REFUSED_SIZE;
#undef GO
    return launch_status();
}

// x: [*, hidden]; delta: [parts][*, hidden] or null; w: float32 [hidden]; sum_out: like x (may be x) or null; rows: int32 [n] or null.
extern "C" int llm_mx_rmsnorm(const void* x, int x_dtype, const void* delta, int delta_dtype, int parts, long long part_stride, const float* w,
                              float eps, void* sum_out, void* made, const int32_t* rows, int n, int hidden, uintptr_t stream) {
    if (n <= 0) return LLM_OK;
    if (hidden <= 0 || parts < 1 || (sum_out && rows)) return LLM_REFUSED_SIZE;
    if (!aligned16(made)) return LLM_REFUSED_ALIGN;
    void *codes = made, *scales = mx_row_scales(made, n, hidden);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (!delta) delta_dtype = LLM_DT_F32;
#define CASE(k, TX, TD) \
    if (x_dtype * 2 + delta_dtype == k) return mx_norm_launch<TX, TD>(x, delta, w, sum_out, codes, scales, rows, n, hidden, eps, parts, part_stride, s);
    CASE(0, float, float)
    CASE(1, float, bf16)
    CASE(2, bf16, float)
    CASE(3, bf16, bf16)
#undef CASE
    return LLM_REFUSED_DTYPE;
}

// Tiles of 128 rows that a weight of N rows (gated: of N gate and N up rows) has: an even number, because products of many rows take two
// at a time, and because a gated product's result is then whole tiles of 128 values.
extern "C" int llm_mx_weight_tiles(int N, int is_gated) { return is_gated ? 2 * ((N + 127) / 128) : (N + 255) / 256 * 2; }

// w: [N, K], gated: [2 N, K] = [gate; up].
extern "C" int llm_mx_weight(const void* w, int dtype, void* tiles, void* scales, int N, int K, int is_gated, uintptr_t stream) {
    if (N <= 0 || K <= 0 || K > MX_MOST_K || N > (1 << 24)) return LLM_REFUSED_SIZE;
    if (!aligned16(tiles) || !aligned16(scales)) return LLM_REFUSED_ALIGN;
    const int ktiles = mx_tiles(K), vec = K % 8 == 0 && aligned16(w);
    const long long pieces = llm_mx_weight_tiles(N, is_gated) * 128LL * ktiles * (MX_K / 8);
    unsigned blocks;
    if (!mx_grid(pieces, &blocks)) return LLM_REFUSED_SIZE;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    unsigned char *t = static_cast<unsigned char*>(tiles), *sc = static_cast<unsigned char*>(scales);
    if (dtype == LLM_DT_F32) launch_pdl(mx_weight_kernel<float>, dim3(blocks), dim3(MX_THREADS), 0, s, static_cast<const float*>(w), t, sc, pieces, N, K, ktiles, is_gated, vec);
    else if (dtype == LLM_DT_BF16) launch_pdl(mx_weight_kernel<bf16>, dim3(blocks), dim3(MX_THREADS), 0, s, static_cast<const bf16*>(w), t, sc, pieces, N, K, ktiles, is_gated, vec);
    else return LLM_REFUSED_DTYPE;
    return launch_status();
}

// format 8: rows of 8 bits [N, K]; 4: a weight of 4 bits, out [N, K] or, gated, [2 N, K].
extern "C" int llm_mx_values(const void* codes, const void* scales, int format, void* out, int dtype, int N, int K, int is_gated, uintptr_t stream) {
    if (N <= 0) return LLM_OK;
    if (K <= 0 || K > MX_MOST_K || (format != MX_E2M1 && format != MX_E4M3) || (is_gated && format != MX_E2M1)) return LLM_REFUSED_SIZE;
    if (!aligned16(codes) || !aligned16(scales)) return LLM_REFUSED_ALIGN;
    const int ktiles = mx_tiles(K), vec = K % 8 == 0 && aligned16(out);
    const long long pieces = (is_gated ? 2LL : 1LL) * N * ((K + 7) / 8);
    unsigned blocks;
    if (!mx_grid(pieces, &blocks)) return LLM_REFUSED_SIZE;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const unsigned char *c = static_cast<const unsigned char*>(codes), *sc = static_cast<const unsigned char*>(scales);
#define GO(FMT, T) launch_pdl(mx_values_kernel<FMT, T>, dim3(blocks), dim3(MX_THREADS), 0, s, c, sc, static_cast<T*>(out), pieces, N, K, ktiles, is_gated, vec)
    if (dtype != LLM_DT_F32 && dtype != LLM_DT_BF16) return LLM_REFUSED_DTYPE;
    if (format == MX_E2M1) {
        if (dtype == LLM_DT_F32) GO(MX_E2M1, float);
        else GO(MX_E2M1, bf16);
    } else {
        if (dtype == LLM_DT_F32) GO(MX_E4M3, float);
        else GO(MX_E4M3, bf16);
    }
#undef GO
    return launch_status();
}
