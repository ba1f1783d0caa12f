// What makes microscaled rows and weights (microscaling.cuh has the format), and what reads them back:
//   rows of 8 bits   from a matrix; from rmsnorm(x + delta) * w, the sum kept as the new residual stream; from act(gate) * up
//   weights of 4     from a matrix, gate and up rows of a fused matrix 64 by 64 beside each other
//   values           of either, as float32 or bfloat16
// Everything is bound by memory: each value is read once and each code written once.  A lane holds eight neighbouring values
// (16 or 32 bytes a load), a block's largest magnitude takes two exchanges between lanes, and the codes are the converter's.
#include "microscaling.cuh"

#define MX_THREADS 256

// A warp takes U pieces of 256 neighbouring values of a row, all of them asked for before the first is used: one piece a thread left
// the memory idle (weights of 12,288 x 4,096 43 us with one, XX with four), several leave the SMs idle where there is little to do.
struct MxSpan {
    long long row;
    int col;                              // of the lane's first piece
    bool there;
};
template <int U> __device__ __forceinline__ MxSpan mx_span(unsigned items, unsigned per_row) {
    const unsigned w = blockIdx.x * (MX_THREADS / 32) + (threadIdx.x >> 5), row = w / per_row;
    return {row, static_cast<int>((w - row * per_row) * (U * 256) + (threadIdx.x & 31) * 8), w < items};
}

// ---- rows of 8 bits from a matrix -----------------------------------------------------------------------------------
template <int U, bool FAST, typename T>
__global__ void __launch_bounds__(MX_THREADS) mx_rows_kernel(const T* __restrict__ x, unsigned char* __restrict__ codes,
                                                             unsigned char* __restrict__ scales, unsigned items, unsigned per_row, int K, int kpad, int vec) {
    pdl_begin();
    const MxSpan at = mx_span<U>(items, per_row);
    if (!at.there) return;                                        // whole warps
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) mx_load8<FAST>(x + at.row * K, at.col + u * 256, K, vec, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) mx_store_row8(v[u], at.col + u * 256 < kpad, at.row, at.col + u * 256, kpad, codes, scales);
}

// ---- rows of 8 bits from act(gate) * up, sums and activation in 32 bits --------------------------------------------
template <int U, bool FAST, typename T>
__global__ void __launch_bounds__(MX_THREADS) mx_act_kernel(const T* __restrict__ gu, unsigned char* __restrict__ codes,
                                                            unsigned char* __restrict__ scales, unsigned items, unsigned per_row, int inter, int kpad, int vec,
                                                            int parts, long long part_stride, const MxAct act) {
    pdl_begin();
    const MxSpan at = mx_span<U>(items, per_row);
    if (!at.there) return;
    const T* g = gu + at.row * 2 * inter;
    float a[U][8], b[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        mx_load8<FAST>(g, at.col + u * 256, inter, vec, a[u]);
        mx_load8<FAST>(g + inter, at.col + u * 256, inter, vec, b[u]);
    }
    for (int p = 1; p < parts; ++p) {                             // a product left as its k-splits
        g += part_stride;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float c[8];
            mx_load8<FAST>(g, at.col + u * 256, inter, vec, c);
#pragma unroll
            for (int i = 0; i < 8; ++i) a[u][i] += c[i];
            mx_load8<FAST>(g + inter, at.col + u * 256, inter, vec, c);
#pragma unroll
            for (int i = 0; i < 8; ++i) b[u][i] += c[i];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int col = at.col + u * 256;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[u][i] = col + i < inter ? mx_gated(a[u][i], b[u][i], act) : 0.0f;
        mx_store_row8(a[u], col < kpad, at.row, col, kpad, codes, scales);
    }
}

// ---- rows of 8 bits from rmsnorm(x + delta) * w ---------------------------------------------------------------------
// One block a row (sum_out may be x: a thread writes what it has read); the row stays in registers between the sum of squares and the codes, CH pieces of eight values a thread.
template <typename TX, typename TD, int CH, bool FAST>
__global__ void __launch_bounds__(1024) mx_norm_kernel(const TX* x, const TD* __restrict__ delta, const float* __restrict__ w,
                                                       TX* sum_out, unsigned char* __restrict__ codes,
                                                       unsigned char* __restrict__ scales, const int32_t* __restrict__ rows, int hidden, int kpad,
                                                       float eps, int vec, int parts, long long part_stride) {
    __shared__ float scratch[32];
    if (FAST)                                                     // the weights are the model's: on their way before the wait
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
        mx_load8<FAST>(xr, col, hidden, vec, v[c]);
        if (delta) {
#pragma unroll 4
            for (int p = 0; p < parts; ++p) {                     // the sublayer's product may come as its k-splits
                float d[8];
                mx_load8<FAST>(delta + src * hidden + p * part_stride, col, hidden, vec, d);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] += d[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += v[c][i] * v[c][i];
        if (sum_out) mx_put8<FAST>(sum_out + src * hidden, col, hidden, vec, v[c]);
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
        mx_load8<FAST>(w, col, hidden, vec, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] = v[c][i] * inv * g[i];
        mx_store_row8(v[c], col < kpad, blockIdx.x, col, kpad, codes, scales);
    }
}

// ---- weights of 4 bits ----------------------------------------------------------------------------------------------
// Rows of the tiles.  It does not invite the kernel behind it: products fetch weights before they wait for what is in front of them.
template <int U, bool FAST, typename T>
__global__ void __launch_bounds__(MX_THREADS) mx_weight_kernel(const T* __restrict__ w, unsigned char* __restrict__ tiles,
                                                               unsigned char* __restrict__ scales, unsigned items, unsigned per_row, int N, int K, int ktiles,
                                                               int gated_rows, int vec) {
    pdl_wait();
    const MxSpan at = mx_span<U>(items, per_row);                 // a row of the tiles
    if (!at.there) return;
    const long long row = at.row;
    long long src = row;                                          // of the matrix; gated: [gate; up] of N rows each
    bool real = row < N;
    if (gated_rows) {
        const long long f = (row >> 7) * 64 + (row & 63);
        real = f < N;
        src = (row & 64) ? N + f : f;
    }
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) mx_load8<FAST>(w + src * K, real ? at.col + u * 256 : K, K, vec, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int col = at.col + u * 256;
        unsigned word;
        const uint2 c = mx_encode8<MX_E2M1>(v[u], word);
        if (col < ktiles * MX_K) {
            const long long tile = (row >> 7) * ktiles + (col >> 7);
            *reinterpret_cast<unsigned*>(tiles + (tile * 128 + (row & 127)) * 64 + (col & 127) / 2) = c.x;
            if ((col & (MX_K - 1)) == 0) *reinterpret_cast<unsigned*>(scales + mx_scale_at(row, col / MX_BLOCK, ktiles)) = word;
        }
    }
}

// ---- the values that codes stand for --------------------------------------------------------------------------------
template <int U, bool FAST, int FMT, typename T>
__global__ void __launch_bounds__(MX_THREADS) mx_values_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                               T* __restrict__ out, unsigned items, unsigned per_row, int N, int K, int ktiles, int gated_rows,
                                                               int vec) {
    pdl_begin();
    const MxSpan at = mx_span<U>(items, per_row);                 // a row of the matrix
    if (!at.there) return;
    long long row = at.row;                                       // of the codes
    if (FMT == MX_E2M1 && gated_rows) {
        const long long f = row < N ? row : row - N;
        row = (f >> 6) * 128 + (row < N ? 0 : 64) + (f & 63);
    }
    uint2 c[U];
    unsigned char s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int col = at.col + u * 256;
        c[u] = make_uint2(0u, 0u);
        s[u] = 0;
        if (col < K) {
            if (FMT == MX_E2M1) c[u].x = *reinterpret_cast<const unsigned*>(codes + (((row >> 7) * ktiles + (col >> 7)) * 128 + (row & 127)) * 64 + (col & 127) / 2);
            else c[u] = *reinterpret_cast<const uint2*>(codes + row * static_cast<long long>(ktiles) * MX_K + col);
            s[u] = scales[mx_scale_at(row, col / MX_BLOCK, ktiles)];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float v[8];
        if (FMT == MX_E2M1) mx_from_e2m1x8(c[u].x, v);
        else {
            mx_from_e4m3x4(c[u].x, v);
            mx_from_e4m3x4(c[u].y, v + 4);
        }
        const float f = mx_value(s[u]);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= f;
        mx_put8<FAST>(out + at.row * K, at.col + u * 256, K, vec, v);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
#define MX_MOST_K (1 << 20)
// How `rows` rows of n values are cut into warps' items of `u` pieces: four pieces where that leaves enough warps and wastes little.
struct MxCut {
    int u;
    unsigned items, per_row, blocks;
};
static inline bool mx_cut(long long rows, int n, MxCut* c) {
    const int pieces = (n + 255) / 256;
    c->u = rows * pieces >= 32768 && (pieces % 4 == 0 || pieces >= 12) ? 4 : rows * pieces >= 16384 && (pieces % 2 == 0 || pieces >= 7) ? 2 : 1;
    c->per_row = static_cast<unsigned>((pieces + c->u - 1) / c->u);
    const long long items = rows * c->per_row;
    c->items = static_cast<unsigned>(items);
    c->blocks = static_cast<unsigned>((items + MX_THREADS / 32 - 1) / (MX_THREADS / 32));
    return items <= 0x7fffffffLL;
}
#define MX_GO(KERNEL, ...)                                                                                                              \
    do {                                                                                                                                \
        const bool fast = vec == 8;                                                                                                     \
        auto kern = cut.u == 4 ? (fast ? KERNEL(4, true) : KERNEL(4, false))                                                            \
                    : cut.u == 2 ? (fast ? KERNEL(2, true) : KERNEL(2, false))                                                          \
                                 : (fast ? KERNEL(1, true) : KERNEL(1, false));                                                         \
        launch_pdl(kern, dim3(cut.blocks), dim3(MX_THREADS), 0, s, __VA_ARGS__);                                                        \
    } while (0)

// x: [T, K] -> rows of 8 bits: codes [padded rows][ktiles * 128], then scales.
extern "C" int llm_mx_rows(const void* x, int dtype, void* rows, int T, int K, uintptr_t stream) {
    if (T <= 0) return LLM_OK;
    if (K <= 0 || K > MX_MOST_K) return LLM_REFUSED_SIZE;
    if (!aligned16(rows)) return LLM_REFUSED_ALIGN;
    const int kpad = mx_tiles(K) * MX_K, vec = mx_vec(K, x, dtype == LLM_DT_F32 ? 4 : 2);
    MxCut cut;
    if (!mx_cut(T, kpad, &cut)) return LLM_REFUSED_SIZE;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    unsigned char *c = static_cast<unsigned char*>(rows), *sc = mx_row_scales(rows, T, K);
#define F32(U, V) mx_rows_kernel<U, V, float>
#define B16(U, V) mx_rows_kernel<U, V, bf16>
    if (dtype == LLM_DT_F32) MX_GO(F32, static_cast<const float*>(x), c, sc, cut.items, cut.per_row, K, kpad, vec);
    else if (dtype == LLM_DT_BF16) MX_GO(B16, static_cast<const bf16*>(x), c, sc, cut.items, cut.per_row, K, kpad, vec);
    else return LLM_REFUSED_DTYPE;
#undef F32
#undef B16
    return launch_status();
}

// gu: [parts][T, 2 * inter] = [gate | up], parts `part_stride` values apart (more than one: float32).
extern "C" int llm_mx_silu_and_mul(const void* gu, int dtype, int parts, long long part_stride, void* rows, int T, int inter, int act, float limit,
                                   uintptr_t stream) {
    if (T <= 0) return LLM_OK;
    MxAct form;
    if (inter <= 0 || inter > MX_MOST_K || parts < 1 || !mx_act(act, limit, &form)) return LLM_REFUSED_SIZE;
    if (!aligned16(rows)) return LLM_REFUSED_ALIGN;
    const int kpad = mx_tiles(inter) * MX_K, vec = part_stride % 8 ? 1 : mx_vec(inter, gu, dtype == LLM_DT_F32 ? 4 : 2);
    MxCut cut;
    if (!mx_cut(T, kpad, &cut)) return LLM_REFUSED_SIZE;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    unsigned char *c = static_cast<unsigned char*>(rows), *sc = mx_row_scales(rows, T, inter);
#define F32(U, V) mx_act_kernel<U, V, float>
#define B16(U, V) mx_act_kernel<U, V, bf16>
    if (dtype == LLM_DT_F32) MX_GO(F32, static_cast<const float*>(gu), c, sc, cut.items, cut.per_row, inter, kpad, vec, parts, part_stride, form);
    else if (dtype == LLM_DT_BF16) MX_GO(B16, static_cast<const bf16*>(gu), c, sc, cut.items, cut.per_row, inter, kpad, vec, parts, part_stride, form);
    else return LLM_REFUSED_DTYPE;
#undef F32
#undef B16
    return launch_status();
}

template <typename TX, typename TD>
static int mx_norm_launch(const void* x, const void* delta, const float* w, void* sum_out, void* codes, void* scales, const int32_t* rows, int n,
                          int hidden, float eps, int parts, long long part_stride, cudaStream_t s) {
    const int kpad = mx_tiles(hidden) * MX_K;
    const int vec = part_stride % 8 ? 1 : mx_vec(mx_vec(mx_vec(hidden, x, sizeof(TX)), mx_vec(hidden, delta, sizeof(TD))),
                                                 mx_vec(mx_vec(hidden, w, 4), mx_vec(hidden, sum_out, sizeof(TX))));
    // Few rows: a piece of eight values a thread, as many threads as that takes.  Many: blocks of up to 256 threads with up to four pieces
    // each, so that more rows are on their way in an SM (4,096 x 4,096: XX us, with a piece a thread YY).
    const int pieces = kpad / 8, most = n >= 1024 ? 256 : 1024, ch = pieces <= most ? 1 : pieces <= 2 * most ? 2 : 4;
    if (pieces > 4096) return LLM_REFUSED_SIZE;
    auto kern = vec == 8 ? (ch == 1 ? mx_norm_kernel<TX, TD, 1, true> : ch == 2 ? mx_norm_kernel<TX, TD, 2, true> : mx_norm_kernel<TX, TD, 4, true>)
                         : (ch == 1 ? mx_norm_kernel<TX, TD, 1, false> : ch == 2 ? mx_norm_kernel<TX, TD, 2, false> : mx_norm_kernel<TX, TD, 4, false>);
    launch_pdl(kern, dim3(n), dim3((pieces + ch * 32 - 1) / (ch * 32) * 32), 0, s, static_cast<const TX*>(x), static_cast<const TD*>(delta), w,
               static_cast<TX*>(sum_out), static_cast<unsigned char*>(codes), static_cast<unsigned char*>(scales), rows, hidden, kpad, eps, vec, parts, part_stride);
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
    const int ktiles = mx_tiles(K), vec = mx_vec(K, w, dtype == LLM_DT_F32 ? 4 : 2);
    MxCut cut;
    if (!mx_cut(llm_mx_weight_tiles(N, is_gated) * 128LL, ktiles * MX_K, &cut)) return LLM_REFUSED_SIZE;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    unsigned char *t = static_cast<unsigned char*>(tiles), *sc = static_cast<unsigned char*>(scales);
#define F32(U, V) mx_weight_kernel<U, V, float>
#define B16(U, V) mx_weight_kernel<U, V, bf16>
    if (dtype == LLM_DT_F32) MX_GO(F32, static_cast<const float*>(w), t, sc, cut.items, cut.per_row, N, K, ktiles, is_gated, vec);
    else if (dtype == LLM_DT_BF16) MX_GO(B16, static_cast<const bf16*>(w), t, sc, cut.items, cut.per_row, N, K, ktiles, is_gated, vec);
    else return LLM_REFUSED_DTYPE;
#undef F32
#undef B16
    return launch_status();
}

// format 8: rows of 8 bits [N, K]; 4: a weight of 4 bits, out [N, K] or, gated, [2 N, K].
extern "C" int llm_mx_values(const void* codes, const void* scales, int format, void* out, int dtype, int N, int K, int is_gated, uintptr_t stream) {
    if (N <= 0) return LLM_OK;
    if (K <= 0 || K > MX_MOST_K || (format != MX_E2M1 && format != MX_E4M3) || (is_gated && format != MX_E2M1)) return LLM_REFUSED_SIZE;
    if (!aligned16(codes) || !aligned16(scales)) return LLM_REFUSED_ALIGN;
    const int ktiles = mx_tiles(K), vec = mx_vec(K, out, dtype == LLM_DT_F32 ? 4 : 2);
    MxCut cut;
    if (!mx_cut((is_gated ? 2LL : 1LL) * N, K, &cut)) return LLM_REFUSED_SIZE;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const unsigned char *c = static_cast<const unsigned char*>(codes), *sc = static_cast<const unsigned char*>(scales);
#define W32(U, V) mx_values_kernel<U, V, MX_E2M1, float>
#define W16(U, V) mx_values_kernel<U, V, MX_E2M1, bf16>
#define R32(U, V) mx_values_kernel<U, V, MX_E4M3, float>
#define R16(U, V) mx_values_kernel<U, V, MX_E4M3, bf16>
    if (dtype != LLM_DT_F32 && dtype != LLM_DT_BF16) return LLM_REFUSED_DTYPE;
    float* of = static_cast<float*>(out);
    bf16* ob = static_cast<bf16*>(out);
    if (format == MX_E2M1) {
        if (dtype == LLM_DT_F32) MX_GO(W32, c, sc, of, cut.items, cut.per_row, N, K, ktiles, is_gated, vec);
        else MX_GO(W16, c, sc, ob, cut.items, cut.per_row, N, K, ktiles, is_gated, vec);
    } else {
        if (dtype == LLM_DT_F32) MX_GO(R32, c, sc, of, cut.items, cut.per_row, N, K, ktiles, is_gated, vec);
        else MX_GO(R16, c, sc, ob, cut.items, cut.per_row, N, K, ktiles, is_gated, vec);
    }
#undef W32
#undef W16
#undef R32
#undef R16
    return launch_status();
}
