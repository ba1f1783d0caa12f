// What makes microscaled rows and weights (microscaling.cuh has the format), and what reads them back:
//   rows of 8 bits   from a matrix; from rmsnorm(x + delta) * w, the sum kept as the new residual stream; from act(gate) * up
//   weights of 4     from a matrix, gate and up rows of a fused matrix 64 by 64 beside each other
//   values           of either, as float32 or bfloat16
// Everything is bound by memory: each value is read once and each code written once.  A lane holds eight neighbouring values
// (16 or 32 bytes a load) and a block's largest magnitude takes two exchanges between lanes; of a bfloat16 matrix of whole, aligned pieces sixteen (two
// loads) and one exchange.  The codes are the converter's.
#include "microscaling.cuh"
#include <type_traits>

#define MX_THREADS 256

// A warp takes U pieces of 256 (or 512) neighbouring values of a row, all of them asked for before the first is used: one piece a thread left
// the memory idle (the values of a weight of 12,288 x 4,096 37 us with one, 24 with four), several leave the SMs idle where there is little to do.
struct MxSpan {
    long long row;
    int col;                              // of the lane's first piece
    bool there;
};
template <int U, int LANE = 8> __device__ __forceinline__ MxSpan mx_span(unsigned items, unsigned per_row) {
    const unsigned w = blockIdx.x * (MX_THREADS / 32) + (threadIdx.x >> 5), row = w / per_row;
    return {row, static_cast<int>((w - row * per_row) * (U * 32 * LANE) + (threadIdx.x & 31) * LANE), w < items};
}

// ---- rows of 8 bits from a matrix -----------------------------------------------------------------------------------
template <int U, bool FAST, typename T>
__global__ void __launch_bounds__(MX_THREADS) mx_rows_kernel(const T* __restrict__ x, unsigned char* __restrict__ codes,
                                                             unsigned char* __restrict__ scales, unsigned items, unsigned per_row, int K, int kpad, int vec) {
    constexpr bool WIDE = FAST && sizeof(T) == 2;
    pdl_begin();
    const MxSpan at = mx_span<U, WIDE ? 16 : 8>(items, per_row);
    if (!at.there) return;                                        // whole warps
    if constexpr (WIDE) {
        uint4 raw[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int col = at.col + u * 512 + h * 8;
                raw[u][h] = make_uint4(0u, 0u, 0u, 0u);
                if (col < K) mx_raw8(x + at.row * K + col, raw[u][h]);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int col = at.col + u * 512;
            unsigned word;
            const uint4 c = mx_encode16<MX_E4M3>(raw[u][0], raw[u][1], word);
            if (col < kpad) {
                *reinterpret_cast<uint4*>(codes + at.row * kpad + col) = c;
                if ((col & (MX_K - 1)) == 0) *reinterpret_cast<unsigned*>(scales + mx_scale_at(at.row, col / MX_BLOCK, kpad / MX_K)) = word;
            }
        }
    } else {
        float v[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) mx_load8<FAST>(x + at.row * K, at.col + u * 256, K, vec, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) mx_store_row8(v[u], mx_most8(v[u]), at.col + u * 256 < kpad, at.row, at.col + u * 256, kpad, codes, scales);
    }
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
        mx_store_row8(a[u], mx_most8(a[u]), col < kpad, at.row, col, kpad, codes, scales);
    }
}

// ---- rows of 8 bits from rmsnorm(x + delta) * w ---------------------------------------------------------------------
// One block a row (sum_out may be x: a thread writes what it has read); the row stays in registers between the sum of squares and the
// codes, CH pieces of eight values a thread.
// A value that is a hair off falls to the other side of a border between two codes and comes out a whole step off, an eighth of it.  So
// everything up to the codes carries what float32 leaves out, where memory bounds the kernel anyway: sums with their remainders, the
// threads' squares added in 64 bits, the factor in two parts, products with their remainders, and a result rounded to odd (its last
// bit says that something is beyond it), which makes the rounding to 8 bits the only one.
__device__ __forceinline__ void mx_two_sum(float a, float b, float& sum, float& rest) {
    sum = a + b;
    const float c = sum - a;
    rest += (a - (sum - c)) + (b - c);
}
// v * (ih + il) * g, v with its remainder, rounded to odd: towards zero, and a one as last bit where that is not the whole of it.
__device__ __forceinline__ float mx_scaled_odd(float v, float rest, float ih, float il, float g) {
    const float p = v * ih, pe = fmaf(v, ih, -p) + fmaf(rest, ih, v * il), q = p * g, qe = fmaf(pe, g, fmaf(p, g, -q));
    const float hi = q + qe, lo = qe - (hi - q);
    const int bits = __float_as_int(hi), odd = (bits + ((__float_as_int(lo) ^ bits) >> 31)) | 1;
    return fabsf(lo) > 0.0f ? __int_as_float(odd) : hi;           // a NaN passes as it is
}
// Only values next to a border need that.  The plain product v * ih * g is off by less than 8 of its last places: v by a half (one sum's remainder),
// ih by 2 and a half (rsqrtf's bound and the mean's rounding), each product by a half, and a place is up to twice as much of one number as of another.  So
// where no value of a warp is within 16 places of a border between two codes, nor a block's largest of one between two scales, nor anything in the
// format's lowest range, the codes of the plain products are those of the carried ones, which few pieces then take: the same codes for
// 4,096 x 4,096 with a sum pending in 41 us instead of 44, for one row in 2.6 instead of 3.2.
#define MX_NEAR 16u
__device__ __forceinline__ bool mx_doubtful(const float (&t)[8], unsigned most, unsigned scale) {
    unsigned border = ~0u, least = ~0u;                           // places from 16 below a border on, in the upper 20 bits; magnitudes without sign, zeros last
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned b = __float_as_uint(t[i]);
        border = min(border, b * 4096u - ((0x80000u - MX_NEAR) << 12));
        least = min(least, b * 2u - 1u);
    }
    return border <= (2u * MX_NEAR << 12) || least < 0x3c800000u * 2u - 1u || scale < 32u || (most & 0x7fffffu) - (0x600000u - MX_NEAR) <= 2u * MX_NEAR;
}
// The codes of a row whose values the block's threads hold; rests(c, r) gives the remainders of piece c.  scratch: a double a warp, for this row
// only.  whole: the remainders may be anything (of several sums).
template <int CH, bool FAST, typename F>
__device__ __forceinline__ void mx_norm_row(const float (&v)[CH][8], F rests, const float* w, double* scratch, unsigned char* codes,
                                            unsigned char* scales, size_t row, int hidden, int kpad, float eps, double per_value, int vec, bool whole) {
    float mine = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) mine = fmaf(v[c][i], v[c][i], mine);
    mine = warp_sum(mine);                                        // many partial sums: their roundings average out; what few warps leave is added in 64 bits
    const int lane = threadIdx.x & 31, warps = (blockDim.x + 31) >> 5;
    if (lane == 0) scratch[threadIdx.x >> 5] = mine;
    __syncthreads();
    double ss = lane < warps ? scratch[lane] : 0.0;
    for (int o = 1; o < warps; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    ss = __shfl_sync(0xffffffffu, ss, 0);
    const double mean = fma(ss, per_value, static_cast<double>(eps));
    // 1 / sqrt(mean) in two parts: a first value, and one step of Newton's with its residue taken in full
    const float mh = static_cast<float>(mean), ml = static_cast<float>(mean - static_cast<double>(mh)), ih = rsqrtf(mh);
    const float sq = ih * ih, left = fmaf(-mh, sq, 1.0f) - fmaf(mh, fmaf(ih, ih, -sq), ml * sq), il = 0.5f * ih * left;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * blockDim.x + threadIdx.x) * 8;
        float g[8], t[8];
        mx_load8<FAST>(w, col, hidden, vec, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = v[c][i] * ih * g[i];
        unsigned most = mx_block_most(mx_most8(t)), scale = mx_scale<MX_E4M3>(most);
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] *= mx_inverse(scale);
        if (__any_sync(0xffffffffu, whole || mx_doubtful(t, most, scale))) {
            float r[8];
            rests(c, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = mx_scaled_odd(v[c][i], r[i], ih, il, g[i]);
            scale = mx_scale<MX_E4M3>(mx_block_most(mx_most8(t)));
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] *= mx_inverse(scale);
        }
        mx_store_codes8(make_uint2(mx_e4m3x4(t[0], t[1], t[2], t[3]), mx_e4m3x4(t[4], t[5], t[6], t[7])), mx_word(scale), col < kpad, row, col, kpad, codes, scales);
    }
}
// Blocks of up to 1,024 threads leave 64 registers a thread: one piece (widths of up to 8,192) fits, of two 12 to 56 bytes are spilled (up to 16,384),
// of four 368 to 912 (up to 32,768), beside the 64 KB and more that a row then moves.
template <typename TX, typename TD, int CH, bool FAST>
__global__ void __launch_bounds__(1024) mx_norm_kernel(const TX* x, const TD* __restrict__ delta, const float* __restrict__ w,
                                                       TX* sum_out, unsigned char* __restrict__ codes,
                                                       unsigned char* __restrict__ scales, const int32_t* __restrict__ rows, int hidden, int kpad,
                                                       float eps, double per_value, int vec, int parts, long long part_stride) {
    __shared__ double scratch[32];
#pragma unroll
    for (int c = 0; c < CH; ++c) {                                // the weights are the model's: on their way before the wait
        const int col = (c * blockDim.x + threadIdx.x) * 8;
        if (col < hidden) asm volatile("prefetch.global.L1 [%0];\n" ::"l"(w + col));
    }
    pdl_begin();
    const size_t src = rows ? static_cast<size_t>(rows[blockIdx.x]) : blockIdx.x;
    const TX* xr = x + src * hidden;
    float v[CH][8], rest[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        mx_load8<FAST>(xr, (c * blockDim.x + threadIdx.x) * 8, hidden, vec, v[c]);
#pragma unroll
        for (int i = 0; i < 8; ++i) rest[c][i] = 0.0f;
    }
    if (delta)
#pragma unroll 1
        for (int p = 0; p < parts; ++p) {                         // the sublayer's product may come as its k-splits
            float d[CH][8];
#pragma unroll
            for (int c = 0; c < CH; ++c) mx_load8<FAST>(delta + src * hidden + p * part_stride, (c * blockDim.x + threadIdx.x) * 8, hidden, vec, d[c]);
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) mx_two_sum(v[c][i], d[c][i], v[c][i], rest[c][i]);
        }
    if (sum_out)
#pragma unroll
        for (int c = 0; c < CH; ++c) mx_put8<FAST>(sum_out + src * hidden, (c * blockDim.x + threadIdx.x) * 8, hidden, vec, v[c]);
    auto rests = [&](int c, float (&r)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = rest[c][i];
    };
    mx_norm_row<CH, FAST>(v, rests, w, scratch, codes, scales, blockIdx.x, hidden, kpad, eps, per_value, vec, parts > 1);
}

// The same for many rows of whole, aligned pieces: a block takes every gridDim-th row, and the next one's values are on their way, each warp's own
// in shared memory (nobody waits for another warp's), while it works on this one.
template <typename TX, typename TD, int CH>
__global__ void __launch_bounds__(256, CH == 4 ? 2 : 4) mx_norm_rows_kernel(const TX* x, const TD* __restrict__ delta, const float* __restrict__ w, TX* sum_out,
                                                           unsigned char* __restrict__ codes, unsigned char* __restrict__ scales, int n, int hidden,
                                                           int kpad, float eps, double per_value) {
    constexpr int XB = 256 * sizeof(TX), DB = 256 * sizeof(TD);   // bytes of a warp's 256 values and of what joins them
    __shared__ double scratch[2][32];
    extern __shared__ __align__(16) unsigned char next_s[];       // [2][CH][warps][XB + DB]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto at = [&](int buf, int c) { return next_s + ((buf * CH + c) * (blockDim.x >> 5) + warp) * (XB + DB); };
    auto copy = [&](unsigned char* to, const void* from) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(static_cast<unsigned>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
    };
    auto fetch = [&](int r, int buf) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = c * blockDim.x * 8 + warp * 256;
            if (r < n) {
#pragma unroll
                for (int b = 0; b < XB; b += 512)
                    if (col + static_cast<int>((b + lane * 16) / sizeof(TX)) < hidden)
                        copy(at(buf, c) + b + lane * 16, reinterpret_cast<const char*>(x + static_cast<size_t>(r) * hidden + col) + b + lane * 16);
                if (delta)
#pragma unroll
                    for (int b = 0; b < DB; b += 512)
                        if (col + static_cast<int>((b + lane * 16) / sizeof(TD)) < hidden)
                            copy(at(buf, c) + XB + b + lane * 16, reinterpret_cast<const char*>(delta + static_cast<size_t>(r) * hidden + col) + b + lane * 16);
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    pdl_begin();
    fetch(blockIdx.x, 0);
    int buf = 0;
#pragma unroll 1
    for (int r = blockIdx.x; r < n; r += gridDim.x, buf ^= 1) {
        __syncwarp();                                             // the block's own reads of two rows ago
        fetch(r + gridDim.x, buf ^ 1);
        asm volatile("cp.async.wait_group 1;\n" ::: "memory");
        __syncwarp();
        float v[CH][8];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * blockDim.x + threadIdx.x) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = 0.0f;
            if (col < hidden) {
                load8(reinterpret_cast<const TX*>(at(buf, c)) + lane * 8, v[c]);
                if (delta) {
                    float d[8];
                    load8(reinterpret_cast<const TD*>(at(buf, c) + XB) + lane * 8, d);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[c][i] += d[i];
                }
                if (sum_out) store8(sum_out + static_cast<size_t>(r) * hidden + col, v[c]);
            }
        }
        auto rests = [&](int c, float (&r)[8]) {                  // from what is still in shared memory
#pragma unroll
            for (int i = 0; i < 8; ++i) r[i] = 0.0f;
            if (delta && static_cast<int>(c * blockDim.x + threadIdx.x) * 8 < hidden) {
                float x8[8], d[8];
                load8(reinterpret_cast<const TX*>(at(buf, c)) + lane * 8, x8);
                load8(reinterpret_cast<const TD*>(at(buf, c) + XB) + lane * 8, d);
#pragma unroll
                for (int i = 0; i < 8; ++i) mx_two_sum(x8[i], d[i], x8[i], r[i]);
            }
        };
        mx_norm_row<CH, true>(v, rests, w, scratch[buf], codes, scales, r, hidden, kpad, eps, per_value, 8, false);
    }
}

// ---- weights of 4 bits ----------------------------------------------------------------------------------------------
// Rows of the tiles, U neighbouring ones a warp and 256 values of each: what a warp writes of a tile lies side by side (U times 64 bytes).  It
// does not invite the kernel behind it: products fetch weights before they wait for what is in front of them.
template <int U, bool FAST, typename T>
__global__ void __launch_bounds__(MX_THREADS) mx_weight_kernel(const T* __restrict__ w, unsigned char* __restrict__ tiles,
                                                               unsigned char* __restrict__ scales, unsigned items, unsigned per_row, int N, int K, int ktiles,
                                                               int gated_rows, int vec) {
    constexpr int LANE = FAST && sizeof(T) == 2 ? 16 : 8;
    pdl_wait();
    const unsigned item = blockIdx.x * (MX_THREADS / 32) + (threadIdx.x >> 5), group = item / per_row;
    const bool mine = item < items;                               // whole warps
    const int col = (item - group * per_row) * (32 * LANE) + (threadIdx.x & 31) * LANE;
    const unsigned row = group * U;                               // of the tiles; gated: 64 rows of gate, 64 of up from [gate; up] of N rows each
    const long long first = gated_rows ? (row >> 7) * 64LL + (row & 63) : row, there = mine ? N - first : 0;
    const T* from = w + (gated_rows && (row & 64) ? N + first : first) * K + col;
    const bool whole = mine && col < ktiles * MX_K;
    unsigned char* to = tiles + ((static_cast<long long>(row >> 7) * ktiles + (col >> 7)) * 128 + (row & 127)) * 64 + (col & 127) / 2;
    unsigned char* to_scales = scales + mx_scale_at(row, col / MX_BLOCK, ktiles);
    auto store = [&](int u, const float (&v)[8], unsigned most) {
        unsigned word;
        const uint2 c = mx_encode8<MX_E2M1>(v, most, word);
        if (whole) {
            *reinterpret_cast<unsigned*>(to + u * 64) = c.x;
            if ((threadIdx.x & 15) == 0) *reinterpret_cast<unsigned*>(to_scales + u * 16) = word;
        }
    };
    if constexpr (LANE == 16) {
        uint4 raw[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                raw[u][h] = make_uint4(0u, 0u, 0u, 0u);
                if (u < there && col + h * 8 < K) mx_raw8(from + static_cast<size_t>(u) * K + h * 8, raw[u][h]);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            unsigned word;
            const uint4 c = mx_encode16<MX_E2M1>(raw[u][0], raw[u][1], word);
            if (whole) {
                *reinterpret_cast<uint2*>(to + u * 64) = make_uint2(c.x, c.y);
                if ((threadIdx.x & 7) == 0) *reinterpret_cast<unsigned*>(to_scales + u * 16) = word;
            }
        }
    } else {
        float v[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) mx_load8<FAST>(from + (u < there ? static_cast<size_t>(u) * K : 0) - col, u < there ? col : K, K, vec, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) store(u, v[u], mx_most8(v[u]));
    }
    __syncthreads();
    if (threadIdx.x == 0) __threadfence();                        // all of the block's codes are there for a product that reads them before its wait
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
// Rows from which blocks fetch ahead.  Few / many rows' kernel, us, float32 sum pending: 1,000 x 4,096 16.1 / 14.3, 700 12.1 / 11.4, 592 9.7 / 10.3;
// 1,000 x 8,192 33.0 / 28.1; 1,200 x 1,024 5.9 / 5.0, 700 4.6 / 4.5, 512 3.9 / 4.1.
#define MX_NORM_ROWS 640
// How `rows` rows of n values are cut into warps' items of `u` pieces of `width`: several pieces where that leaves enough warps and wastes little; with 512
// two at most (4,096 x 4,096: one and two 9.1 us, four 9.8; 700 x 4,096: 2.9, 3.6, 4.1).
struct MxCut {
    int u;
    unsigned items, per_row, blocks;
};
static inline bool mx_cut(long long rows, int n, MxCut* c, int width = 256) {
    const int pieces = (n + width - 1) / width;
    const bool many = rows * pieces >= 32768, two = pieces % 2 == 0 || pieces >= 7;
    if (width == 512) c->u = many && two ? 2 : 1;
    else c->u = many && (pieces % 4 == 0 || pieces >= 12) ? 4 : rows * pieces >= 16384 && two ? 2 : 1;
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
    if (!mx_cut(T, kpad, &cut, vec == 8 && dtype == LLM_DT_BF16 ? 512 : 256)) return LLM_REFUSED_SIZE;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    unsigned char *c = static_cast<unsigned char*>(rows), *sc = mx_row_scales(rows, T, K);
#define F32(U, V) mx_rows_kernel<U, V, float>
#define B16(U, V) mx_rows_kernel<(V && U == 4 ? 2 : U), V, bf16>         // of 512 values two pieces at most
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
    // Many rows: blocks that fetch ahead.  Few: a piece of eight values a thread, as many threads as that takes.
    const int pieces = kpad / 8;
    if (pieces > 4096) return LLM_REFUSED_SIZE;
    if (n >= MX_NORM_ROWS && vec == 8 && parts == 1 && !rows && pieces <= 1024) {
        const int ch = pieces <= 256 ? 1 : pieces <= 512 ? 2 : 4, threads = (pieces + ch * 32 - 1) / (ch * 32) * 32;
        const size_t smem = static_cast<size_t>(2) * ch * threads * 8 * (sizeof(TX) + sizeof(TD));
        auto kern = ch == 1 ? mx_norm_rows_kernel<TX, TD, 1> : ch == 2 ? mx_norm_rows_kernel<TX, TD, 2> : mx_norm_rows_kernel<TX, TD, 4>;
        int dev = 0, sms = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return LLM_REFUSED_SIZE;
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return static_cast<int>(e);
        const int per_sm = static_cast<int>(216 * 1024 / (smem + 1536)), fit = per_sm * threads > 1024 ? 1024 / threads : per_sm;
        launch_pdl(kern, dim3(n < sms * fit ? n : sms * fit), dim3(threads), smem, s, static_cast<const TX*>(x), static_cast<const TD*>(delta), w,
                   static_cast<TX*>(sum_out), static_cast<unsigned char*>(codes), static_cast<unsigned char*>(scales), n, hidden, kpad, eps, 1.0 / hidden);
        return launch_status();
    }
    const int ch = pieces <= 1024 ? 1 : pieces <= 2048 ? 2 : 4;
    auto kern = vec == 8 ? (ch == 1 ? mx_norm_kernel<TX, TD, 1, true> : ch == 2 ? mx_norm_kernel<TX, TD, 2, true> : mx_norm_kernel<TX, TD, 4, true>)
                         : (ch == 1 ? mx_norm_kernel<TX, TD, 1, false> : ch == 2 ? mx_norm_kernel<TX, TD, 2, false> : mx_norm_kernel<TX, TD, 4, false>);
    launch_pdl(kern, dim3(n), dim3((pieces + ch * 32 - 1) / (ch * 32) * 32), 0, s, static_cast<const TX*>(x), static_cast<const TD*>(delta), w,
               static_cast<TX*>(sum_out), static_cast<unsigned char*>(codes), static_cast<unsigned char*>(scales), rows, hidden, kpad, eps, 1.0 / hidden, vec,
               parts, part_stride);
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
    const long long rows = llm_mx_weight_tiles(N, is_gated) * 128LL;
    MxCut cut;
    const int wide = vec == 8 && dtype == LLM_DT_BF16 ? 4 : 2;   // tiles of K that a warp takes
    cut.per_row = (ktiles + wide - 1) / wide;
    // rows a warp; of 512 values each 4,096 x 4,096: one 10.2 us, two 8.7, four 9.6; 12,288 x 4,096: 27.5, 22.4, 21.9
    cut.u = rows * cut.per_row >= (wide == 4 ? 65536 : 32768) ? 4 : rows * cut.per_row >= 16384 ? 2 : 1;
    const long long items = rows / cut.u * cut.per_row;
    if (items > 0x7fffffffLL) return LLM_REFUSED_SIZE;
    cut.items = static_cast<unsigned>(items);
    cut.blocks = (cut.items + MX_THREADS / 32 - 1) / (MX_THREADS / 32);
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
