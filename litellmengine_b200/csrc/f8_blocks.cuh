// Numbers in 8 bits (e4m3: sign, four bits of exponent, three of mantissa, up to 448) under float32 scales: one scale for each block of
// 128 x 128 values of a weight, one for each 128 neighbouring values of a row of activations.
//
//   scale  the block's largest magnitude / 448, rounded to float32, at least 2^-126
//   code   x * 448 / largest (x * 2^126 under the least scale) to the format's nearest value, ties to even, of the quotient as a real number
//          (rows that products in tiles of 128 and 256 rows make of gate and up values: nearest to the float32 quotient, x * (448 / largest) rounded twice, which can lie
//          on the other side of a middle where the real one is within 2^-22 of it)
// A block with an infinity or a NaN has the scale NaN: all of it reads as NaN, and so does every sum that it is in.
// Scales are multiplied with each other in float32 before a tile's sum is: results below 2^-126 * 448 * 448 or so lose digits, and blocks whose scales' product passes
// float32's range give infinities and NaNs.
//
// Where the bytes lie: K is padded with zeros to whole tiles of 128 values.
//   rows     codes [tile of K][rows, padded][128], behind them float32 scales [rows, padded][tiles of K, padded to fours]: the products take a tile of K of
//            neighbouring rows as one box, whatever row it starts at
//   weights  codes [matrix of a stack][tile of 128 rows][tile of K][128][128], 16 KB that lie side by side; behind them float32 scales
//            [...][3][tiles of K, padded to fours].  An even number of tiles.  A gated weight [gate; up] has 64 gate rows and the 64 up rows beside them in a tile; its
//            values are those of the same matrix without that, whose blocks count from the first row of gate.  So the 64 up rows may lie in two blocks, where the
//            number of gate rows is no multiple of 64: the three scales of a tile are those of its first 64 rows, of its 65th, and of its last
#pragma once

#include "microscaling.cuh"

#define F8_K 128                  // values of a tile's row
#define F8_MOST_EXPERTS 4096      // that a call routes to
#define F8_TILE (128 * F8_K)      // bytes of a weight's tile
#define F8_TOP 448.0f
#define F8_LEAST 1.17549435082228750797e-38f          // 2^-126

// Rows that stand behind T rows: hardly a box of a product (16, 32, 64 or 128 rows) then reaches beyond them, which takes longer.
static inline long long f8_padded_rows(long long T) { return T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : (T + 127) / 128 * 128; }
static inline int f8_tiles(int k) { return (k + F8_K - 1) / F8_K; }
static inline int f8_k4(int k) { return (f8_tiles(k) + 3) / 4 * 4; }       // room for a row's scales
// Gated: the first of a tile's 64 up rows that lie in the second of two blocks; 64: none does.  i: the tile's number in its matrix.
__host__ __device__ __forceinline__ int f8_split(int gate_rows, int i) {
    const int at = 128 - (gate_rows + 64 * i) % 128;
    return at < 64 ? at : 64;
}
static inline float* f8_row_scales(void* rows, long long padded, int ktiles) {
    return reinterpret_cast<float*>(static_cast<unsigned char*>(rows) + padded * ktiles * F8_K);
}

// A block's scale, and what its values are multiplied by, from the bits of its largest magnitude (as integers these are in order, NaN above infinity
// above all).
struct F8Scale {
    float scale, inverse;
};
__device__ __forceinline__ F8Scale f8_scale(unsigned most) {
    const float m = __uint_as_float(most);
    if (most >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.0f};
    if (m <= F8_TOP * F8_LEAST) return {F8_LEAST, 8.50705917302346158658e37f};       // 2^126
    return {__fdiv_rn(m, F8_TOP), __fdiv_rn(F8_TOP, m)};
}

// x * inverse, ready for the converter.  x * 448 / largest as float32 has it is off by less than 2^-22, which matters where the quotient lies next to a middle
// between two codes.  Of bfloat16 values it either is such a middle m or is 2^-14 of it away: x * 448 - m * largest, in units of the last places of both, is a whole
// number, of terms below 2^14.  So rounding to 18 bits puts the quotients that are middles there and moves none across.
__device__ __forceinline__ float f8_near_16(float q) { return __uint_as_float((__float_as_uint(q) + 16u) & ~31u); }
// Of float32 values the doubtful ones, within 2^-20 of a middle (one in 60,000), are compared with it as real numbers: x * 448 against m * largest, both
// as float32 and what that leaves of it, which multiplication and addition in one have exactly.  All differences are exact there, so the sign is that of the real one,
// and the middle itself or its neighbour on that side goes to the converter.  Both sides are first brought where neither overflows nor what is left of them is cut.
// Measured, with a division in 64 bits of these and of all that is below the format's normal range instead, and so (us): float32 rows 4,096 x 4,096 19.9 and 18.5, 4,096 x 12,288
// 52 and 49, weights 12,288 x 4,096 61 and 46, 1,003 x 1,358 6.0 and 4.6.
__device__ __forceinline__ float f8_place(float q) {              // the last 20 bits: 0x80000 in a middle
    const float a = fabsf(q);
    return a < 0.015625f ? a + 0.015625f : a;                     // 2^-6: below it codes lie 2^-9 apart, as they do in the octave from there on
}
#define F8_BESIDE (16u << 12)
__device__ __forceinline__ unsigned f8_beside(float q) {          // up to F8_BESIDE: within eight places of a middle
    return __float_as_uint(f8_place(q)) * 4096u - ((0x80000u - 8u) << 12);
}
__device__ __forceinline__ float f8_settled(float q, float x, unsigned most) {
    const unsigned at = (__float_as_uint(f8_place(q)) & ~0xfffffu) | 0x80000u;
    const float m = __uint_as_float(at) - (fabsf(q) < 0.015625f ? 0.015625f : 0.0f);       // the middle
    // Under the least scale the quotient is x * 2^126 and nothing is left to settle.
    if (f8_beside(q) > F8_BESIDE || most >= 0x7f800000u || most <= __float_as_uint(F8_TOP * F8_LEAST)) return q;
    const float by = most < 0x3f800000u ? 1.26765060022822940150e30f : 9.5367431640625e-7f;      // 2^100, 2^-20
    const float y = fabsf(x) * by, z = __uint_as_float(most) * by;
    const float p = __fmul_rn(y, F8_TOP), t = __fmul_rn(m, z), d = __fadd_rn(__fsub_rn(p, t), __fsub_rn(fmaf(y, F8_TOP, -p), fmaf(m, z, -t)));
    return copysignf(__uint_as_float(__float_as_uint(m) + (d > 0.0f) - (d < 0.0f)), x);
}
// q: x * inverse of values that share a block.
template <int N> __device__ __forceinline__ void f8_settle(float (&q)[N], const float (&x)[N], unsigned most) {
    unsigned border = ~0u;
#pragma unroll
    for (int i = 0; i < N; ++i) border = min(border, f8_beside(q[i]));
    if (border > F8_BESIDE) return;
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = f8_settled(q[i], x[i], most);
}
// Eight values that share a block.
__device__ __forceinline__ uint2 f8_codes8(const uint4& raw, unsigned, float inverse) {
    float v[8];
    mx_raw_values(raw, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f8_near_16(v[i] * inverse);
    return make_uint2(mx_e4m3x4(v[0], v[1], v[2], v[3]), mx_e4m3x4(v[4], v[5], v[6], v[7]));
}
__device__ __forceinline__ uint2 f8_codes8(const float (&x)[8], unsigned most, float inverse) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[i] * inverse;
    f8_settle(v, x, most);
    return make_uint2(mx_e4m3x4(v[0], v[1], v[2], v[3]), mx_e4m3x4(v[4], v[5], v[6], v[7]));
}
// The largest magnitude of sixteen neighbouring lanes.
__device__ __forceinline__ unsigned f8_most16(unsigned most) {
#pragma unroll
    for (int o = 1; o < 16; o *= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    return most;
}

// Rows that a router has sorted by expert.  Items are up to a tile's rows of one expert; what stands behind the last is not read.  Or, for a token or a few, the picks
// as they are, each a row and an item of its own (ids, [tokens][top]; weights [tokens][top]).
struct F8Groups {
    const int32_t* ids;                   // or null
    int top, E;
    const int32_t* counts;                // items, rows
    const int4* items;                    // expert, first row, rows
    const float* weights;                 // [rows] its weight, or null
};
extern "C" int llm_f8_rows(const void* x, int dtype, void* rows, long long padded, int T, int K, const int32_t* places, int top, uintptr_t stream);
