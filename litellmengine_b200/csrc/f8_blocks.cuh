// Numbers in 8 bits (e4m3: sign, four bits of exponent, three of mantissa, up to 448) under float32 scales: one scale for each block of
// 128 x 128 values of a weight, one for each 128 neighbouring values of a row of activations.
//
//   scale  the block's largest magnitude / 448, rounded to float32, at least 2^-126
//   code   x * 448 / largest (x * 2^126 under the least scale) to the format's nearest value, ties to even, of the quotient as a real number
// A block with an infinity or a NaN has the scale NaN: all of it reads as NaN, and so does every sum that it is in.
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
// Of float32 values the doubtful ones (one in 60,000, and what is below the format's normal range) are divided in 64 bits, where a middle comes
// out as one and what is none, which is 2^-30 away at least, does not; rounding that to odd (towards zero, and a one as last bit where that is not the
// whole of it) makes the converter's rounding the only one.
static __device__ __noinline__ float f8_divided(float x, unsigned most) {
    const float m = __uint_as_float(most);
    const double q = m <= F8_TOP * F8_LEAST ? static_cast<double>(x) * 8.50705917302346158658e37 : static_cast<double>(x) * 448.0 / m;
    const float f = __double2float_rz(q);
    return f == q ? f : __uint_as_float(__float_as_uint(f) | 1u);
}
__device__ __forceinline__ float f8_near_32(float q, float x, unsigned most) {
    const unsigned b = __float_as_uint(q) & 0x7fffffffu;
    const bool doubtful = (b & 0xfffffu) - (0x80000u - 8u) <= 16u || (b < 0x3c800000u && b);       // 2^-6
    return doubtful && most < 0x7f800000u ? f8_divided(x, most) : q;
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
    for (int i = 0; i < 8; ++i) v[i] = f8_near_32(x[i] * inverse, x[i], most);
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
