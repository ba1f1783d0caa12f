// Microscaled numbers: blocks of 32 neighbouring values of a row share one scale, a power of two, and each value keeps 8 bits
// (e4m3: sign, four bits of exponent, three of mantissa, up to 448) or 4 (e2m1: up to 6).
//
//   scale  the smallest power of two s with max |x| <= largest * s (at least 2^-127), stored as its exponent plus 127
//   code   x / s to the format's nearest value, ties to even: dividing by s is exact, so this is the only rounding, half a step
// A block with an infinity or a NaN has the scale 255: all of it reads as NaN.  A block of zeros has scale 0 (2^-127) and codes 0.
// Such a scale never saturates: a smaller one (the exponent of the largest value) would cut up to a quarter off the largest values.
//
// Where the bytes lie: rows are padded with zeros to whole tiles of 128 values, whose four scales are one 32-bit word.  The words of
// 128 rows are a piece of 512 bytes: the word of row r (of 128) at 16 (r % 32) + 4 (r / 32), which is how the block-scaled tensor-core
// products take them (32 lanes of 16 bytes).  Pieces lie by tile of 128 rows, then by tile of 128 values.
//   rows (8 bits): codes [rows][padded k], one byte each
//   a weight (4 bits): tiles [tile of 128 rows][tile of 128 values][128][64 bytes], the lower half of a byte the earlier value; a
//   product fetches a tile as one box of 8 KB
#pragma once

#include "common.cuh"

#include <cstddef>

#define MX_BLOCK 32
#define MX_K 128                  // values of a tile's row
#define MX_PIECE 512              // bytes of the scales of 128 rows x 128 values
#define MX_E2M1 4
#define MX_E4M3 8

// Where the scale of block `kb` of a row lies (the byte; of kb = 4 n the word).
__host__ __device__ __forceinline__ size_t mx_scale_at(size_t row, int kb, int ktiles) {
    return ((row >> 7) * ktiles + (kb >> 2)) * MX_PIECE + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (kb & 3);
}
// Rows that stand behind T rows of 8 bits, so that hardly a box of a product (16, 32 or 64 rows, or 192 of a pair) reaches beyond them, which takes
// longer, nor beyond whole pieces of scales; the scales stand behind the codes.
static inline long long mx_padded_rows(int T) { return T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : T <= 128 ? 128 : (T + 383LL) / 384 * 384; }
static inline int mx_tiles(int k) { return (k + MX_K - 1) / MX_K; }
static inline unsigned char* mx_row_scales(void* rows, int T, int K) { return static_cast<unsigned char*>(rows) + mx_padded_rows(T) * mx_tiles(K) * MX_K; }
extern "C" int llm_mx_rows(const void* x, int dtype, void* rows, int T, int K, uintptr_t stream);

// The stored scale of a block from the bits of its largest magnitude (as integers these are in order, NaN above infinity above all).
template <int FMT> __device__ __forceinline__ unsigned mx_scale(unsigned most) {
    constexpr unsigned EXP = FMT == MX_E4M3 ? 8 : 2, MANT = FMT == MX_E4M3 ? 0x600000u : 0x400000u;      // largest: 1.75 * 2^8, 1.5 * 2^2
    const unsigned e = (most >> 23) + ((most & 0x7fffffu) > MANT ? 1u : 0u);
    return most >= 0x7f800000u ? 255u : e > EXP ? e - EXP : 0u;
}
__device__ __forceinline__ float mx_inverse(unsigned scale) { return __uint_as_float((254u - min(scale, 253u)) << 23); }      // 1 / s, exact
__device__ __forceinline__ float mx_value(unsigned scale) {
    return __uint_as_float(scale == 255u ? 0x7fc00000u : scale ? scale << 23 : 0x400000u);
}
__device__ __forceinline__ unsigned mx_abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Four values, already divided by their scale: 32 bits of e4m3, 16 bits of e2m1; the first value lowest.
__device__ __forceinline__ unsigned mx_e4m3x4(float a, float b, float c, float d) {
    unsigned r;
    asm("{\n .reg .b16 lo, hi;\n cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n mov.b32 %0, {lo, hi};\n}\n"
        : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}
__device__ __forceinline__ unsigned mx_e2m1x8(const float (&v)[8]) {
    unsigned r;
    asm("{\n .reg .b8 a, b, c, d;\n cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n mov.b32 %0, {a, b, c, d};\n}\n"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// Eight values of 4 bits, or four of 8 bits, as float32 (through 16-bit floats, which hold all of them).
__device__ __forceinline__ float2 mx_halves(unsigned h) {
    float2 f;
    asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %2;\n cvt.f32.f16 %0, lo;\n cvt.f32.f16 %1, hi;\n}\n" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}
__device__ __forceinline__ void mx_from_e2m1x8(unsigned r, float (&v)[8]) {
    unsigned h[4];
    asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
        " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}\n" : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(r));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = mx_halves(h[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void mx_from_e4m3x4(unsigned r, float* v) {
    unsigned lo, hi;
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}\n" : "=r"(lo), "=r"(hi) : "r"(r));
    const float2 a = mx_halves(lo), b = mx_halves(hi);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}

// Eight values as they lie in memory, read in one or two loads; their largest magnitude's bits (of float32), and themselves.
__device__ __forceinline__ void mx_raw8(const bf16* p, uint4& raw) { raw = *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ unsigned mx_most8(const uint4& r) {    // two 16-bit magnitudes an instruction
    const unsigned m = __vmaxu2(__vmaxu2(r.x & 0x7fff7fffu, r.y & 0x7fff7fffu), __vmaxu2(r.z & 0x7fff7fffu, r.w & 0x7fff7fffu));
    return max(m & 0xffff0000u, m << 16);
}
__device__ __forceinline__ void mx_raw_values(const uint4& r, float (&v)[8]) {
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
__device__ __forceinline__ unsigned mx_most8(const float (&v)[8]) {
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, mx_abs_bits(v[i]));
    return most;
}
// Eight neighbouring values a lane, four lanes a block, sixteen a tile's row: the lane's codes, and the four blocks' scales as one
// word in every lane of the sixteen.  most: of the lane's values.  All lanes of a warp are here.
__device__ __forceinline__ unsigned mx_block_most(unsigned most) {
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    return max(most, __shfl_xor_sync(0xffffffffu, most, 2));
}
__device__ __forceinline__ unsigned mx_word(unsigned scale) {
    unsigned word = scale << (8 * ((threadIdx.x >> 2) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    return word | __shfl_xor_sync(0xffffffffu, word, 8);
}
template <int FMT> __device__ __forceinline__ uint2 mx_encode8(const float (&v)[8], unsigned most, unsigned& word) {
    const unsigned scale = mx_scale<FMT>(mx_block_most(most));
    const float inv = mx_inverse(scale);
    word = mx_word(scale);
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = v[i] * inv;
    if constexpr (FMT == MX_E2M1) return make_uint2(mx_e2m1x8(q), 0u);
    else return make_uint2(mx_e4m3x4(q[0], q[1], q[2], q[3]), mx_e4m3x4(q[4], q[5], q[6], q[7]));
}
template <int FMT> __device__ __forceinline__ uint2 mx_encode8(const float (&v)[8], unsigned& word) { return mx_encode8<FMT>(v, mx_most8(v), word); }
// Sixteen neighbouring values a lane as they lie in memory, two lanes a block, eight a tile's row: the same with half the exchanges and scales.
template <int FMT> __device__ __forceinline__ uint4 mx_encode16(const uint4& a, const uint4& b, unsigned& word) {
    unsigned most = max(mx_most8(a), mx_most8(b));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    const unsigned scale = mx_scale<FMT>(most);
    const float inv = mx_inverse(scale);
    word = scale << (8 * ((threadIdx.x >> 1) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 2);
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    float p[8], q[8];
    mx_raw_values(a, p);
    mx_raw_values(b, q);
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] *= inv, q[i] *= inv;
    if constexpr (FMT == MX_E2M1) return make_uint4(mx_e2m1x8(p), mx_e2m1x8(q), 0u, 0u);
    else return make_uint4(mx_e4m3x4(p[0], p[1], p[2], p[3]), mx_e4m3x4(p[4], p[5], p[6], p[7]), mx_e4m3x4(q[0], q[1], q[2], q[3]), mx_e4m3x4(q[4], q[5], q[6], q[7]));
}
__device__ __forceinline__ void mx_store_codes8(uint2 c, unsigned word, bool there, size_t row, int col, int kpad, unsigned char* codes, unsigned char* scales) {
    if (!there) return;
    *reinterpret_cast<uint2*>(codes + row * kpad + col) = c;
    if ((col & (MX_K - 1)) == 0) *reinterpret_cast<unsigned*>(scales + mx_scale_at(row, col / MX_BLOCK, kpad / MX_K)) = word;
}
// The row's eight values from column `col` on (a multiple of 8), which lane threadIdx.x % 16 == col / 8 % 16 holds, to rows of 8 bits.
__device__ __forceinline__ void mx_store_row8(const float (&v)[8], unsigned most, bool there, size_t row, int col, int kpad, unsigned char* codes, unsigned char* scales) {
    unsigned word;
    const uint2 c = mx_encode8<MX_E4M3>(v, most, word);
    mx_store_codes8(c, word, there, row, col, kpad, codes, scales);
}
// Eight values from column `col` on of a row of `n`; zeros beyond it.  vec 8: rows of whole, aligned pieces of eight; 2: of pairs; 1: any.
__device__ __forceinline__ float2 mx_load2(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 mx_load2(const bf16* p) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p)); }
__device__ __forceinline__ void mx_store2(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void mx_store2(bf16* p, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b); }
template <bool FAST, typename T> __device__ __forceinline__ void mx_load8(const T* row, int col, int n, int vec, float (&v)[8]) {
    if constexpr (FAST) {                                         // vec 8, without a branch around the loads
        if (col < n) load8(row + col, v);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        if (vec == 2) {
#pragma unroll
            for (int i = 0; i < 8; i += 2)
                if (col + i < n) {
                    const float2 f = mx_load2(row + col + i);
                    v[i] = f.x, v[i + 1] = f.y;
                }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (col + i < n) v[i] = to_f32(row[col + i]);
        }
    }
}
template <bool FAST, typename T> __device__ __forceinline__ void mx_put8(T* row, int col, int n, int vec, const float (&v)[8]) {
    if constexpr (FAST) {
        if (col < n) store8(row + col, v);
    } else if (vec == 2) {
#pragma unroll
        for (int i = 0; i < 8; i += 2)
            if (col + i < n) mx_store2(row + col + i, v[i], v[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < n) row[col + i] = from_f32<T>(v[i]);
    }
}
// How rows of n values of `size` bytes from p on (null: nothing) can be read or written.
static inline int mx_vec(int n, const void* p, int size) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return n % 8 == 0 && (at & 15) == 0 ? 8 : n % 2 == 0 && (at & (2 * size - 1)) == 0 ? 2 : 1;
}
static inline int mx_vec(int a, int b) { return a < b ? a : b; }

// A gated feed-forward's middle, all of its kinds in one form without branches: g * sigmoid(z) * (u + shift), z = g * (alpha + beta g^2), g and u
// clamped by `limit` (infinity: not).  silu: z = g; the tanh form of gelu is g * sigmoid(2 sqrt(2/pi) (g + 0.044715 g^3)), because
// (1 + tanh(z / 2)) / 2 = sigmoid(z); the clamped form: z = 1.702 g, shift 1.  The division is the fast one and one of Newton's steps, which
// squares its error, so that the result is as near as float32 has it: a value that is off crosses a border between two codes more often.  With
// the compiler's division and a branch a kind eight values took a thread of the product's result 3,200 clocks, longer than the products.
// A NaN stays one.
struct MxAct {
    float limit, alpha, beta, shift;
    double alpha64, beta64;
    unsigned near;                        // places beside a border within which a value is made in 64 bits: more than mx_gated is off by (mx_act)
};
__device__ __forceinline__ float mx_gated(float g, float u, const MxAct& a) {
    g = g > a.limit ? a.limit : g;
    u = u > a.limit ? a.limit : u < -a.limit ? -a.limit : u;
    const float d = 1.0f + expf(-g * (a.alpha + a.beta * g * g)), s = __fdividef(1.0f, d), t = fmaf(-d, s, 1.0f);
    return g * (fabsf(t) <= 1.0f ? fmaf(s, t, s) : s) * (u + a.shift);       // t is none of these where d is infinite or beyond what the fast form takes
}
// The same in 64 bits, rounded to odd (towards zero, and a one as last bit where that is not the whole of it), which makes the rounding to 8 bits
// the only one.
static __device__ __noinline__ float mx_gated_carried(float g, float u, double alpha, double beta, float limit, float shift) {
    const double x = g > limit ? limit : g, y = u > limit ? limit : u < -limit ? -limit : u;
    const double r = x * (1.0 / (1.0 + exp(-x * (alpha + beta * x * x)))) * (y + shift);
    const float f = __double2float_rz(r);
    return f == r ? f : __int_as_float(__float_as_int(f) | 1);
}
// Codes and scale of four neighbouring features of a token, eight lanes a block.  CARRY: a value beside a border between two codes, or a block whose
// largest is beside one between two scales, is made in 64 bits, one in 30,000 (the lowest codes, 2^-15 of a block's largest, may be a step off): what
// is left is the rounding of the sums.  Of 25 million codes 26 are off without it, as with float32 throughout, 11 with it; it costs products of
// few rows nothing, those of many 5 to 33 % (300 x 2 x 4,096 x 4,096 18.3 to 19.3 us, 2,045 x 2 x 12,288 x 4,096 162 to 215), which do without, as rows made of gate and up values in memory do.
template <bool CARRY> __device__ __forceinline__ unsigned mx_gated_codes(const float4& g, const float4& u, const MxAct& a, unsigned& scale) {
    float v[4] = {mx_gated(g.x, u.x, a), mx_gated(g.y, u.y, a), mx_gated(g.z, u.z, a), mx_gated(g.w, u.w, a)};
    auto largest = [&]() {
        unsigned most = max(max(mx_abs_bits(v[0]), mx_abs_bits(v[1])), max(mx_abs_bits(v[2]), mx_abs_bits(v[3])));
#pragma unroll
        for (int o = 1; o < 8; o *= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        return most;
    };
    const unsigned most = largest();
    scale = mx_scale<MX_E4M3>(most);
    float inv = mx_inverse(scale);
    if constexpr (!CARRY) return mx_e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    const bool all = (most & 0x7fffffu) - (0x600000u - a.near) <= 2u * a.near;
    unsigned border = ~0u;                                        // places from `near` below a border on, in the upper 20 bits
#pragma unroll
    for (int i = 0; i < 4; ++i) border = min(border, __float_as_uint(v[i] * inv) * 4096u - ((0x80000u - a.near) << 12));
    if (__any_sync(0xffffffffu, all || border <= (2u * a.near << 12))) {
        const float gs[4] = {g.x, g.y, g.z, g.w}, us[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (all || __float_as_uint(v[i] * inv) * 4096u - ((0x80000u - a.near) << 12) <= (2u * a.near << 12))
                v[i] = mx_gated_carried(gs[i], us[i], a.alpha64, a.beta64, a.limit, a.shift);
        __syncwarp();
        scale = mx_scale<MX_E4M3>(largest());
        inv = mx_inverse(scale);
    }
    return mx_e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
}
// mx_gated is off by up to 10 places (expf 2 of 2^-23, the division as much, each other step a half); where its exponent z is itself rounded, by up to 8 more for
// each of z, which is at most 75 before a value is nothing beside 2^-95: 610.  What is taken as beside a border is the next power of two, 16 and 1,024.
static inline bool mx_act(int kind, float limit, MxAct* a) {
    if (kind < 0 || kind > 2 || (kind == 2 && !(limit > 0.0f))) return false;
    constexpr double gelu = 1.5957691216057308;                   // 2 sqrt(2 / pi)
    const float none = __builtin_inff();
    const double alpha = kind == 2 ? 1.702 : kind == 1 ? gelu : 1.0, beta = kind == 1 ? gelu * 0.044715 : 0.0;
    *a = {kind == 2 ? limit : none, static_cast<float>(alpha), static_cast<float>(beta), kind == 2 ? 1.0f : 0.0f, alpha, beta, kind == 0 ? 16u : 1024u};
    return true;
}
