// FP4 values with shared scales (the OCP microscaling format): groups of 32 values along a
// row share a scale 2^(b - 127), b one byte (255: the group is NaN), and a value is one of
// 0, 0.5, 1, 1.5, 2, 3, 4, 6 times the scale, with a sign in bit 3 of its 4-bit code. A value
// has two significant bits, so value times scale is exact in bf16 (subnormals included; 2^128 and
// more is infinite there): every kernel here feeds the bf16 matrix cores what is stored, no scale meets an accumulator, and kernels that read
// the same codes see the same numbers. gfx950 turns two codes and a scale into two bf16 in one
// instruction of the full VALU rate (v_cvt_scalef32_pk_bf16_fp4; a scale of exponent 255 gives
// NaN for every code).
//
// Quantisation: the scale is the least power of two with max |x| <= 7 * scale, at least
// 2^-125 (so that no value needs a bf16 subnormal) and at most 2^125 (so that none is infinite;
// larger groups are NaN), and a value is rounded to the nearest of
// the grid, of two as near to the one with the even code. Up to 7 the nearest is at most half
// a step of the grid away. Scaling by a power of two is exact, so for bf16 inputs the codes
// are defined bit for bit.
#pragma once
#include "common.hpp"

namespace efm {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kFp4Group = 32;
constexpr uint32_t kFp4ScaleNan = 255;
// A grid's threads stay below 2^32: past that the runtime starts the remainder alone, without an error.
constexpr int64_t kGridThreads = 0xffffffffll;
constexpr int kFp4MinExp = -125, kFp4MaxExp = 125;

// The scale as fp32 (byte 0 comes out as 0, which the conversion reads as 2^-127).
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Byte i of a word of scale bytes, for the conversions, which take the exponent bits alone: the
// word's other bytes are not cleared from the sign and mantissa.
__device__ __forceinline__ float fp4_scale_at(uint32_t bytes, int i) {
    return __uint_as_float(i < 3 ? bytes << (23 - 8 * i) : bytes >> 1);
}

// Codes 2 B and 2 B + 1 of a word (low half byte first) as packed bf16.
template <int B>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t word, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, B));
}

// The 8 codes of a word, in order.
__device__ __forceinline__ bf16x8_t fp4_unpack8(uint32_t word, float scale) {
    const uint4 u = make_uint4(fp4_pair<0>(word, scale), fp4_pair<1>(word, scale), fp4_pair<2>(word, scale),
                               fp4_pair<3>(word, scale));
    return __builtin_bit_cast(bf16x8_t, u);
}

// Exponent of the scale for a group whose largest magnitude is m * 2^E, 1 <= m < 2.
__device__ __forceinline__ int fp4_exp(int E, bool over_1_75) { return max(E - 2 + (over_1_75 ? 1 : 0), kFp4MinExp); }

// Scale byte for the largest magnitude of a group, given as its fp32 bits (sign cleared).
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t abs_bits) {
    const int e = fp4_exp((int)(abs_bits >> 23) - 127, (abs_bits & 0x7fffffu) > 0x600000u);
    return e > kFp4MaxExp ? kFp4ScaleNan : (uint32_t)(e + 127);
}

// Two codes of values already divided by the scale, in the low byte: v_cvt_scalef32_pk_fp4_f32
// rounds to nearest even and saturates at 6.
__device__ __forceinline__ uint32_t fp4_encode2(float a, float b) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a, b, 1.0f, 0) & 0xffu;
}

// Eight values of a group as one word of codes.
__device__ __forceinline__ uint32_t fp4_encode8(const float* x, uint32_t byte) {
    if (byte == kFp4ScaleNan) return 0;
    const int e = 127 - (int)byte;
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= fp4_encode2(ldexpf(x[2 * i], e), ldexpf(x[2 * i + 1], e)) << (8 * i);
    return w;
}

// The same for values held in 64 bits. The conversion takes fp32, and an fp32 rounding that
// lands on a border of the grid (whose mantissas are 4 bits long) would lose the side that the
// value is on: those are moved one step of fp32 back to it.
__device__ __forceinline__ float fp4_sticky_f32(double a) {
    const float f = (float)a;
    const double d = a - (double)f;
    const uint32_t bits = __float_as_uint(f);
    if ((bits & 0x7ffffu) != 0 || d == 0.0 || f == 0.f) return f;
    return __uint_as_float((d > 0.0) == (f > 0.f) ? bits + 1 : bits - 1);
}

__device__ __forceinline__ uint32_t fp4_encode8(const double* x, uint32_t byte) {
    if (byte == kFp4ScaleNan) return 0;
    const int e = 127 - (int)byte;
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w |= fp4_encode2(fp4_sticky_f32(ldexp(x[2 * i], e)), fp4_sticky_f32(ldexp(x[2 * i + 1], e))) << (8 * i);
    return w;
}

// The same for a magnitude in 64 bits.
__device__ __forceinline__ uint32_t fp4_scale_byte(uint64_t abs_bits) {
    const int E = (int)(abs_bits >> 52) - 1023;
    const int e = fp4_exp(E, (abs_bits & 0xfffffffffffffull) > 0xc000000000000ull);
    return e > kFp4MaxExp ? kFp4ScaleNan : (uint32_t)(e + 127);
}

// Geometry of an FP4 cache of one layer for Hkv heads of HD channels and T rows (a multiple of
// 32). Four regions follow each other; Hkv * T * HD * 17 / 16 bytes in all:
//   K codes   [Hkv][T][4 pieces g][HD / 32 words w]: word w of piece g holds channels
//             32 w + 8 g .. + 7, so that the lanes of a 16-key operand tile of the matrix cores
//             (key lane % 16, piece lane / 16) take their words of every 32-channel step in one
//             load
//   V codes   [Hkv][T / 8][HD / 8 octets][8 rows]: a word holds 8 consecutive channels of a row;
//             a lane that multiplies 8 consecutive rows takes its octet of them in 32 bytes
//   K scales  [Hkv][T][HD / 32] bytes
//   V scales  [Hkv][T / 8][HD / 32][8 rows] bytes
struct KvFp4Layout {
    size_t T;
    int Hkv, HD;
    __host__ __device__ static size_t rows(uint32_t max_rows) { return ((size_t)max_rows + 31) / 32 * 32; }
    __host__ __device__ KvFp4Layout(size_t T_, int Hkv_, int HD_) : T(T_), Hkv(Hkv_), HD(HD_) {}
    __host__ __device__ size_t codes() const { return (size_t)Hkv * T * (HD / 2); }
    __host__ __device__ size_t scales() const { return (size_t)Hkv * T * (HD / 32); }
    __host__ __device__ size_t bytes() const { return 2 * (codes() + scales()); }
    __host__ __device__ size_t k(int h) const { return (size_t)h * T * (HD / 2); }
    __host__ __device__ size_t v(int h) const { return codes() + k(h); }
    __host__ __device__ size_t ks(int h) const { return 2 * codes() + (size_t)h * T * (HD / 32); }
    __host__ __device__ size_t vs(int h) const { return scales() + ks(h); }
    // offsets inside a head's region: word of octet j (channels 8 j ..) of a row, and scale
    // byte of its group j / 4
    __host__ __device__ size_t k_word(size_t row, int j) const {
        return row * (HD / 2) + (j % 4) * (HD / 8) + (j / 4) * 4;
    }
    __host__ __device__ size_t v_word(size_t row, int j) const { return ((row / 8) * (HD / 8) + j) * 32 + row % 8 * 4; }
    __host__ __device__ size_t k_scale(size_t row, int j) const { return row * (HD / 32) + j / 4; }
    __host__ __device__ size_t v_scale(size_t row, int j) const {
        return ((row / 8) * (HD / 32) + j / 4) * 8 + row % 8;
    }
};

}  // namespace efm
