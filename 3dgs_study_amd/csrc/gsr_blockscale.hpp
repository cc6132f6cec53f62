// gsr_blockscale.hpp — 8-bit optimiser states: e4m3 codes (OCP: 4 exponent bits,
// bias 7, 3 mantissa bits, largest 448, no infinity) in blocks of 64 consecutive
// elements of the flattened tensor, each with a power-of-two scale 2^(byte - 127)
// in one byte (the E8M0 form).
//
// The scale brings the block's largest finite magnitude to [128, 256): byte =
// max(E - 7, 0) with E that value's fp32 exponent field.  A power of two, so that a
// value that moves to a block of another scale (evicted rows close up) keeps its
// mantissa, and rescaling is exact; one binade below the top, so that rounding up
// never reaches past 256 and nothing saturates.  2^17 of range is left below it.
//
// Encoding by hand (the stochastic rounding of the optimiser step): u = |x| 2^(7 - byte)
// puts e4m3's smallest normal value (2^-6, in units of the scale) on fp32's smallest
// normal (2^-126).  e4m3's subnormals are then fp32's, and code = (bits(u) + 20 random
// bits) >> 20 for every magnitude: the expected value is u.
// A 16-lane DPP row holds one block, 4 elements a lane.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gsr {

constexpr int SCALE_BLOCK = 64;

__device__ __forceinline__ float as_f32(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t as_u32(float f) { return __builtin_bit_cast(uint32_t, f); }

__device__ __forceinline__ float block_scale(uint32_t byte) { return as_f32(byte ? byte << 23 : 0x400000u); }

// four codes (one 32-bit word, the lowest byte first) in units of their scale
__device__ __forceinline__ void e4m3_decode4(uint32_t w, float x[4]) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
}

// magnitude bits that count for a block's largest: an infinity or NaN takes the code
// 0x7F (NaN) for itself and leaves the other 63 elements alone.  So does a magnitude of
// 2^127 or more, which could round up past fp32.
constexpr uint32_t E4M3_TOP = 0x7F000000u;
__device__ __forceinline__ uint32_t coded_bits(float x) {
    const uint32_t a = as_u32(x) & 0x7FFFFFFFu;
    return a < E4M3_TOP ? a : 0u;
}

// largest over the 16 lanes of a DPP row (every lane of the wave active)
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true));  // row_ror:8
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, true));  // row_ror:4
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, true));  // row_ror:2
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, true));  // row_ror:1
    return v;
}
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) { return (uint32_t)max((int)(amax >> 23) - 7, 0); }

// The code of x under the scale byte, rounded up where 16 random bits, centred in the 20 that
// are dropped, carry.  SIGNED: the first moment; else magnitudes (the root of the second
// moment), of which none but zero may become zero: it divides.  TEST: x may be past the
// codes' range.
template <bool SIGNED, bool TEST>
__device__ __forceinline__ uint32_t e4m3_stochastic(float x, uint32_t byte, uint32_t dither) {
    const uint32_t bits = as_u32(x), a = bits & 0x7FFFFFFFu;
    const float v = TEST ? as_f32(coded_bits(x)) : __builtin_fabsf(x);
    uint32_t c = (as_u32(__builtin_ldexpf(v, 7 - (int)byte)) + (dither << 4 | 8u)) >> 20;
    if (!SIGNED) c = max(c, min(a, 1u));
    if (TEST) c = a < E4M3_TOP ? c : 0x7Fu;
    return SIGNED ? c | ((bits >> 24) & 0x80u) : c;
}

// A 32-bit mixing of the published xor-shift-multiply form (shifts by 16, 15 and 16 around
// two odd multipliers; these are the fractional bits of the roots of 2 and 3), and the random word of element i of a tensor from the tensor's key: a pure
// function, so a run repeats and every replica of a data-parallel job rounds alike.
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x ^= x >> 16;
    x *= 0x6A09E667u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}
__host__ __device__ __forceinline__ uint32_t dither_key(uint64_t seed, uint32_t step, uint32_t ordinal) {
    return mix32(mix32(mix32(mix32((uint32_t)seed) + (uint32_t)(seed >> 32)) + step) + ordinal);
}
__device__ __forceinline__ uint32_t dither_word(uint64_t i, uint32_t key) {
    return mix32((uint32_t)i * 0x9E3779B9u + (uint32_t)(i >> 32) * 0x3C6EF373u + key);
}

// vectors at their elements' alignment only (views of flat buffers start anywhere):
// the global loads and stores of gfx950 take them at full width
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint16_t u16x4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32_u __attribute__((aligned(1)));
typedef uint16_t u16_u __attribute__((aligned(1)));

}  // namespace gsr
