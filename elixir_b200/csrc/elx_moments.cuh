// Part of the elixir_b200 CUDA library (C ABI: include/elixir_b200.h): the 8-bit form of the two Adam moments.
//
// A shard of n elements has one state array per moment: n codes, then, from the next multiple of 16 bytes, one
// exponent byte E per block of 256 elements.  A code is a small float relative to 2^(E - 127):
//   first moment    sign, 4 exponent bits f, 3 mantissa bits t:  (f ? 1 + t/8 : t/4) * 2^(f - 15)
//   second moment         5 exponent bits f, 3 mantissa bits t:  (f ? 1 + t/8 : t/4) * 2^(f - 31)
// (t/4 * 2^-15 is the t/8 * 2^-14 of a subnormal).  Why floats and not evenly spaced levels: an update divides an
// element's first moment by the root of its own second moment, so what matters is each moment's relative precision
// down to elements far below the largest of their block; 2^-18 and 2^-33 of the block's top are still representable.
// The scale is a power of two so that decoding, scaling and the choice of the code are exact operations on the bits
// of fp32 numbers: no table, no division, and the same code on every path.
//
// E = 0: all zero.  E = 255: the block held an inf or a NaN; every element decodes to NaN.  Otherwise E is the fp32
// exponent field of the largest magnitude, one more when that magnitude is above 1.875 of its power of two (the top
// code), so no rounding passes the top code.
#pragma once

#include "elx_common.cuh"

namespace elx {

constexpr int kMomentBlock = 256;

struct FirstMoment {
    static constexpr uint32_t kTop = 127;
    static constexpr bool kSigned = true;
    static __device__ __forceinline__ float up() { return __uint_as_float((112u + 127u) << 23); }     // 2^112
    static __device__ __forceinline__ float down() { return __uint_as_float((127u - 112u) << 23); }   // 2^-112
};
struct SecondMoment {
    static constexpr uint32_t kTop = 255;
    static constexpr bool kSigned = false;
    static __device__ __forceinline__ float up() { return __uint_as_float((96u + 127u) << 23); }
    static __device__ __forceinline__ float down() { return __uint_as_float((127u - 96u) << 23); }
};

__host__ __device__ inline int64_t moment_blocks(int64_t n) { return (n + kMomentBlock - 1) / kMomentBlock; }
// Where the exponent bytes start, and the size of a state array.
__host__ __device__ inline int64_t moment_exps_at(int64_t n) { return (n + 15) / 16 * 16; }
__host__ __device__ inline int64_t moment_state_bytes(int64_t n) { return moment_exps_at(n) + (moment_blocks(n) + 15) / 16 * 16; }

// Scale of a block when its codes are read: 2^(E - 127), 0 or NaN.
__device__ __forceinline__ float decode_scale(uint32_t e) { return __uint_as_float(e == 255u ? 0x7FC00000u : e << 23); }

// The code's bits as an fp32 number (possibly subnormal) times a power of two times the scale: both products exact
// unless the moment itself is below fp32's normal range.
template <class M>
__device__ __forceinline__ float decode(uint32_t code, float scale) {
    const float x = __uint_as_float((code & M::kTop) << 20) * M::up() * scale;
    return M::kSigned ? __uint_as_float(__float_as_uint(x) | ((code & 0x80u) << 24)) : x;
}

// Exponent byte of a block from the bits of its largest magnitude.
__device__ __forceinline__ uint32_t block_exponent(uint32_t top_bits) {
    if (top_bits >= 0x7F800000u) return 255u;
    const uint32_t e = (top_bits + 0xFFFFFu) >> 23;
    return top_bits == 0u ? 0u : min(max(e, 1u), 253u);
}
// 2^(127 - E), the first factor of an encoding (any E: the codes of an all-zero or non-finite block do not matter).
__device__ __forceinline__ float encode_scale(uint32_t e) { return __uint_as_float((254u - min(max(e, 1u), 253u)) << 23); }

// `dither` (20 bits) is added below the kept bits: 1 << 19 rounds to nearest, uniform bits round up with the
// probability that makes the expected value exact -- the codes are evenly spaced between two powers of two, and so
// are the bits of fp32.  A positive second moment never becomes zero: a zero there with a first moment that is not
// would be a division by eps alone.
template <class M>
__device__ __forceinline__ uint32_t encode(float x, float scale, uint32_t dither) {
    const float z = fabsf(x) * scale * M::down();
    uint32_t c = min((__float_as_uint(z) + dither) >> 20, M::kTop);
    if (M::kSigned) return c | ((__float_as_uint(x) >> 24) & 0x80u);
    return x > 0.0f ? max(c, 1u) : c;
}

constexpr uint32_t kRoundNearest = 0x80000u;

// 32 mixed bits: three xor-shifts around two multiplications.  The multipliers are odd numbers without structure; the first, which
// also spreads the places, is the prime next to 2^32 over the golden ratio.  What is asked of them, measured: a flipped input bit
// flips each output bit with a probability within 0.019 of a half (4 Mi inputs), and the two halves of a draw, like those
// of neighbouring places, are correlated by less than 0.001 (5 Mi draws).
__device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x9E3779B1u;
    x = (x ^ (x >> 15)) * 0x85157AF5u;
    return x ^ (x >> 16);
}
// The dither of an update: a function of the step, the descriptor's index in its table, the block and the place in
// the block, so it depends on no launch shape and repeats when a step is repeated.
__device__ __forceinline__ uint32_t dither_key(int step, int index, int64_t block) {
    uint32_t k = mix32(static_cast<uint32_t>(step) * 0x632BE5ABu + static_cast<uint32_t>(index) * 0x9E3779B1u + 0x2545F491u);
    k = mix32(k ^ static_cast<uint32_t>(block));
    return mix32(k ^ static_cast<uint32_t>(static_cast<uint64_t>(block) >> 32));
}
__device__ __forceinline__ uint32_t dither_bits(uint32_t key, int place) {
    return mix32(key + static_cast<uint32_t>(place) * 0x9E3779B1u);
}

}  // namespace elx
