// 16-bit operands of the two attention kernels over pages.
#pragma once
#include "common.cuh"
#include "tc_common.cuh"

namespace hf2q {
namespace paged {

// one of two bf16 numbers is infinite or NaN
__device__ __forceinline__ bool holds_nonfinite(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }

// A power of two above |v| (v finite) and at most twice that, between 2^-100 and 2^100 so that what it divides and what divides it are numbers.
__device__ __forceinline__ float unit_above(float v) {
    return fminf(fmaxf(__uint_as_float((__float_as_uint(v) & 0x7f800000u) + 0x00800000u), 0x1p-100f), 0x1p100f);
}

// two numbers in the type that the products over a cache of codes (f16) or of bf16 take
template <bool CODES> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (CODES) return tc::pack_h2(a, b);
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace paged
}  // namespace hf2q
