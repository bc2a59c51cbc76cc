// tt_wave.h -- device helpers shared by the attention kernels: constants, lane
// reductions, matrix-core types and conversions.
#pragma once
#include "tt_common.h"

namespace tt {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_huge_valf();

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, false));
}

// Sum over the 16 lanes of a DPP row. Butterfly pairs (xor 1, xor 2, then the
// half-row and row mirrors, which pair equal-valued quads / octets) so every
// lane of the row ends with the bit-identical total.
__device__ __forceinline__ float row_sum16(float x) {
    x = x + dpp<0xB1>(x);   // quad_perm [1,0,3,2]
    x = x + dpp<0x4E>(x);   // quad_perm [2,3,0,1]
    x = x + dpp<0x141>(x);  // row_half_mirror
    x = x + dpp<0x140>(x);  // row_mirror
    return x;
}

// A wave-uniform value as a scalar. Counts that come from the engine's device
// state or from the kernel arguments would otherwise be read with one vector
// load whose address is selected, a round trip before a workgroup knows its
// share of the work. (With the tier pointers of tt_attn.hip: partials of 32/8 heads at
// 32k 15.0 -> 14.2 us, at 4k 7.5 -> 7.3, head_dim 64 at 32k 11.7 -> 11.3; an
// engine step of four layers at 4k 69.0 -> 66.4.)
__device__ __forceinline__ int scalar(const int x) { return __builtin_amdgcn_readfirstlane(x); }

// A pointer into global memory whose origin does not tell (an integer, or read
// from memory): without the address space in its type the accesses become flat
// ones, which LDS waits include.
template <typename T>
__device__ __forceinline__ T* global_ptr(const uint64_t a) {
    typedef __attribute__((address_space(1))) T* gptr;
    return (T*)reinterpret_cast<gptr>(a);
}
template <typename T>
__device__ __forceinline__ T* global_ptr(T* p) {
    return global_ptr<T>(reinterpret_cast<uint64_t>(p));
}
typedef _Float16 mf_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 mf_h2 __attribute__((ext_vector_type(2)));
typedef float mf_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t mf_u4 __attribute__((ext_vector_type(4)));


// max(a, b) for operands that are never NaN: one v_max_f32, without the
// quieting of the operands that fmaxf adds for values it cannot see the origin of.
__device__ __forceinline__ float fmax_nn(float a, float b) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
// max(|a|, |b|), likewise
__device__ __forceinline__ float fmax_abs_nn(float a, float b) {
    float r;
    asm("v_max_f32_e64 %0, |%1|, |%2|" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// Reductions over the four 16-lane rows of a wave (lanes n, n+16, n+32, n+48).
__device__ __forceinline__ float xrow_max(float x) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmax_nn(__uint_as_float(s[0]), __uint_as_float(s[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmax_nn(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float xrow_sum(float x) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}

// Orders this wave's LDS writes before its later LDS reads of other lanes'
// data (LDS instructions of one wave execute in issue order).
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ mf_f4 mfma16x16x32(mf_u4 a, mf_u4 b, mf_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(mf_h8, a), __builtin_bit_cast(mf_h8, b), c, 0,
                                                  0, 0);
}

// x - m * f16 (low / high half of h), one v_fma_mix_f32 (exact for m = 1
// and h a rounding of x: the difference fits in f32).
__device__ __forceinline__ float fma_mix_lo(uint32_t h, float negm, float x) {
    float r;
    asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(negm), "v"(x));
    return r;
}
__device__ __forceinline__ float fma_mix_hi(uint32_t h, float negm, float x) {
    float r;
    asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(negm), "v"(x));
    return r;
}

}  // namespace
}  // namespace tt
