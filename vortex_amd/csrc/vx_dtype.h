// Element types of the token-model operators (vx_embed.hip, vx_linear.hip, vx_verify.hip) and their conversions.
// Arithmetic is fp32 (or wider); a value is rounded to its 16-bit type once, to nearest even, when it is stored.
#pragma once
#include "vx_common.h"

template <int DT> struct vx_elem;
template <> struct vx_elem<VX_DTYPE_F32>  { typedef float type; };
template <> struct vx_elem<VX_DTYPE_F16>  { typedef _Float16 type; };
template <> struct vx_elem<VX_DTYPE_BF16> { typedef __bf16 type; };

__host__ __device__ __forceinline__ int vx_elem_size(int dtype) { return dtype == VX_DTYPE_F32 ? 4 : 2; }
static inline bool vx_dtype_ok(int dtype) { return dtype == VX_DTYPE_F32 || dtype == VX_DTYPE_F16 || dtype == VX_DTYPE_BF16; }

// Calls BODY with `constexpr int DT` = dtype (already checked).
#define VX_DISPATCH_DTYPE(dtype, ...)                                          \
    do {                                                                       \
        if ((dtype) == VX_DTYPE_F32) { constexpr int DT = VX_DTYPE_F32; __VA_ARGS__; }        \
        else if ((dtype) == VX_DTYPE_F16) { constexpr int DT = VX_DTYPE_F16; __VA_ARGS__; }   \
        else { constexpr int DT = VX_DTYPE_BF16; __VA_ARGS__; }                \
    } while (0)

// fp32 -> the stored type, to nearest even.  The empty asm keeps the fp32 value as computed: hipcc otherwise folds a product
// and its conversion to fp16 into one instruction that skips the fp32 rounding, and the same operator would then round
// differently in its three types.
template <int DT>
__device__ __forceinline__ typename vx_elem<DT>::type vx_store_cast(float y) {
    if (DT == VX_DTYPE_F16) asm("" : "+v"(y));
    return (typename vx_elem<DT>::type)y;
}
