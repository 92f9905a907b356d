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

// A launch of `blocks` workgroups and the number of one.  HIP takes fewer than 2^32 threads along an axis, and drops the others
// without an error: beyond 2^21 workgroups (of up to 1024 threads) they are laid out along two axes, in the same order.  The last
// of the second axis may be numbers from `blocks` on: the kernels have nothing to do there.
static inline dim3 vx_grid(int64_t blocks) {
    const int64_t y = (blocks + (1 << 21) - 1) >> 21;
    return dim3((unsigned)((blocks + y - 1) / y), (unsigned)y);
}
__device__ __forceinline__ unsigned vx_block() { return blockIdx.y * gridDim.x + blockIdx.x; }

// fp32 -> the stored type, to nearest even.  The empty asm keeps the fp32 value as computed: hipcc otherwise folds a product
// and its conversion to fp16 into one instruction that skips the fp32 rounding, and the same operator would then round
// differently in its three types.
template <int DT>
__device__ __forceinline__ typename vx_elem<DT>::type vx_store_cast(float y) {
    if (DT == VX_DTYPE_F16) asm("" : "+v"(y));
    return (typename vx_elem<DT>::type)y;
}

// 16 bytes of a row: VEC = 16 / sizeof(element) values.  Rows start at any multiple of the element (odd widths, slices), so
// the access is declared with the element's alignment only: gfx950 loads and stores 16 bytes at any address.
template <int DT>
union vx_vec {
    vx_v4 raw;
    typename vx_elem<DT>::type e[16 / sizeof(typename vx_elem<DT>::type)];
};
typedef float vx_v2 __attribute__((ext_vector_type(2)));
typedef float vx_v2_at2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float vx_v4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float vx_v4_at4 __attribute__((ext_vector_type(4), aligned(4)));
template <int DT>
__device__ __forceinline__ vx_v4 vx_load16(const typename vx_elem<DT>::type *p) {
    return DT == VX_DTYPE_F32 ? (vx_v4)*(const vx_v4_at4 *)p : (vx_v4)*(const vx_v4_at2 *)p;
}

// VEC values at p, `left` of them inside the row (none for left <= 0): the others are 0 and not read.
template <int DT>
__device__ __forceinline__ vx_vec<DT> vx_load_vec(const typename vx_elem<DT>::type *p, int left) {
    constexpr int VEC = 16 / sizeof(typename vx_elem<DT>::type);
    vx_vec<DT> v;
    v.raw = vx_v4{0.f, 0.f, 0.f, 0.f};
    if (left >= VEC) {
        v.raw = vx_load16<DT>(p);
    } else {
#pragma unroll
        for (int k = 0; k < VEC - 1; ++k)
            if (k < left) v.e[k] = p[k];
    }
    return v;
}

// A lane's VEC columns [c, c + VEC) of a row of D: where they stick out of the row, the lane works on the row's last VEC
// columns instead (`at`), so that every load is one unconditional 16-byte load, and stores only columns from c on.
// TINY: the row itself is shorter than VEC.
template <int DT>
struct vx_cols {
    static constexpr int VEC = 16 / sizeof(typename vx_elem<DT>::type);
    int c, at;
    __device__ __forceinline__ vx_cols(int c_, int D) : c(c_), at(c_ <= D - VEC ? c_ : (D > VEC ? D - VEC : 0)) {}
    // values of the row at its columns `at`
    template <bool TINY>
    __device__ __forceinline__ vx_vec<DT> load(const typename vx_elem<DT>::type *row, int D) const {
        vx_vec<DT> v;
        if (!TINY) {
            v.raw = vx_load16<DT>(row + at);
        } else {
            v.raw = vx_v4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < VEC - 1; ++k)
                if (k < D) v.e[k] = row[k];
        }
        return v;
    }
    // NT: past the caches (see vx_past_caches)
    template <bool NT = false>
    __device__ __forceinline__ void store(typename vx_elem<DT>::type *row, const float *f, int D) const {
        vx_vec<DT> v;
#pragma unroll
        for (int k = 0; k < VEC; ++k) v.e[k] = vx_store_cast<DT>(f[k]);
        if (c == at && c + VEC <= D) {
            if (NT) __builtin_nontemporal_store(v.raw, (vx_v4 *)(row + c));
            else if (DT == VX_DTYPE_F32) *(vx_v4_at4 *)(row + c) = v.raw;
            else *(vx_v4_at2 *)(row + c) = v.raw;
        } else if (c < D) {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (at + k >= c && at + k < D) row[at + k] = v.e[k];
        }
    }
};

// Whether a result of `rows` rows of D values is written past the caches: more than the 32 MB of the chip's L2, so that none
// of it would stay there, and rows of whole 128-byte lines.  Measured (ordinary / past the caches): lookup of 32768 x 4096 bf16
// 73 / 63 us, every row of a gradient of 131072 x 4096 bf16 385 / 366; rows of 2000 bytes 37 / 44.  (A pure fill is faster by
// ordinary stores.)
static inline bool vx_past_caches(const void *out, int64_t rows, int D, int dtype) {
    const int64_t row = (int64_t)D * vx_elem_size(dtype);
    return rows * row > (32 << 20) && row % 128 == 0 && ((uintptr_t)out & 127) == 0;
}
