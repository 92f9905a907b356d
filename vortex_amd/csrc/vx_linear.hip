// Matrix product in 8-bit integers with a scale for each token (row of x) and each channel (row of w):
//   q[m,k] = rint(127 x[m,k] / amax_m), s_m = amax_m / 127, amax_m = max_k |x[m,k]|
//   y[m,n] = s_m * sw_n * (sum_k q[m,k] w[n,k]) + bias_n          (the sum is exact in 32-bit integers: K <= 131072)
#include "vx_dtype.h"
#include "vx_profile.h"

// rint(127 x / amax), exactly (ties to even), for x and amax of the input type.
//  16-bit types: 127 x is exact in fp32 (11 + 7 bits) and the quotient of an (11+7)-bit by an 11-bit number, at most 127,
//  is either a tie itself or further than 2^-12 from one: the rounded fp32 quotient falls on the same side.
//  fp32: the same argument holds for fp64 (24 + 7 bits over 24 bits: at least 2^-25 from a tie, rounding 2^-47).
template <int DT>
__device__ __forceinline__ int vx_quant1(float x, float amax) {
    if (DT == VX_DTYPE_F32) return (int)rint(((double)x * 127.0) / (double)amax);
    return (int)rintf((x * 127.0f) / amax);
}

// One workgroup per row.  A row with a NaN or an infinity gets the scale NaN (and q = 0): its products are all NaN.
template <int DT>
__global__ __launch_bounds__(256) void vx_k_quant_rows(const void *__restrict__ x, int K, long long xs, int8_t *__restrict__ q,
                                                       long long qs, float *__restrict__ scale) {
    typedef typename vx_elem<DT>::type E;
    __shared__ float s_max[4];
    __shared__ int s_bad[4];
    const long long m = blockIdx.x;
    const E *row = (const E *)x + m * xs;
    float mx = 0.f;
    bool bad = false;
    for (int k = threadIdx.x; k < K; k += 256) {
        const float a = fabsf((float)row[k]);
        bad |= !(a <= 3.4028234663852886e38f);
        mx = fmaxf(mx, a);
    }
    for (int i = 32; i >= 1; i >>= 1) mx = fmaxf(mx, __shfl_xor(mx, i, VX_WAVE));
    const bool wbad = __any(bad);
    if (vx_lane() == 0) { s_max[threadIdx.x >> 6] = mx; s_bad[threadIdx.x >> 6] = wbad; }
    __syncthreads();
    mx = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    bad = s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3];
    int8_t *dst = q + m * qs;
    const bool zero = bad || mx == 0.f;
    for (int k = threadIdx.x; k < qs; k += 256) dst[k] = (zero || k >= K) ? 0 : (int8_t)vx_quant1<DT>((float)row[k], mx);
    if (threadIdx.x == 0) scale[m] = bad ? __builtin_nanf("") : mx / 127.0f;
}

static int vx_quant_launch(const void *x, int dtype, long long M, int K, long long xs, int8_t *q, long long qs, float *s, hipStream_t st) {
    vx_prof_begin(VX_PROF_QUANT, st);
    VX_DISPATCH_DTYPE(dtype, hipLaunchKernelGGL((vx_k_quant_rows<DT>), dim3((unsigned)M), dim3(256), 0, st, x, K, xs, q, qs, s));
    vx_prof_end(VX_PROF_QUANT, st);
    return hipGetLastError() == hipSuccess ? VX_OK : VX_ERR_LAUNCH;
}

extern "C" int vx_quantize_rows_i8(const void *d_x, int dtype, int64_t M, int K, int64_t x_stride, int8_t *d_q,
                                   int64_t q_stride, float *d_scale, void *stream) {
    if (!d_x || !d_q || !d_scale || M <= 0 || K <= 0 || x_stride < K || q_stride < K || !vx_dtype_ok(dtype)) return VX_ERR_INVALID_ARG;
    if (M > VX_MAX_TOKENS || K > VX_MAX_I8_DEPTH || q_stride > VX_MAX_I8_DEPTH) return VX_ERR_UNSUPPORTED;
    if (((uintptr_t)d_x & (vx_elem_size(dtype) - 1)) || ((uintptr_t)d_scale & 3)) return VX_ERR_ALIGNMENT;
    return vx_quant_launch(d_x, dtype, M, K, x_stride, d_q, q_stride, d_scale, (hipStream_t)stream);
}

// 64 x 64 outputs for each workgroup, 64 bytes of K staged at a time; a thread owns 4 x 4 outputs (4-byte dot products).
template <int DT>
__global__ __launch_bounds__(256) void vx_k_linear_i8(const int8_t *__restrict__ q, long long qs, const float *__restrict__ s,
                                                      long long M, const int8_t *__restrict__ w, long long ws,
                                                      const float *__restrict__ sw, long long N, int K,
                                                      const float *__restrict__ bias, void *__restrict__ out, long long os) {
    typedef typename vx_elem<DT>::type E;
    __shared__ int s_q[64][17], s_w[64][17];
    const long long m0 = (long long)blockIdx.y * 64, n0 = (long long)blockIdx.x * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += 64) {
        __syncthreads();
        for (int i = threadIdx.x; i < 64 * 64; i += 256) {
            const int r = i >> 6, k = i & 63;
            ((int8_t *)&s_q[r][0])[k] = (m0 + r < M && k0 + k < K) ? q[(m0 + r) * qs + k0 + k] : 0;
            ((int8_t *)&s_w[r][0])[k] = (n0 + r < N && k0 + k < K) ? w[(n0 + r) * ws + k0 + k] : 0;
        }
        __syncthreads();
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = __builtin_amdgcn_sdot4(s_q[ty + 16 * i][k], s_w[tx + 16 * j][k], acc[i][j], false);
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const long long m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (m < M && n < N) {
                float y = (float)acc[i][j] * (s[m] * sw[n]);
                if (bias) y = y + bias[n];
                ((E *)out)[m * os + n] = vx_store_cast<DT>(y);
            }
        }
}

static int vx_linear_launch(const int8_t *q, long long qs, const float *s, long long M, const int8_t *w, long long ws,
                            const float *sw, long long N, int K, const float *bias, void *out, int out_dtype, long long os,
                            hipStream_t st) {
    const dim3 grid((unsigned)((N + 63) / 64), (unsigned)((M + 63) / 64));
    vx_prof_begin(VX_PROF_LINEAR, st);
    VX_DISPATCH_DTYPE(out_dtype, hipLaunchKernelGGL((vx_k_linear_i8<DT>), grid, dim3(256), 0, st, q, qs, s, M, w, ws, sw, N, K,
                                                    bias, out, os));
    vx_prof_end(VX_PROF_LINEAR, st);
    return hipGetLastError() == hipSuccess ? VX_OK : VX_ERR_LAUNCH;
}

static int vx_linear_check(const void *a, long long as, const int8_t *w, long long ws, const float *sw, long long M,
                           long long N, int K, const float *bias, void *out, int out_dtype, long long os) {
    if (!a || !w || !sw || !out || M <= 0 || N <= 0 || K <= 0 || as < K || ws < K || os < N || !vx_dtype_ok(out_dtype)) return VX_ERR_INVALID_ARG;
    if (M > VX_MAX_LINEAR_ROWS || N > VX_MAX_LINEAR_ROWS || K > VX_MAX_I8_DEPTH) return VX_ERR_UNSUPPORTED;
    if (((uintptr_t)out & (vx_elem_size(out_dtype) - 1)) || (((uintptr_t)sw | (uintptr_t)bias) & 3)) return VX_ERR_ALIGNMENT;
    return VX_OK;
}

extern "C" size_t vx_linear_i8_workspace_bytes(int64_t M, int64_t N, int K) {
    return M <= 0 || N <= 0 || K <= 0 || M > VX_MAX_LINEAR_ROWS || N > VX_MAX_LINEAR_ROWS || K > VX_MAX_I8_DEPTH ? 0 : 256;
}

extern "C" int vx_linear_i8(const int8_t *d_q, int64_t q_stride, const float *d_scale, int64_t M, const int8_t *d_w,
                            int64_t w_stride, const float *d_w_scale, int64_t N, int K, const float *d_bias, void *d_out,
                            int out_dtype, int64_t out_stride, void *d_workspace, size_t workspace_bytes, void *stream) {
    if (!d_scale || !d_workspace) return VX_ERR_INVALID_ARG;
    const int rc = vx_linear_check(d_q, q_stride, d_w, w_stride, d_w_scale, M, N, K, d_bias, d_out, out_dtype, out_stride);
    if (rc != VX_OK) return rc;
    if (((uintptr_t)d_scale & 3) || ((uintptr_t)d_workspace & 255)) return VX_ERR_ALIGNMENT;
    if (workspace_bytes < vx_linear_i8_workspace_bytes(M, N, K)) return VX_ERR_WORKSPACE;
    return vx_linear_launch(d_q, q_stride, d_scale, M, d_w, w_stride, d_w_scale, N, K, d_bias, d_out, out_dtype, out_stride,
                            (hipStream_t)stream);
}

static size_t vx_up256(size_t n) { return (n + 255) & ~(size_t)255; }

extern "C" size_t vx_linear_w8a8_workspace_bytes(int64_t M, int64_t N, int K) {
    const size_t rest = vx_linear_i8_workspace_bytes(M, N, K);
    return rest ? rest + vx_up256((size_t)M * 4) + vx_up256((size_t)M * (size_t)K) : 0;
}

extern "C" int vx_linear_w8a8(const void *d_x, int x_dtype, int64_t x_stride, int64_t M, const int8_t *d_w, int64_t w_stride,
                              const float *d_w_scale, int64_t N, int K, const float *d_bias, void *d_out, int out_dtype,
                              int64_t out_stride, void *d_workspace, size_t workspace_bytes, void *stream) {
    if (!d_workspace || !vx_dtype_ok(x_dtype)) return VX_ERR_INVALID_ARG;
    int rc = vx_linear_check(d_x, x_stride, d_w, w_stride, d_w_scale, M, N, K, d_bias, d_out, out_dtype, out_stride);
    if (rc != VX_OK) return rc;
    if (((uintptr_t)d_x & (vx_elem_size(x_dtype) - 1)) || ((uintptr_t)d_workspace & 255)) return VX_ERR_ALIGNMENT;
    if (workspace_bytes < vx_linear_w8a8_workspace_bytes(M, N, K)) return VX_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    float *s = (float *)d_workspace;
    int8_t *q = (int8_t *)d_workspace + vx_up256((size_t)M * 4);
    rc = vx_quant_launch(d_x, x_dtype, M, K, x_stride, q, K, s, st);
    if (rc != VX_OK) return rc;
    return vx_linear_launch(q, K, s, M, d_w, w_stride, d_w_scale, N, K, d_bias, d_out, out_dtype, out_stride, st);
}
