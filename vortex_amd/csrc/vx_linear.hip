// Matrix product in 8-bit integers with a scale for each token (row of x) and each channel (row of w):
//   q[m,k] = rint(127 x[m,k] / amax_m), s_m = amax_m / 127, amax_m = max_k |x[m,k]|
//   y[m,n] = s_m * sw_n * (sum_k q[m,k] w[n,k]) + bias_n          (the sum is exact in 32-bit integers: K <= 131072)
#include "vx_dtype.h"
#include "vx_profile.h"
#include <type_traits>

// rint(127 x / top), exactly, ties to even: with n = floor of the quotient (one below or above it by rounding does no harm) it is
// n or n + 1 by 127 |x| against (n + 1/2) top.  Each product is taken as its rounded value and what the rounding left (a fma);
// where the two are close, their difference and that of the rests are exact.  Rows near the ends of the range are scaled first.
__device__ __forceinline__ unsigned vx_quant_exact(float x, float top) {
    const float up = top < 1e-30f ? 0x1p64f : (top > 1e30f ? 0x1p-64f : 1.f), xs = fabsf(x) * up, ts = top * up;
    const float n = floorf(xs * (127.0f / ts)), a = xs * 127.0f, b = (n + 0.5f) * ts;
    const float d = (a - b) + (__builtin_fmaf(xs, 127.0f, -a) - __builtin_fmaf(n + 0.5f, ts, -b));
    const int i = (int)n, v = i + (d > 0.f || (d == 0.f && (i & 1)) ? 1 : 0);
    return (unsigned)(x < 0.f ? -v : v);
}

// What a row's largest |x| says: q = rint(x r), s = scale.  |x| is compared by its bits: they order as the values do, with
// infinity and NaN above all.  A row that holds one gets the scale NaN (and q = 0): its products are all NaN.
struct vx_quant_row {
    float top, r;                                                 // 127 / top
    bool bad, zero, tiny;
    __device__ __forceinline__ explicit vx_quant_row(unsigned bits) {
        bad = bits >= 0x7f800000u;
        zero = bad || bits == 0;
        top = __uint_as_float(bits);
        r = zero ? 0.f : 127.0f / top;
        tiny = !zero && !(r <= 3.4028234663852886e38f);
    }
    __device__ __forceinline__ float scale() const { return bad ? __builtin_nanf("") : top / 127.0f; }
};
template <int DT>
__device__ __forceinline__ unsigned vx_quant_look(const vx_vec<DT> &a, unsigned top) {
#pragma unroll
    for (int k = 0; k < 16 / (int)sizeof(typename vx_elem<DT>::type); ++k) top = max(top, __float_as_uint((float)a.e[k]) & 0x7fffffffu);
    return top;
}
// largest value of the wave, in a scalar register: by rows of 16 lanes (1, 2, 4, 8 lanes up), then row to row and half to half
__device__ __forceinline__ unsigned vx_wave_max(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
    return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
template <int DT>
struct vx_quant_out {
    unsigned w[4 / sizeof(typename vx_elem<DT>::type)];           // four integers each
};
// The quotient is a product with r; added to 1.5 * 2^23 it is rounded to an integer, in the sum's low byte.
//  fp32: r is off by at most half a step, the product (in the fma) by 127 * 2^-24 < 7.6e-6; where that could change the integer
//  (closer than 1e-5 to a tie) the exact way is taken.
//  16-bit types: ties are frequent (rows whose largest value has a short mantissa), but other quotients are at least 2^-19 of
//  their size away from one: |254 x - odd top| is a whole number over 254 |x| < 2^19, in units of x's last bit.  The product is
//  within two steps of fp32 of the quotient; rounded to a multiple of 8 of them (2^-20) it is the tie if there is one, and
//  otherwise stays on its side.
// r overflows for a largest value below 127 / FLT_MAX: such rows go the exact way throughout.
template <int DT>
__device__ __forceinline__ vx_quant_out<DT> vx_quant_piece(const vx_vec<DT> &a, const vx_quant_row &row) {
    constexpr int VEC = 16 / sizeof(typename vx_elem<DT>::type);
    constexpr float SHIFT = 12582912.f;
    vx_quant_out<DT> o;
    unsigned t[VEC];
    bool exact = row.tiny;
    if (DT == VX_DTYPE_F32) {
        float off = 0.f;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const float x = (float)a.e[k], sum = __builtin_fmaf(x, row.r, SHIFT);
            off = fmaxf(off, fabsf(__builtin_fmaf(x, row.r, SHIFT - sum)));
            t[k] = __float_as_uint(sum);
        }
        exact |= off > 0.49999f;
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            t[k] = __float_as_uint(__uint_as_float((__float_as_uint((float)a.e[k] * row.r) + 4u) & ~7u) + SHIFT);
    }
    if (exact) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) t[k] = vx_quant_exact((float)a.e[k], row.top);
    }
#pragma unroll
    for (int k = 0; k < VEC / 4; ++k)
        o.w[k] = row.zero ? 0u : __builtin_amdgcn_perm(t[4 * k + 1], t[4 * k], 0x0c0c0400u) | __builtin_amdgcn_perm(t[4 * k + 3], t[4 * k + 2], 0x04000c0cu);
    return o;
}

// WAVES waves per row, U 16-byte pieces of it in the registers of each lane between the two passes (maximum, quotients);
// longer rows are read again.
template <int DT, int WAVES, int U>
__global__ __launch_bounds__(256) void vx_k_quant_rows(const void *__restrict__ x, long long M, int K, long long xs,
                                                       int8_t *__restrict__ q, long long qs, float *__restrict__ scale) {
    typedef typename vx_elem<DT>::type E;
    constexpr int VEC = 16 / sizeof(E), THREADS = WAVES * 64;
    __shared__ unsigned s_max[4];
    const int w = threadIdx.x >> 6, tid = WAVES == 1 ? vx_lane() : (int)threadIdx.x;
    const long long m = WAVES == 1 ? (long long)vx_block() * 4 + w : (long long)vx_block();
    if (m >= M) return;                                           // WAVES == 1 has no barrier behind this
    const E *row = (const E *)x + m * xs;
    unsigned top = 0;
    vx_vec<DT> v[U];
    const bool once = K <= THREADS * VEC * U;
    auto look = [&](const vx_vec<DT> &a) { top = vx_quant_look<DT>(a, top); };
    if (once) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = vx_load_vec<DT>(row + (u * THREADS + tid) * VEC, K - (u * THREADS + tid) * VEC);
#pragma unroll
        for (int u = 0; u < U; ++u) look(v[u]);
    } else {
        for (int c = tid * VEC; c < K; c += THREADS * VEC) look(vx_load_vec<DT>(row + c, K - c));
    }
    top = vx_wave_max(top);
    if (WAVES > 1) {
        if (vx_lane() == 0) s_max[w] = top;
        __syncthreads();
        top = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
    }
    const vx_quant_row what(top);
    int8_t *dst = q + m * qs;
    auto put = [&](const vx_vec<DT> &a, int c) {
        const vx_quant_out<DT> o = vx_quant_piece<DT>(a, what);
        if (c + VEC <= qs) {                                      // columns K .. qs - 1 come out as 0
            typedef unsigned u32_at1 __attribute__((aligned(1)));
#pragma unroll
            for (int k = 0; k < VEC / 4; ++k) *(u32_at1 *)(dst + c + 4 * k) = o.w[k];
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (c + k < qs) dst[c + k] = (int8_t)(o.w[k / 4] >> (k % 4 * 8));
        }
    };
    if (once) {
#pragma unroll
        for (int u = 0; u < U; ++u) put(v[u], (u * THREADS + tid) * VEC);
    }
    for (long long c = (once ? THREADS * VEC * U : 0) + tid * VEC; c < qs; c += THREADS * VEC)
        put(vx_load_vec<DT>(row + c, K - (int)c), (int)c);
    if (tid == 0) scale[m] = what.scale();
}

static int vx_quant_launch(const void *x, int dtype, long long M, int K, long long xs, int8_t *q, long long qs, float *s, hipStream_t st) {
    vx_prof_begin(VX_PROF_QUANT, st);
    // a row that one wave holds needs no barrier; with few rows four waves share one
    VX_DISPATCH_DTYPE(dtype, {
        constexpr int PIECE = 64 * 16 / (int)sizeof(typename vx_elem<DT>::type);
        if (K <= 4 * PIECE && M >= 256)
            hipLaunchKernelGGL((vx_k_quant_rows<DT, 1, 4>), vx_grid((M + 3) / 4), dim3(256), 0, st, x, M, K, xs, q, qs, s);
        else if (K <= 8 * PIECE && M >= 256)
            hipLaunchKernelGGL((vx_k_quant_rows<DT, 1, 8>), vx_grid((M + 3) / 4), dim3(256), 0, st, x, M, K, xs, q, qs, s);
        else
            hipLaunchKernelGGL((vx_k_quant_rows<DT, 4, 4>), vx_grid(M), dim3(256), 0, st, x, M, K, xs, q, qs, s);
    });
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

typedef int vx_i4 __attribute__((ext_vector_type(4)));
typedef int vx_i16 __attribute__((ext_vector_type(16)));
typedef vx_i4 vx_i4_at1 __attribute__((aligned(1)));

// y for one output; the same expression in every kernel, so that all variants give the same bits
__device__ __forceinline__ float vx_linear_out(int acc, float s, float sw, bool has_bias, float bias) {
    const float y = (float)acc * (s * sw);
    return has_bias ? y + bias : y;
}

// ---- few tokens: the weights stream once from memory into registers, no LDS between.
// One workgroup per 16 NT channels, its waves share K; mfma 16x16x64 with the weights as rows: lane l holds 16 bytes of
// channel l % 16 at k = 64 b + 16 (l / 16), and MT tiles of 16 tokens stand against them.  Bound by the read of the weights:
// 131 MB in 25 us (5.3 TB/s) for one token against 32000 x 4096.  (Times in this file, where nothing else is said: a call in a
// graph of calls, each with weights of its own, 600 MB of them in turn; the median of 9 replays.)
__device__ __forceinline__ vx_i4 vx_i8_tail(const int8_t *row, int k, int K) {      // bytes k .. k+15, 0 from K on
    union { vx_i4 v; int8_t b[16]; } o;
    o.v = vx_i4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (k + i < K) o.b[i] = row[k + i];
    return o.v;
}

template <int DT, int MT, int NT>
__global__ __launch_bounds__(1024) void vx_k_linear_stream(const int8_t *__restrict__ q, long long qs, const float *__restrict__ s,
                                                          long long M, const int8_t *__restrict__ w, long long ws,
                                                          const float *__restrict__ sw, long long N, int K,
                                                          const float *__restrict__ bias, void *__restrict__ out, long long os) {
    typedef typename vx_elem<DT>::type E;
    constexpr int UN = MT * NT == 1 ? 8 : (MT + NT <= 4 ? 4 : 2);
    extern __shared__ int s_part[];                               // [waves][MT][16 tokens][16 NT channels]
    const int lane = vx_lane(), wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const long long n0 = (long long)blockIdx.x * 16 * NT, m0 = (long long)blockIdx.y * 16 * MT;
    const int8_t *wrow[NT], *qrow[MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) wrow[i] = w + min(n0 + i * 16 + (lane & 15), N - 1) * ws;
#pragma unroll
    for (int t = 0; t < MT; ++t) qrow[t] = q + min(m0 + t * 16 + (lane & 15), M - 1) * qs;
    vx_i4 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[i][t] = vx_i4{0, 0, 0, 0};
    const int blocks = (K + 63) >> 6, per = (blocks + waves - 1) / waves, full = K >> 6;
    int b = min(blocks, wave * per);
    const int end = min(blocks, b + per), end_full = min(end, full);
    const int koff = (lane >> 4) * 16;
    auto run = [&](auto un) {
        constexpr int N_ = decltype(un)::value;
        vx_i4 a[N_][NT], x[N_][MT];
#pragma unroll
        for (int u = 0; u < N_; ++u) {
#pragma unroll
            for (int i = 0; i < NT; ++i) a[u][i] = *(const vx_i4_at1 *)(wrow[i] + (b + u) * 64 + koff);
        }
#pragma unroll
        for (int u = 0; u < N_; ++u) {
#pragma unroll
            for (int t = 0; t < MT; ++t) x[u][t] = *(const vx_i4_at1 *)(qrow[t] + (b + u) * 64 + koff);
        }
#pragma unroll
        for (int u = 0; u < N_; ++u)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[i][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u][i], x[u][t], acc[i][t], 0, 0, 0);
        b += N_;
    };
    while (b + UN <= end_full) run(std::integral_constant<int, UN>());
    if (UN > 4 && b + 4 <= end_full) run(std::integral_constant<int, 4>());
    if (UN > 2 && b + 2 <= end_full) run(std::integral_constant<int, 2>());
    if (b < end_full) run(std::integral_constant<int, 1>());
    if (b < end) {
        // The last 64 bytes stick out of the rows.  The tokens' bytes from K on are made 0, so the channels' may be anything
        // that lies inside the matrix: only its last rows are read byte by byte.
        const int k = b * 64 + koff;
        vx_i4 a[NT], x[MT];
#pragma unroll
        for (int i = 0; i < NT; ++i)
            a[i] = wrow[i] + k + 16 <= w + (N - 1) * ws + K ? (vx_i4)*(const vx_i4_at1 *)(wrow[i] + k) : vx_i8_tail(wrow[i], k, K);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            x[t] = qrow[t] + k + 16 <= q + (M - 1) * qs + K ? (vx_i4)*(const vx_i4_at1 *)(qrow[t] + k) : vx_i8_tail(qrow[t], k, K);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int left = K - k - 4 * i;                   // bytes of this word inside the row
                x[t][i] = left >= 4 ? x[t][i] : (left <= 0 ? 0 : x[t][i] & (int)(0xffffffffu >> (32 - 8 * left)));
            }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[i][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i], x[t], acc[i][t], 0, 0, 0);
    }
    // lane l holds token l % 16, channels 4 (l / 16) .. + 3 of each tile
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t)
            *(vx_i4 *)&s_part[((wave * MT + t) * 16 + (lane & 15)) * 16 * NT + i * 16 + (lane >> 4) * 4] = acc[i][t];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * NT * 256; i += blockDim.x) {
        int sum = 0;
        for (int k = 0; k < waves; ++k) sum += s_part[k * MT * NT * 256 + i];
        const long long m = m0 + i / (16 * NT), n = n0 + i % (16 * NT);
        if (m < M && n < N) ((E *)out)[m * os + n] = vx_store_cast<DT>(vx_linear_out(sum, s[m], sw[n], bias != nullptr, bias ? bias[n] : 0.f));
    }
}

// The same for one token that is quantised on the way: every workgroup does it for itself, in LDS, while its first weights are
// coming, and then takes several tiles of 16 channels.  The loads of a tile's first weights are on their way while the waves
// join the sums of the tile before.  32000 x 4096: 131 MB, 26 us for the whole call, against 29 in two
// launches.
template <int DT>
__global__ __launch_bounds__(1024) void vx_k_linear_one(const void *__restrict__ x, const int8_t *__restrict__ w, long long ws,
                                                        const float *__restrict__ sw, long long N, int K, const float *__restrict__ bias,
                                                        void *__restrict__ out, int out_dtype, int tiles) {
    typedef typename vx_elem<DT>::type E;
    constexpr int VEC = 16 / sizeof(E), UN = 8;
    extern __shared__ __attribute__((aligned(16))) int8_t s_one[];    // q: K rounded up to 64; sums: 2 x [waves][16 channels]
    __shared__ unsigned s_top[16];
    const int lane = vx_lane(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int k64 = (K + 63) & ~63, koff = (lane >> 4) * 16;
    int *s_sum = (int *)(s_one + k64);
    const int blocks = k64 >> 6, per = (blocks + waves - 1) / waves, full = K >> 6;
    const int b0 = min(blocks, wave * per), end = min(blocks, b0 + per), end_full = min(end, full);
    auto row_of = [&](int tile) { return w + min((long long)tile * 16 + (lane & 15), N - 1) * ws + koff; };
    auto load = [](const int8_t *row, int at) { return (vx_i4)*(const vx_i4_at1 *)(row + at * 64); };
    const int8_t *wrow = row_of(blockIdx.x);
    vx_i4 a[UN];
    const bool ahead = b0 + UN <= end_full;
    if (ahead) {
#pragma unroll
        for (int u = 0; u < UN; ++u) a[u] = load(wrow, b0 + u);
    }
    const E *row = (const E *)x;
    unsigned top = 0;
    for (int c = threadIdx.x * VEC; c < K; c += blockDim.x * VEC) top = vx_quant_look<DT>(vx_load_vec<DT>(row + c, K - c), top);
    top = vx_wave_max(top);
    if (lane == 0) s_top[wave] = top;
    __syncthreads();
    for (int i = 0; i < waves; ++i) top = max(top, s_top[i]);
    const vx_quant_row what(top);
    for (int c = threadIdx.x * VEC; c < k64; c += blockDim.x * VEC) {
        const vx_quant_out<DT> o = vx_quant_piece<DT>(vx_load_vec<DT>(row + c, K - c), what);
#pragma unroll
        for (int k = 0; k < VEC / 4; ++k) *(unsigned *)(s_one + c + 4 * k) = o.w[k];
    }
    __syncthreads();
    const int8_t *q = s_one + koff;                               // all 16 columns of the matrix instruction are this token
    for (int tile = blockIdx.x, buf = 0; tile < tiles; tile += gridDim.x, buf ^= 1) {
        const int8_t *next = row_of(min(tile + (int)gridDim.x, tiles - 1));
        vx_i4 acc[2] = {};
        auto multiply = [&](const vx_i4 &weights, int at, int i) {
            acc[i & 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(weights, *(const vx_i4 *)(q + at * 64), acc[i & 1], 0, 0, 0);
        };
        int b = b0;
        if (ahead) {
            for (; b + 2 * UN <= end_full; b += UN) {
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    multiply(a[u], b + u, u);
                    a[u] = load(wrow, b + UN + u);
                }
            }
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                multiply(a[u], b + u, u);
                if (tile + (int)gridDim.x < tiles) a[u] = load(next, b0 + u);
            }
            b += UN;
        }
        for (; b + 4 <= end_full; b += 4) {
            vx_i4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = load(wrow, b + u);
#pragma unroll
            for (int u = 0; u < 4; ++u) multiply(v[u], b + u, u);
        }
        for (; b < end_full; ++b) multiply(load(wrow, b), b, 0);
        if (b < end) {                                            // weights from K on meet zeros; those outside the matrix are not read
            const int k = b * 64;
            multiply(wrow + k + 16 <= w + (N - 1) * ws + K ? load(wrow, b) : vx_i8_tail(wrow, k, K - koff), b, 0);
        }
        int *sums = s_sum + buf * waves * 16;
        if ((lane & 15) == 0) *(vx_i4 *)&sums[wave * 16 + (lane >> 4) * 4] = acc[0] + acc[1];
        __syncthreads();
        const long long n = (long long)tile * 16 + threadIdx.x;
        if (threadIdx.x < 16 && n < N) {
            int sum = 0;
            for (int i = 0; i < waves; ++i) sum += sums[i * 16 + threadIdx.x];
            const float y = vx_linear_out(sum, what.scale(), sw[n], bias != nullptr, bias ? bias[n] : 0.f);
            if (out_dtype == VX_DTYPE_F32) ((float *)out)[n] = y;
            else if (out_dtype == VX_DTYPE_F16) ((_Float16 *)out)[n] = vx_store_cast<VX_DTYPE_F16>(y);
            else ((__bf16 *)out)[n] = vx_store_cast<VX_DTYPE_BF16>(y);
        }
        wrow = next;
    }
}

// Which single tokens go this way (us, this / quantise and stream; bf16): 1000 x 512 3.7/6.7, 4096 x 4096 7.7/10.1,
// 8192 x 8192 17/20, 32000 x 1024 10/13, 32000 x 4096 26/29; beyond two tiles a workgroup the next kernel is faster (this / the
// next: 50021 x 1000 17/14, 50021 x 4000 49/40, 65536 x 512 13/11; 32000 x 4096 26/27).
#define VX_ONE_MAX_N 32768
#define VX_ONE_MAX_K 32768
static bool vx_linear_by_one(int64_t M, int64_t N, int K) { return M == 1 && N <= VX_ONE_MAX_N && K <= VX_ONE_MAX_K; }

static int vx_linear_one_launch(const void *x, int dtype, const int8_t *w, long long ws, const float *sw, long long N, int K,
                                const float *bias, void *out, int out_dtype, hipStream_t st) {
    vx_prof_begin(VX_PROF_LINEAR, st);
    const int waves = N <= 4096 ? 16 : 4;                         // few channels: more waves side by side along K
    // up to four workgroups a compute unit, with equally many tiles (512 / 1280 / 2048 of them: 28 / 26 / 28 instead of 26 us)
    const int tiles = (int)((N + 15) / 16), each = (tiles + 1023) / 1024;
    const dim3 grid((unsigned)((tiles + each - 1) / each));
    const size_t lds = (size_t)((K + 63) & ~63) + (size_t)2 * waves * 64;
    VX_DISPATCH_DTYPE(dtype, {
        hipLaunchKernelGGL((vx_k_linear_one<DT>), grid, dim3(waves * 64), lds, st, x, w, ws, sw, N, K, bias, out, out_dtype, tiles);
    });
    vx_prof_end(VX_PROF_LINEAR, st);
    return hipGetLastError() == hipSuccess ? VX_OK : VX_ERR_LAUNCH;
}

// four results next to each other, `left` of them inside the row
template <int OT>
__device__ __forceinline__ void vx_store4(void *out, long long at, const float y[4], long long left) {
    typedef typename vx_elem<OT>::type O;
    O *to = (O *)out + at;
    union { O e[4]; vx_v2 v2; vx_v4 v4; } o;
#pragma unroll
    for (int k = 0; k < 4; ++k) o.e[k] = vx_store_cast<OT>(y[k]);
    if (left >= 4) {
        if (sizeof(O) == 2) *(vx_v2_at2 *)to = o.v2;
        else *(vx_v4_at4 *)to = o.v4;
    } else {
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (k < left) to[k] = o.e[k];
    }
}

// ---- few tokens, in LDS: one persistent workgroup of 16 waves a compute unit holds them all (quantised on the way, or copied) and
// its waves take tiles of 16 channels, the first weights of each on their way since the tile before.  With fewer than 16 tiles
// a compute unit 2 to 16 waves share a tile's K and join their sums in LDS.  Rows in LDS are an odd number of 16-byte pieces
// long: 16 of them lie in all banks.  Bound by the read of the weights and, with more tokens, of LDS:
// 37 x 50021 x 1000 bf16 in 21 us of the whole call (54 MB), where quantising to memory first takes 24.
#define VX_SRC_I8 3                                               // the tokens come quantised, with their scales
template <int SRC, int MT, int UN>
__global__ __launch_bounds__(1024) void vx_k_linear_few(const void *__restrict__ x, long long xs, const float *__restrict__ s, int M,
                                                        const int8_t *__restrict__ w, long long ws, const float *__restrict__ sw,
                                                        long long N, int K, const float *__restrict__ bias, void *__restrict__ out,
                                                        int out_dtype, long long os, int tiles, int ks_log2) {
    extern __shared__ __attribute__((aligned(16))) int8_t s_few[];    // q: [M][K rounded up to 64, + 16]; sums: [16 waves][MT][256] if waves share K
    __shared__ float s_scale[16 * MT];
    __shared__ unsigned s_top[16];
    const int lane = vx_lane(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), KS = 1 << ks_log2, CT = 16 >> ks_log2;
    const int ct = wave >> ks_log2, ks = wave & (KS - 1), grid = gridDim.x;
    const int slot = grid == 256 ? (blockIdx.x & 7) * 32 + (blockIdx.x >> 3) : blockIdx.x;
    const int k64 = (K + 63) & ~63, pitch = k64 + 16, koff = (lane >> 4) * 16;
    const int blocks = k64 >> 6, per = (blocks + KS - 1) >> ks_log2, full = K >> 6;
    const int b0 = min(blocks, ks * per), end = min(blocks, b0 + per), end_full = min(end, full);
    auto row_of = [&](int tile) { return w + min((long long)tile * 16 + (lane & 15), N - 1) * ws + koff; };
    auto load = [](const int8_t *row, int at) { return (vx_i4)*(const vx_i4_at1 *)(row + at * 64); };
    // columns c, c + step, .. of token m
    auto quantise = [&](const auto *row, int m, int c, int step, const vx_quant_row &what) {
        if constexpr (SRC != VX_SRC_I8) {
            constexpr int VEC = 16 / sizeof(*row);
            if (c == lane * VEC && lane == 0) s_scale[m] = what.scale();
            auto put = [&](const vx_vec<SRC> &v, int c) {
                const vx_quant_out<SRC> o = vx_quant_piece<SRC>(v, what);
#pragma unroll
                for (int k = 0; k < VEC / 4; ++k) *(unsigned *)(s_few + m * pitch + c + 4 * k) = o.w[k];
            };
#pragma unroll 4
            for (; c - lane * VEC + 64 * VEC <= K; c += step) {
                vx_vec<SRC> v;
                v.raw = vx_load16<SRC>(row + c);
                put(v, c);
            }
            if (c < k64) put(vx_load_vec<SRC>(row + c, K - c), c);
        }
    };
    int tile = slot + grid * ct;
    const int8_t *wrow = row_of(min(tile, tiles - 1));
    vx_i4 a[UN];
    const bool ahead = b0 + UN <= end_full;
    if (ahead && tile < tiles) {
#pragma unroll
        for (int u = 0; u < UN; ++u) a[u] = load(wrow, b0 + u);
    }
    if constexpr (SRC == VX_SRC_I8) {
        for (int m = wave; m < M; m += 16) {
            const int8_t *row = (const int8_t *)x + m * xs;
            for (int c = lane * 16; c < k64; c += 1024)
                *(vx_i4 *)(s_few + m * pitch + c) = c + 16 <= K ? (vx_i4)*(const vx_i4_at1 *)(row + c) : vx_i8_tail(row, c, K);
            if (lane == 0) s_scale[m] = s[m];
        }
    } else {
        // 1, 2, 4, 8 or 16 waves a row
        typedef typename vx_elem<SRC>::type E;
        constexpr int VEC = 16 / sizeof(E);
        const int wl = M == 1 ? 4 : (M > 8 ? 0 : 4 - (32 - __builtin_clz(M - 1))), step = 64 * VEC << wl;
        for (int m = wave >> wl; m < M; m += 16 >> wl) {          // wl > 0: one row each at most
            const E *row = (const E *)x + m * xs;
            const int lead = (wave & ((1 << wl) - 1)) * 64 * VEC, c0 = lead + lane * VEC;
            unsigned top = 0;
            int c = c0;
#pragma unroll 4
            for (; c - lane * VEC + 64 * VEC <= K; c += step) {
                vx_vec<SRC> v;
                v.raw = vx_load16<SRC>(row + c);
                top = vx_quant_look<SRC>(v, top);
            }
            if (c < K) top = vx_quant_look<SRC>(vx_load_vec<SRC>(row + c, K - c), top);
            top = vx_wave_max(top);
            if (wl) {
                if (lane == 0) s_top[wave] = top;
            } else {
                quantise(row, m, c0, step, vx_quant_row(top));
            }
        }
        if (wl) {
            __syncthreads();
            const int m = wave >> wl;
            if (m < M) {
                unsigned top = 0;
                for (int i = 0; i < 1 << wl; ++i) top = max(top, s_top[(m << wl) + i]);
                quantise((const E *)x + m * xs, m, ((wave & ((1 << wl) - 1)) * 64 + lane) * VEC, step, vx_quant_row(top));
            }
        }
    }
    __syncthreads();
    auto put = [&](int m, long long n, int sum) {
        const float y = vx_linear_out(sum, s_scale[m], sw[n], bias != nullptr, bias ? bias[n] : 0.f);
        if (out_dtype == VX_DTYPE_F32) ((float *)out)[m * os + n] = y;
        else if (out_dtype == VX_DTYPE_F16) ((_Float16 *)out)[m * os + n] = vx_store_cast<VX_DTYPE_F16>(y);
        else ((__bf16 *)out)[m * os + n] = vx_store_cast<VX_DTYPE_BF16>(y);
    };
    int *s_sum = (int *)(s_few + M * pitch);
    const int8_t *q[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) q[t] = s_few + min(t * 16 + (lane & 15), M - 1) * pitch + koff;
    for (int first = slot; first < tiles; first += grid * CT, tile += grid * CT) {      // first: the tile of the first wave
        const bool more = tile + grid * CT < tiles;
        const int8_t *next = row_of(more ? tile + grid * CT : tiles - 1);
        vx_i4 acc[MT] = {};
        const long long n0 = (long long)tile * 16 + (lane >> 4) * 4;
        float scale[4], plus[4];
        if (KS == 1) {                                            // in front of the next tile's weights
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                scale[k] = sw[min(n0 + k, N - 1)];
                plus[k] = bias ? bias[min(n0 + k, N - 1)] : 0.f;
            }
        }
        if (tile < tiles) {
            auto multiply = [&](const vx_i4 &weights, int at) {
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(weights, *(const vx_i4 *)(q[t] + at * 64), acc[t], 0, 0, 0);
            };
            int b = b0;
            if (ahead) {
                for (; b + 2 * UN <= end_full; b += UN) {
#pragma unroll
                    for (int u = 0; u < UN; ++u) {
                        multiply(a[u], b + u);
                        a[u] = load(wrow, b + UN + u);
                    }
                }
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    multiply(a[u], b + u);
                    if (more) a[u] = load(next, b0 + u);
                }
                b += UN;
            }
            for (; b + 4 <= end_full; b += 4) {
                vx_i4 v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = load(wrow, b + u);
#pragma unroll
                for (int u = 0; u < 4; ++u) multiply(v[u], b + u);
            }
            for (; b < end_full; ++b) multiply(load(wrow, b), b);
            if (b < end) {                                        // weights from K on meet zeros; those outside the matrix are not read
                const int k = b * 64;
                multiply(wrow + k + 16 <= w + (N - 1) * ws + K ? load(wrow, b) : vx_i8_tail(wrow, k, K - koff), b);
            }
        }
        wrow = next;
        // lane l holds token l % 16, channels 4 (l / 16) .. + 3
        if (KS == 1) {
            if (tile < tiles) {
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const int m = t * 16 + (lane & 15);
                    if (m >= M) continue;
                    float y[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) y[k] = vx_linear_out(acc[t][k], s_scale[m], scale[k], bias != nullptr, plus[k]);
                    if (out_dtype == VX_DTYPE_F32) vx_store4<VX_DTYPE_F32>(out, m * os + n0, y, N - n0);
                    else if (out_dtype == VX_DTYPE_F16) vx_store4<VX_DTYPE_F16>(out, m * os + n0, y, N - n0);
                    else vx_store4<VX_DTYPE_BF16>(out, m * os + n0, y, N - n0);
                }
            }
        } else {
            __syncthreads();                                      // the sums of the tiles before are read
            if (tile < tiles) {
#pragma unroll
                for (int t = 0; t < MT; ++t) *(vx_i4 *)&s_sum[(wave * MT + t) * 256 + (lane & 15) * 16 + (lane >> 4) * 4] = acc[t];
            }
            __syncthreads();
            for (int i = threadIdx.x; i < CT * MT * 256; i += 1024) {
                const int c = i / (MT * 256), r = i - c * (MT * 256), m = r >> 4, at = first + grid * c;
                const long long n = (long long)at * 16 + (r & 15);
                if (m >= M || at >= tiles || n >= N) continue;
                int sum = 0;
                for (int k = 0; k < KS; ++k) sum += s_sum[((c << ks_log2) + k) * MT * 256 + r];
                put(m, n, sum);
            }
        }
    }
}

static int vx_few_ks(int64_t N) {                                 // log2 of the waves that share K: as many as leave none without a tile
    const int64_t tiles = (N + 15) / 16;
    int l = 0;
    while (l < 4 && (tiles << (l + 1)) <= 256 * 16) ++l;
    return l;
}
static size_t vx_few_lds(int64_t M, int64_t N, int K) {
    return (size_t)M * (((K + 63) & ~63) + 16) + (vx_few_ks(N) ? (size_t)16 * ((M + 15) / 16) * 1024 : 0);
}
#define VX_FEW_MAX 64
static bool vx_few_fits(int64_t M, int64_t N, int K) { return M <= VX_FEW_MAX && vx_few_lds(M, N, K) <= 160 * 1024 - 512; }
// Which products with quantisation go this way (us, this / quantise and multiply; bf16): every workgroup quantises all M x K values,
// which costs it what the saved launch cost at about 32768 of them:
//   32000 x 4096, M = 4: 28/29, 8: 29/30    4096 x 4096, M = 4: 10/11, 8: 11/11, 16: 13/11    8192 x 8192, M = 4: 19/20, 8: 22/21
//   131072 x 2048, M = 16: 55/56, 32: 60/58    16384 x 1024, M = 32: 11/12, 64: 16/13
// With K not a multiple of 16 the quantised tokens would not go by tiles but by this kernel (more than 16384 channels) or the
// streaming one, both slower at odd addresses, and it is about 65536 (with few channels less, where neither is far behind):
//   50021 x 1000, M = 32: 19/22, 37: 21/24, 64: 25/27    16000 x 1000, M = 64: 17/18    16000 x 1500, M = 40: 18/19
//   4096 x 1001, M = 33: 10/11    4096 x 1000, M = 64: 13/12    8192 x 600, M = 64: 14/12    12000 x 1023, M = 64: 24/22
//   8192 x 8201, M = 5: 31/33    32000 x 5000, M = 8: 37/37    32000 x 4001, M = 16: 51/50    32000 x 2001, M = 32: 32/32
static bool vx_linear_by_few(int64_t M, int64_t N, int K) { return vx_few_fits(M, N, K) && M * K <= (K % 16 ? 65536 : 32768); }
// Which products of quantised tokens: many channels, and few tokens or K not a multiple of 16 (us, this / streaming or tiles):
//   32000 x 4096, M = 4: 26/26, 8: 26/30, 16: 27/32    131072 x 2048, M = 1: 47/46, 8: 50/56, 16: 52/53, 32: 55/54
//   50021 x 1000, M = 4: 15/18, 16: 15/22, 37: 20/34, 64: 23/43    4096 x 4096, M = 8: 7.7/6.7    16384 x 1024, M = 16: 7/7
static bool vx_i8_by_few(int64_t M, int64_t N, int K) { return M > 1 && N > 16384 && (M <= 16 || K % 16) && vx_few_fits(M, N, K); }

template <int SRC>
static void vx_few_launch(const void *x, long long xs, const float *s, int M, const int8_t *w, long long ws, const float *sw, long long N,
                          int K, const float *bias, void *out, int out_dtype, long long os, hipStream_t st) {
    const int tiles = (int)((N + 15) / 16), ks = vx_few_ks(N);
    const dim3 grid((unsigned)min(tiles, 256));
    const size_t lds = vx_few_lds(M, N, K);
    if (M <= 16) hipLaunchKernelGGL((vx_k_linear_few<SRC, 1, 12>), grid, dim3(1024), lds, st, x, xs, s, M, w, ws, sw, N, K, bias, out, out_dtype, os, tiles, ks);
    else if (M <= 32) hipLaunchKernelGGL((vx_k_linear_few<SRC, 2, 12>), grid, dim3(1024), lds, st, x, xs, s, M, w, ws, sw, N, K, bias, out, out_dtype, os, tiles, ks);
    else if (M <= 48) hipLaunchKernelGGL((vx_k_linear_few<SRC, 3, 8>), grid, dim3(1024), lds, st, x, xs, s, M, w, ws, sw, N, K, bias, out, out_dtype, os, tiles, ks);
    else hipLaunchKernelGGL((vx_k_linear_few<SRC, 4, 8>), grid, dim3(1024), lds, st, x, xs, s, M, w, ws, sw, N, K, bias, out, out_dtype, os, tiles, ks);
}

// ---- many tokens: TM x TN outputs for each workgroup, WM x WN waves of 32x32x32 mfma tiles (weights as rows, tokens as
// columns, so a lane's four accumulators in a row are four neighbouring channels of one token).
// K goes by stages of 128 bytes, a whole cache line of each row (requests of 64 bytes found the line of the request before
// still on its way), through LDS that the loads fill directly: three stages of weights, two of tokens, all 160 KB of a
// compute unit.  A stage is worked off in two halves; each wave reads its operands of the next half into registers while
// the matrix instructions of this one run.  One barrier a stage: behind it stage d + 1 is there for every wave and nobody
// reads stage d any more.
// The 16-byte pieces of an LDS row are stored at piece ^ ((row >> 1) & 7), so the 16 rows that a quarter of a wave's 16-byte
// LDS read covers lie in all 64 banks.
// 8192 x 16384 x 4096: 508 us (the kernel's median), 2.16 Pop/s; the matrix instructions are busy 58 % of the cycles (counted), at a
// clock that the card has brought down to 1.8 GHz.
// Needs 16-byte aligned rows; q padded with zeros to a multiple of 128, w's pieces beyond K read as piece 0 (K % 16 == 0).
template <int N>
__device__ __forceinline__ void vx_wait_stage() {                 // at most N loads and no LDS read outstanding, then the barrier
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (0 << 8) | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int DT, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void vx_k_linear_tile(const int8_t *__restrict__ q, long long qs,
                                                                 const float *__restrict__ s, long long M,
                                                                 const int8_t *__restrict__ w, long long ws,
                                                                 const float *__restrict__ sw, long long N, int K,
                                                                 const float *__restrict__ bias, void *__restrict__ out,
                                                                 long long os, int gm, int gn) {
    typedef typename vx_elem<DT>::type E;
    constexpr int WAVES = WM * WN, NI = TN / WN / 32, MJ = TM / WM / 32;
    constexpr int LW = TN / 8 / WAVES, LQ = TM / 8 / WAVES;       // loads of one wave for a stage, 8 rows each
    constexpr int RING = 3 * TN * 128 + 2 * TM * 128;
    __shared__ __attribute__((aligned(1024))) int8_t s_ring[RING];
    const int tile = vx_xcd_tile(blockIdx.x, gm * gn);
    if (tile < 0) return;
    // eight tiles of tokens by four of channels are in flight on an XCD: its L2 holds what they share
    const int band = tile / (8 * gn), in_band = tile - band * 8 * gn, bh = min(8, gm - band * 8);
    const long long m0 = (long long)(band * 8 + in_band % bh) * TM, n0 = (long long)(in_band / bh) * TN;
    const int lane = vx_lane(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int stages = (K + 127) >> 7;

    // what this wave loads of a stage: 8 rows with each instruction, 8 lanes a row; the lane's slot holds piece `piece`
    const int8_t *src_w[LW], *src_q[LQ];
    const int row8 = wave * 8 + (lane >> 3), piece = ((lane & 7) ^ ((row8 >> 1) & 7)) * 16;  // the same for rows 8 WAVES further
#pragma unroll
    for (int i = 0; i < LW; ++i) src_w[i] = w + min(n0 + i * WAVES * 8 + row8, N - 1) * ws;
#pragma unroll
    for (int i = 0; i < LQ; ++i) src_q[i] = q + min(m0 + i * WAVES * 8 + row8, M - 1) * qs + piece;
    auto request_w = [&](int d, int slot, int i) {
        const int k = d * 128 + piece;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(src_w[i] + (k < K ? k : 0)),
                                         (__attribute__((address_space(3))) void *)(s_ring + slot + (i * WAVES + wave) * 1024), 16, 0, 0);
    };
    auto request_q = [&](int d, int i) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(src_q[i] + d * 128),
                                         (__attribute__((address_space(3))) void *)(s_ring + 3 * TN * 128 + (d & 1) * TM * 128 + (i * WAVES + wave) * 1024),
                                         16, 0, 0);
    };
    // the lane's byte offsets of its operands inside a stage, for its four quarters of 32 bytes
    const int lr = lane & 31;
    int at_w[4], at_q[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        const int p = ((2 * h + (lane >> 5)) ^ ((lr >> 1) & 7)) * 16;
        at_w[h] = (wn * (TN / WN) + lr) * 128 + p;
        at_q[h] = 3 * TN * 128 + (wm * (TM / WM) + lr) * 128 + p;
    }
    vx_i4 fw[2][2][NI], fq[2][2][MJ];                             // operands of the two halves of a stage
    vx_i16 acc[NI][MJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MJ; ++j)
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[i][j][k] = 0;
    // Half `set` of a stage: its matrix instructions, with an LDS read (of half set ^ 1: of this stage, or of the next one)
    // or a request in front of each, in this order.
    auto half = [&](int set, bool read, int base_w, int base_q, auto request, int requests) {
        constexpr int READS = 2 * (NI + MJ), MULS = 2 * NI * MJ, TOTAL = READS + (LW > LQ ? LW : LQ);
#pragma unroll
        for (int k = 0; k < (MULS > TOTAL ? MULS : TOTAL); ++k) {
            if (k < READS) {
                const int h = k / (NI + MJ), r = k % (NI + MJ), h4 = 2 * (set ^ 1) + h;
                if (read) {
                    if (r < NI) fw[set ^ 1][h][r] = *(const vx_i4 *)(s_ring + base_w + at_w[h4] + r * 4096);
                    else fq[set ^ 1][h][r - NI] = *(const vx_i4 *)(s_ring + base_q + at_q[h4] + (r - NI) * 4096);
                }
            } else if (k - READS < requests) {
                request(k - READS);
            }
            if (k < MULS) {
                const int h = k / (NI * MJ), i = k / MJ % NI, j = k % MJ;
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[set][h][i], fq[set][h][j], acc[i][j], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto nothing = [](int) {};

    int slot = 0, slot1 = TN * 128, slot2 = 2 * TN * 128;         // of the weights of stages d, d + 1, d + 2
#pragma unroll
    for (int i = 0; i < LW; ++i) request_w(0, slot, i);
#pragma unroll
    for (int i = 0; i < LQ; ++i) request_q(0, i);
    if (stages > 1) {
#pragma unroll
        for (int i = 0; i < LW; ++i) request_w(1, slot1, i);
#pragma unroll
        for (int i = 0; i < LQ; ++i) request_q(1, i);
        vx_wait_stage<LW + LQ>();
    } else {
        vx_wait_stage<0>();
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < NI; ++i) fw[0][h][i] = *(const vx_i4 *)(s_ring + at_w[h] + i * 4096);
#pragma unroll
        for (int j = 0; j < MJ; ++j) fq[0][h][j] = *(const vx_i4 *)(s_ring + at_q[h] + j * 4096);
    }
    int d = 0;
    for (; d + 2 < stages; ++d) {
        const int here = (d & 1) * TM * 128, next = TM * 128 - here;
        half(0, true, slot, here, [&](int i) { request_w(d + 2, slot2, i); }, LW);   // slot2: stage d - 1's, done with since the last barrier
        vx_wait_stage<LW>();
        half(1, true, slot1, next, [&](int i) { request_q(d + 2, i); }, LQ);         // into stage d's place
        const int s0 = slot;
        slot = slot1; slot1 = slot2; slot2 = s0;
    }
    for (; d < stages; ++d) {
        const int here = (d & 1) * TM * 128, next = TM * 128 - here;
        half(0, true, slot, here, nothing, 0);
        vx_wait_stage<0>();
        half(1, d + 1 < stages, slot1, next, nothing, 0);
        slot = slot1; slot1 = slot2;
    }

    // Results.  Accumulator r of a tile: channel 8 (r / 4) + 4 (lane / 32) + r % 4, token lane % 32.  Stored from there, a
    // wave's store would touch 32 rows with 16 bytes each (400 of 900 us at 8192 x 16384 x 4096); instead they go through
    // the wave's part of the ring, 32 tokens at a time, and leave as whole rows of its channels.  A row's 16-byte pieces are
    // stored at piece ^ ((row >> 1) & 7): writes and reads both spread over all banks.
    constexpr int CH = TN / WN, PIECES = CH * (int)sizeof(E) / 16, ROWS = 64 / PIECES;       // rows of one store instruction
    static_assert(WAVES * 32 * CH * 4 <= RING, "a wave's 32 rows of results fit its part of the ring");
    vx_wait_stage<0>();                                           // every wave is done with the ring
    int8_t *mine = s_ring + wave * (32 * CH * 4);
    const long long nw = n0 + wn * CH;
    float scale[NI][4][4], plus[NI][4][4];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const long long n = min(nw + i * 32 + 8 * g + 4 * (lane >> 5) + k, N - 1);
                scale[i][g][k] = sw[n];
                plus[i][g][k] = bias ? bias[n] : 0.f;
            }
#pragma unroll
    for (int j = 0; j < MJ; ++j) {
        const long long mj = m0 + wm * (TM / WM) + j * 32;
        const float sm = s[min(mj + lr, M - 1)];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                union { E e[4]; vx_v2 v2; vx_v4 v4; } o;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    o.e[k] = vx_store_cast<DT>(vx_linear_out(acc[i][j][4 * g + k], sm, scale[i][g][k], bias != nullptr, plus[i][g][k]));
                const int col = (i * 32 + 8 * g + 4 * (lane >> 5)) * (int)sizeof(E), piece = (col >> 4) ^ ((lr >> 1) & (PIECES < 8 ? PIECES - 1 : 7));
                int8_t *to = mine + lr * (CH * (int)sizeof(E)) + piece * 16 + (col & 15);
                if (sizeof(E) == 2) *(vx_v2 *)to = o.v2;
                else *(vx_v4 *)to = o.v4;
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += ROWS) {
            const int r = r0 + lane / PIECES, p = lane % PIECES;
            union { vx_v4 v; E e[16 / sizeof(E)]; } o;
            o.v = *(const vx_v4 *)(mine + r * (CH * (int)sizeof(E)) + (p ^ ((r >> 1) & (PIECES < 8 ? PIECES - 1 : 7))) * 16);
            const long long m = mj + r, n = nw + p * (16 / (int)sizeof(E));
            if (m < M) {
                E *to = (E *)out + m * os + n;
                if (n + 16 / (int)sizeof(E) <= N) {
                    if (sizeof(E) == 2) *(vx_v4_at2 *)to = o.v;
                    else *(vx_v4_at4 *)to = o.v;
                } else {
#pragma unroll
                    for (int k = 0; k < 16 / (int)sizeof(E); ++k)
                        if (n + k < N) to[k] = o.e[k];
                }
            }
        }
    }
}

// ---- many tokens, few channels: the weights stay in registers and x passes by once; no quantised copy of it in memory.
// A persistent workgroup of 16 waves, each with 16 channels x KC bytes of weights (16x16x64 as in the streaming kernel).  For each
// tile of 16 tokens a wave quantises one row into LDS from registers that were filled two tiles ahead, multiplies the tile with
// its channels, and stores one row of the results of the tile before: one barrier a tile, all LDS double.  Rows in LDS are an
// odd number of 16-byte pieces long: 16 of them lie in all banks.  With KC = 1024 a third of the weights is in LDS instead: 128
// registers are all that 16 waves have.
// Bound by the read of x: 43264 x 255 x 1024 (1x1 convolution in front of a YOLO layer) fp32 in 54 us, 221 MB at 4.1 TB/s;
// quantised to memory and multiplied by tiles 71.  A workgroup for each 64 / 32 / 16 tokens that read the weights from L2 took
// 70 / 92 / 122.
// Needs K a multiple of 16 (the pieces of weights beyond K lie inside the row before) and up to 256 channels.
#define VX_ROWS_MAX_N 256
template <int OT>
__device__ __forceinline__ void vx_linear_put_row(const float *y, void *out, long long at, int N) {
    typedef typename vx_elem<OT>::type O;
    constexpr int OV = 16 / sizeof(O);
    const int c = vx_lane() * OV;
    if (c >= N) return;
    vx_vec<OT> o;
#pragma unroll
    for (int k = 0; k < OV; k += 4) {
        const vx_v4 v = *(const vx_v4 *)(y + c + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) o.e[k + j] = vx_store_cast<OT>(v[j]);
    }
    O *to = (O *)((char *)out + at * (long long)sizeof(O) + vx_lane() * 16u);
    if (c + OV <= N) {
        if (sizeof(O) == 2) *(vx_v4_at2 *)to = o.raw;
        else *(vx_v4_at4 *)to = o.raw;
    } else {
#pragma unroll
        for (int k = 0; k < OV; ++k)
            if (c + k < N) to[k] = o.e[k];
    }
}

template <int DT, int KC>
__global__ __launch_bounds__(1024) void vx_k_linear_rows(const void *__restrict__ x, long long xs, long long M,
                                                         const int8_t *__restrict__ w, long long ws, const float *__restrict__ sw,
                                                         int N, int K, const float *__restrict__ bias, void *__restrict__ out,
                                                         int out_dtype, long long os) {
    typedef typename vx_elem<DT>::type E;
    constexpr int VEC = 16 / sizeof(E), U = KC > 64 * VEC ? KC / (64 * VEC) : 1, B = KC / 64, PITCH = KC + 16, YP = VX_ROWS_MAX_N + 4;
    constexpr int BL = KC > 512 ? 5 : 0, BR = B - BL;         // 64-byte blocks of weights in LDS and in registers
    __shared__ __attribute__((aligned(16))) int8_t s_w[BL ? BL * 16384 : 16];
    __shared__ __attribute__((aligned(16))) int8_t s_q[2][16 * PITCH];
    __shared__ __attribute__((aligned(16))) float s_y[2][16 * YP], s_sw[VX_ROWS_MAX_N], s_bias[VX_ROWS_MAX_N];
    __shared__ float s_scale[2][16];
    const int lane = vx_lane(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long tiles = (M + 15) >> 4;
    auto fetch = [&](vx_vec<DT> (&v)[U], long long tile) {       // without a branch: the loads in flight stay countable
        const char *row = (const char *)((const E *)x + min(tile * 16 + wave, M - 1) * xs);
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].raw = vx_load16<DT>((const E *)(row + min((u * 64 + lane) * 16u, (unsigned)(K * sizeof(E) - 16))));
    };
    vx_vec<DT> va[U], vb[U];
    fetch(va, blockIdx.x);
    fetch(vb, (long long)blockIdx.x + gridDim.x);
    const int n = wave * 16 + (lane & 15), koff = (lane >> 4) * 16;
    const int8_t *wrow = w + min(n, N - 1) * ws;
    // pieces from K on meet zeros of q: what they hold does not matter
    auto load_w = [&](int b) { return (vx_i4)*(const vx_i4_at1 *)(wrow + min(b * 64 + koff, K - 16)); };
    vx_i4 weights[BR];
#pragma unroll
    for (int b = 0; b < BR; ++b) weights[b] = load_w(b);
    for (int b = 0; b < BL; ++b) *(vx_i4 *)(s_w + ((b * 16 + wave) * 64 + lane) * 16) = load_w(BR + b);   // read by this lane only
    if (threadIdx.x < N) {
        s_sw[threadIdx.x] = sw[threadIdx.x];
        s_bias[threadIdx.x] = bias ? bias[threadIdx.x] : 0.f;
    }
    auto put = [&](int buf, long long tile) {
        const long long m = tile * 16 + wave;
        if (m >= M) return;
        const float *y = &s_y[buf][wave * YP];
        if (out_dtype == VX_DTYPE_F32) vx_linear_put_row<VX_DTYPE_F32>(y, out, m * os, N);
        else if (out_dtype == VX_DTYPE_F16) vx_linear_put_row<VX_DTYPE_F16>(y, out, m * os, N);
        else vx_linear_put_row<VX_DTYPE_BF16>(y, out, m * os, N);
    };
    auto step = [&](vx_vec<DT> (&v)[U], int buf, long long tile) {
        unsigned top = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if ((u * 64 + lane) * VEC >= K) v[u].raw = vx_v4{0.f, 0.f, 0.f, 0.f};
            top = vx_quant_look<DT>(v[u], top);
        }
        top = vx_wave_max(top);
        const vx_quant_row what(top);
        if (lane == 0) s_scale[buf][wave] = what.scale();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = (u * 64 + lane) * VEC;
            const vx_quant_out<DT> o = vx_quant_piece<DT>(v[u], what);
            if (U * 64 * VEC == KC || c < KC) {
#pragma unroll
                for (int k = 0; k < VEC / 4; ++k) *(unsigned *)(&s_q[buf][wave * PITCH + c + 4 * k]) = o.w[k];
            }
        }
        __syncthreads();
        if (tile != blockIdx.x) put(buf ^ 1, tile - gridDim.x);
        fetch(v, tile + 2 * (long long)gridDim.x);
        vx_i4 acc[2] = {};
        const int8_t *q = &s_q[buf][(lane & 15) * PITCH + koff];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const vx_i4 a = b < BR ? weights[b < BR ? b : 0] : *(const vx_i4 *)(s_w + (((b - BR) * 16 + wave) * 64 + lane) * 16);
            acc[b & 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, *(const vx_i4 *)(q + b * 64), acc[b & 1], 0, 0, 0);
            if (b % 4 == 3) __builtin_amdgcn_sched_barrier(0);    // no more operands on their way than registers left
        }
        // lane l holds token l % 16, channels 4 (l / 16) .. + 3 of the wave's
        const int n4 = wave * 16 + (lane >> 4) * 4;
        const float sm = s_scale[buf][lane & 15];
        vx_v4 y;
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = vx_linear_out(acc[0][k] + acc[1][k], sm, s_sw[n4 + k], bias != nullptr, s_bias[n4 + k]);
        *(vx_v4 *)&s_y[buf][(lane & 15) * YP + n4] = y;
    };
    long long tile = blockIdx.x;                                  // the grid has no more workgroups than tiles
    while (true) {
        step(va, 0, tile);
        if (tile + gridDim.x >= tiles) { __syncthreads(); put(0, tile); return; }
        tile += gridDim.x;
        step(vb, 1, tile);
        if (tile + gridDim.x >= tiles) { __syncthreads(); put(1, tile); return; }
        tile += gridDim.x;
    }
}

// Which products with quantisation go this way (us, this / quantise and multiply; N = 255, x fp32):
// M = 43264: K = 256 23/39, 512 31/48, 1024 54/69; M = 8192: 8/13, 11/16, 20/19; M = 65: 5/8, 7/8, 12/10 (the weights take longer to
// arrive than to be used; called one by one, 15/17, the saved launch is worth more).  N = 64 behaves alike.
#define VX_STREAM_MAX 64
#define VX_ROWS_MAX_K 1024
static bool vx_linear_by_rows(int64_t M, int64_t N, int K) {
    return M > VX_STREAM_MAX && N <= VX_ROWS_MAX_N && K <= VX_ROWS_MAX_K && K % 16 == 0;
}

static int vx_linear_rows_launch(const void *x, int dtype, long long xs, long long M, const int8_t *w, long long ws, const float *sw, int N,
                                 int K, const float *bias, void *out, int out_dtype, long long os, hipStream_t st) {
    vx_prof_begin(VX_PROF_LINEAR, st);
    const dim3 grid((unsigned)min((M + 15) / 16, 256LL));         // one workgroup a compute unit
    VX_DISPATCH_DTYPE(dtype, {
        if (K <= 256) hipLaunchKernelGGL((vx_k_linear_rows<DT, 256>), grid, dim3(1024), 0, st, x, xs, M, w, ws, sw, N, K, bias, out, out_dtype, os);
        else if (K <= 512) hipLaunchKernelGGL((vx_k_linear_rows<DT, 512>), grid, dim3(1024), 0, st, x, xs, M, w, ws, sw, N, K, bias, out, out_dtype, os);
        else hipLaunchKernelGGL((vx_k_linear_rows<DT, 1024>), grid, dim3(1024), 0, st, x, xs, M, w, ws, sw, N, K, bias, out, out_dtype, os);
    });
    vx_prof_end(VX_PROF_LINEAR, st);
    return hipGetLastError() == hipSuccess ? VX_OK : VX_ERR_LAUNCH;
}

// rows of K bytes to rows of `pitch` (a multiple of 128), padded with zeros
__global__ __launch_bounds__(256) void vx_k_pad_rows(const int8_t *__restrict__ src, long long stride, long long rows, int K,
                                                     int8_t *__restrict__ dst, int pitch) {
    const int pieces = pitch / 16;
    const long long i = (long long)vx_block() * 256 + threadIdx.x;
    if (i >= rows * pieces) return;
    const long long r = i / pieces;
    const int k = (int)(i - r * pieces) * 16;
    const int8_t *row = src + r * stride;
    *(vx_i4 *)(dst + r * pitch + k) = k + 16 <= K ? (vx_i4)*(const vx_i4_at1 *)(row + k) : vx_i8_tail(row, k, K);
}

// Which kernel takes M quantised tokens (us of the product, N x K), streaming / 64 x 64 tiles:
//   M <= 8: streaming (16000 x 4096: 18/22, 4096 x 4096 7/17)
//   M <= 16: streaming up to 16384 channels (4096 x 4096 8/17, 12000 x 2048 9/11, 16000 x 4096 19/20)
//   M <= 32: streaming up to 10240 channels (M = 32: 4096 x 4096 13/17, 8192 x 4096 15/18, but 12000 x 2048 13/11, 16000 x 4096 23/21;
//            M = 64: 4096 x 4096 17/17, 8192 x 1024 9/7, 8192 x 4096 19/18, 8192 x 8192 31/32)
//   M <= 64: streaming with K not a multiple of 16, which the tiles would have to copy (5000 x 1000, M = 64: 9/16)
//   more: the largest tile that is at least half full of tokens and gives at least 192 workgroups, three for four compute
//   units (by 64 / 128 / 256.  32000 x 4096: M = 64 32/35/55, 96 40/39/55, 384 99/70/67.  8192 x 4096: M = 1024, 128 tiles of
//   256, 63/42/57; M = 1536, 192 of them, 87/66/61.  8192 x 8192: M = 128, 64 tiles of 128, 45/56/94; M = 512, 256 of them, 65/58/97)
static bool vx_linear_streams(int64_t M, int64_t N, int K) {
    return vx_i8_by_few(M, N, K) || M <= 8 || (M <= 16 && N <= 16384) || (M <= 32 && N <= 10240) || (M <= VX_STREAM_MAX && K % 16);
}

static size_t vx_up256(size_t n) { return (n + 255) & ~(size_t)255; }
static long long vx_k_pitch(int K) { return ((long long)K + 127) / 128 * 128; }

template <int DT, int T, int WM, int WN>
static void vx_linear_tiles(const int8_t *q, long long qs, const float *s, long long M, const int8_t *w, long long ws, const float *sw,
                            long long N, int K, const float *bias, void *out, long long os, hipStream_t st) {
    const int gm = (int)((M + T - 1) / T), gn = (int)((N + T - 1) / T);
    hipLaunchKernelGGL((vx_k_linear_tile<DT, T, T, WM, WN>), dim3((unsigned)(8 * (((long long)gm * gn + 7) / 8))), dim3(WM * WN * 64), 0, st,
                       q, qs, s, M, w, ws, sw, N, K, bias, out, os, gm, gn);
}

// q_padded: columns K .. vx_k_pitch(K) - 1 of q are zeros.  pad: 256-byte aligned room for the padded copies that
// vx_linear_i8_workspace_bytes counts.
static int vx_linear_launch(const int8_t *q, long long qs, bool q_padded, const float *s, long long M, const int8_t *w, long long ws,
                            const float *sw, long long N, int K, const float *bias, void *out, int out_dtype, long long os,
                            int8_t *pad, hipStream_t st) {
    const long long pitch = vx_k_pitch(K);
    bool tiles = !vx_linear_streams(M, N, K);
    vx_prof_begin(VX_PROF_LINEAR, st);
    if (vx_i8_by_few(M, N, K)) {
        vx_few_launch<VX_SRC_I8>(q, qs, s, (int)M, w, ws, sw, N, K, bias, out, out_dtype, os, st);
        vx_prof_end(VX_PROF_LINEAR, st);
        return hipGetLastError() == hipSuccess ? VX_OK : VX_ERR_LAUNCH;
    }
    if (tiles) {
        if (K % 128 && !q_padded) {
            const long long n = M * (pitch / 16);
            hipLaunchKernelGGL(vx_k_pad_rows, vx_grid((n + 255) / 256), dim3(256), 0, st, q, qs, M, K, pad, (int)pitch);
            q = pad;
            qs = pitch;
            pad += vx_up256((size_t)(M * pitch));
        }
        if (K % 16) {
            const long long n = N * (pitch / 16);
            hipLaunchKernelGGL(vx_k_pad_rows, vx_grid((n + 255) / 256), dim3(256), 0, st, w, ws, N, K, pad, (int)pitch);
            w = pad;
            ws = pitch;
        }
        // rows at odd addresses go by the streaming kernel, 64 tokens at a time
        tiles = !(((uintptr_t)q | (uintptr_t)w) & 15) && !((qs | ws) & 15);
    }
    if (tiles) {
        auto count = [&](int t) { return ((M + t - 1) / t) * ((N + t - 1) / t); };
        VX_DISPATCH_DTYPE(out_dtype, {
            if (M > 128 && count(256) >= 192) vx_linear_tiles<DT, 256, 2, 4>(q, qs, s, M, w, ws, sw, N, K, bias, out, os, st);
            else if (M > 64 && count(128) >= 192) vx_linear_tiles<DT, 128, 2, 2>(q, qs, s, M, w, ws, sw, N, K, bias, out, os, st);
            else vx_linear_tiles<DT, 64, 2, 2>(q, qs, s, M, w, ws, sw, N, K, bias, out, os, st);
        });
    } else {
        // two tiles of channels share the tokens' loads where there is more than one tile of tokens, and eight waves their K
        // (16000 x 2048, M = 32: 13 us, two / four waves 16 / 14); one tile: four waves, or 16 with few channels
        const int mt = (int)min(4LL, (M + 15) / 16), nt = mt == 1 ? 1 : 2;
        const int waves = mt > 1 ? 8 : (N <= 4096 ? 16 : 4);
        const dim3 grid((unsigned)((N + 16 * nt - 1) / (16 * nt)), (unsigned)((M + 16 * mt - 1) / (16 * mt)));
        const size_t lds = (size_t)waves * mt * nt * 1024;
        VX_DISPATCH_DTYPE(out_dtype, {
            if (mt == 1) hipLaunchKernelGGL((vx_k_linear_stream<DT, 1, 1>), grid, dim3(waves * 64), lds, st, q, qs, s, M, w, ws, sw, N, K, bias, out, os);
            else if (mt == 2) hipLaunchKernelGGL((vx_k_linear_stream<DT, 2, 2>), grid, dim3(waves * 64), lds, st, q, qs, s, M, w, ws, sw, N, K, bias, out, os);
            else if (mt == 3) hipLaunchKernelGGL((vx_k_linear_stream<DT, 3, 2>), grid, dim3(waves * 64), lds, st, q, qs, s, M, w, ws, sw, N, K, bias, out, os);
            else hipLaunchKernelGGL((vx_k_linear_stream<DT, 4, 2>), grid, dim3(waves * 64), lds, st, q, qs, s, M, w, ws, sw, N, K, bias, out, os);
        });
    }
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

static bool vx_linear_sizes_ok(int64_t M, int64_t N, int K) {
    return M > 0 && N > 0 && K > 0 && M <= VX_MAX_LINEAR_ROWS && N <= VX_MAX_LINEAR_ROWS && K <= VX_MAX_I8_DEPTH;
}

// the padded copies of vx_linear_launch
static size_t vx_linear_pad_bytes(int64_t M, int64_t N, int K, bool q_padded) {
    if (vx_linear_streams(M, N, K)) return 0;
    const size_t pitch = (size_t)vx_k_pitch(K);
    return (K % 128 && !q_padded ? vx_up256((size_t)M * pitch) : 0) + (K % 16 ? vx_up256((size_t)N * pitch) : 0);
}

extern "C" size_t vx_linear_i8_workspace_bytes(int64_t M, int64_t N, int K) {
    return vx_linear_sizes_ok(M, N, K) ? 256 + vx_linear_pad_bytes(M, N, K, false) : 0;
}

extern "C" int vx_linear_i8(const int8_t *d_q, int64_t q_stride, const float *d_scale, int64_t M, const int8_t *d_w,
                            int64_t w_stride, const float *d_w_scale, int64_t N, int K, const float *d_bias, void *d_out,
                            int out_dtype, int64_t out_stride, void *d_workspace, size_t workspace_bytes, void *stream) {
    if (!d_scale || !d_workspace) return VX_ERR_INVALID_ARG;
    const int rc = vx_linear_check(d_q, q_stride, d_w, w_stride, d_w_scale, M, N, K, d_bias, d_out, out_dtype, out_stride);
    if (rc != VX_OK) return rc;
    if (((uintptr_t)d_scale & 3) || ((uintptr_t)d_workspace & 255)) return VX_ERR_ALIGNMENT;
    if (workspace_bytes < vx_linear_i8_workspace_bytes(M, N, K)) return VX_ERR_WORKSPACE;
    return vx_linear_launch(d_q, q_stride, false, d_scale, M, d_w, w_stride, d_w_scale, N, K, d_bias, d_out, out_dtype, out_stride,
                            (int8_t *)d_workspace, (hipStream_t)stream);
}

extern "C" size_t vx_linear_w8a8_workspace_bytes(int64_t M, int64_t N, int K) {
    if (!vx_linear_sizes_ok(M, N, K)) return 0;
    return 256 + vx_up256((size_t)M * 4) + vx_up256((size_t)(M * vx_k_pitch(K))) + vx_linear_pad_bytes(M, N, K, true);
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
    if (vx_linear_by_one(M, N, K))
        return vx_linear_one_launch(d_x, x_dtype, d_w, w_stride, d_w_scale, N, K, d_bias, d_out, out_dtype, st);
    if (vx_linear_by_few(M, N, K)) {
        vx_prof_begin(VX_PROF_LINEAR, st);
        VX_DISPATCH_DTYPE(x_dtype, vx_few_launch<DT>(d_x, x_stride, nullptr, (int)M, d_w, w_stride, d_w_scale, N, K, d_bias, d_out, out_dtype, out_stride, st););
        vx_prof_end(VX_PROF_LINEAR, st);
        return hipGetLastError() == hipSuccess ? VX_OK : VX_ERR_LAUNCH;
    }
    if (vx_linear_by_rows(M, N, K))
        return vx_linear_rows_launch(d_x, x_dtype, x_stride, M, d_w, w_stride, d_w_scale, (int)N, K, d_bias, d_out, out_dtype, out_stride, st);
    const long long pitch = vx_k_pitch(K);
    float *s = (float *)d_workspace;
    int8_t *q = (int8_t *)d_workspace + vx_up256((size_t)M * 4), *pad = q + vx_up256((size_t)(M * pitch));
    rc = vx_quant_launch(d_x, x_dtype, M, K, x_stride, q, pitch, s, st);
    if (rc != VX_OK) return rc;
    return vx_linear_launch(q, pitch, true, s, M, d_w, w_stride, d_w_scale, N, K, d_bias, d_out, out_dtype, out_stride, pad, st);
}
