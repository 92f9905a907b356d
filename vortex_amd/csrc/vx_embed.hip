// Embedding lookup with scaling and its gradient.
//   out[t,:]     = scale * table[ids[t],:]                        (id < 0: padding, a row of zeros)
//   d_table[v,:] = scale * sum over t with ids[t] == v of grad_out[t,:]
#include "vx_dtype.h"
#include "vx_profile.h"

__device__ __forceinline__ long long vx_id_at(const void *ids, int id_bytes, long long t) {
    return id_bytes == 8 ? ((const long long *)ids)[t] : (long long)((const int *)ids)[t];
}

// One workgroup per token.
template <int DT>
__global__ __launch_bounds__(256) void vx_k_embed(const void *__restrict__ ids, int id_bytes, const void *__restrict__ table,
                                                  long long n_rows, int D, long long stride, float scale,
                                                  void *__restrict__ out, int *__restrict__ status) {
    typedef typename vx_elem<DT>::type E;
    const long long t = blockIdx.x;
    const long long id = vx_id_at(ids, id_bytes, t);
    const bool ok = id >= 0 && id < n_rows;
    if (id >= n_rows && status && threadIdx.x == 0) atomicOr(status, VX_STATUS_BAD_TOKEN);
    const E *src = (const E *)table + (ok ? id * stride : 0);
    E *dst = (E *)out + t * D;
    for (int c = threadIdx.x; c < D; c += 256) dst[c] = ok ? vx_store_cast<DT>((float)src[c] * scale) : (E)0.0f;
}

extern "C" int vx_embed_tokens(const void *d_ids, int id_bytes, int64_t n_tokens, const void *d_table, int64_t n_rows,
                               int D, int64_t table_stride, int dtype, float scale, void *d_out, int32_t *d_status,
                               void *stream) {
    if (!d_ids || !d_table || !d_out || n_tokens <= 0 || n_rows <= 0 || D <= 0 || table_stride < D) return VX_ERR_INVALID_ARG;
    if ((id_bytes != 4 && id_bytes != 8) || !vx_dtype_ok(dtype)) return VX_ERR_INVALID_ARG;
    if (n_tokens > VX_MAX_TOKENS || n_rows > VX_MAX_VOCAB || D > VX_MAX_TOKEN_WIDTH) return VX_ERR_UNSUPPORTED;
    const int es = vx_elem_size(dtype);
    if ((((uintptr_t)d_table | (uintptr_t)d_out) & (es - 1)) || ((uintptr_t)d_ids & (id_bytes - 1)) || ((uintptr_t)d_status & 3))
        return VX_ERR_ALIGNMENT;
    hipStream_t st = (hipStream_t)stream;
    vx_prof_begin(VX_PROF_EMBED, st);
    VX_DISPATCH_DTYPE(dtype, hipLaunchKernelGGL((vx_k_embed<DT>), dim3((unsigned)n_tokens), dim3(256), 0, st, d_ids, id_bytes,
                                                d_table, (long long)n_rows, D, (long long)table_stride, scale, d_out, d_status));
    vx_prof_end(VX_PROF_EMBED, st);
    return hipGetLastError() == hipSuccess ? VX_OK : VX_ERR_LAUNCH;
}

// One wave per (table row, 64 columns): the ids are scanned in order, so the sum has one order.
template <int GT, int TT>
__global__ __launch_bounds__(64) void vx_k_embed_grad(const void *__restrict__ ids, int id_bytes, long long T,
                                                      const void *__restrict__ grad, long long n_rows, int D, float scale,
                                                      void *__restrict__ out, int accumulate, int *__restrict__ status) {
    typedef typename vx_elem<GT>::type G;
    typedef typename vx_elem<TT>::type E;
    const long long v = blockIdx.x;
    const int lane = vx_lane(), c = blockIdx.y * 64 + lane;
    float sum = 0.f;
    bool any = false;
    for (long long t0 = 0; t0 < T; t0 += 64) {
        const long long id = t0 + lane < T ? vx_id_at(ids, id_bytes, t0 + lane) : -1;
        const bool hit = id == v;
        if (v == 0 && status && id >= n_rows) atomicOr(status, VX_STATUS_BAD_TOKEN);
        u64 m = __ballot(hit);
        while (m) {
            const long long t = t0 + __builtin_ctzll(m);
            m &= m - 1;
            any = true;
            if (c < D) sum += (float)((const G *)grad)[t * D + c];
        }
    }
    if (c >= D) return;
    E *dst = (E *)out + v * D + c;
    if (!accumulate) *dst = vx_store_cast<TT>(sum * scale);
    else if (any) *dst = vx_store_cast<TT>((float)*dst + sum * scale);
}

extern "C" size_t vx_embed_tokens_grad_workspace_bytes(int64_t n_tokens, int64_t n_rows, int D) {
    if (n_tokens <= 0 || n_rows <= 0 || D <= 0 || n_tokens > VX_MAX_TOKENS || n_rows > VX_MAX_VOCAB || D > VX_MAX_TOKEN_WIDTH) return 0;
    return 256;
}

extern "C" int vx_embed_tokens_grad(const void *d_ids, int id_bytes, int64_t n_tokens, const void *d_grad_out,
                                    int grad_dtype, int64_t n_rows, int D, float scale, void *d_grad_table,
                                    int table_dtype, int accumulate, int32_t *d_status, void *d_workspace,
                                    size_t workspace_bytes, void *stream) {
    if (!d_ids || !d_grad_out || !d_grad_table || !d_workspace || n_tokens <= 0 || n_rows <= 0 || D <= 0) return VX_ERR_INVALID_ARG;
    if ((id_bytes != 4 && id_bytes != 8) || !vx_dtype_ok(grad_dtype) || !vx_dtype_ok(table_dtype)) return VX_ERR_INVALID_ARG;
    if (n_tokens > VX_MAX_TOKENS || n_rows > VX_MAX_VOCAB || D > VX_MAX_TOKEN_WIDTH) return VX_ERR_UNSUPPORTED;
    if (table_dtype != grad_dtype && table_dtype != VX_DTYPE_F32) return VX_ERR_UNSUPPORTED;
    if (workspace_bytes < vx_embed_tokens_grad_workspace_bytes(n_tokens, n_rows, D)) return VX_ERR_WORKSPACE;
    if (((uintptr_t)d_grad_out & (vx_elem_size(grad_dtype) - 1)) || ((uintptr_t)d_grad_table & (vx_elem_size(table_dtype) - 1)) ||
        ((uintptr_t)d_ids & (id_bytes - 1)) || ((uintptr_t)d_status & 3) || ((uintptr_t)d_workspace & 255))
        return VX_ERR_ALIGNMENT;
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)n_rows, (unsigned)((D + 63) / 64));
    vx_prof_begin(VX_PROF_EMBED_GRAD, st);
    VX_DISPATCH_DTYPE(grad_dtype, {
        if (table_dtype == DT)
            hipLaunchKernelGGL((vx_k_embed_grad<DT, DT>), grid, dim3(64), 0, st, d_ids, id_bytes, (long long)n_tokens,
                               d_grad_out, (long long)n_rows, D, scale, d_grad_table, accumulate, d_status);
        else
            hipLaunchKernelGGL((vx_k_embed_grad<DT, VX_DTYPE_F32>), grid, dim3(64), 0, st, d_ids, id_bytes,
                               (long long)n_tokens, d_grad_out, (long long)n_rows, D, scale, d_grad_table, accumulate,
                               d_status);
    });
    vx_prof_end(VX_PROF_EMBED_GRAD, st);
    return hipGetLastError() == hipSuccess ? VX_OK : VX_ERR_LAUNCH;
}
