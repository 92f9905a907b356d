// Verification of drafted tokens against the target's distribution, from given uniform numbers.
// For sequence b with n_b drafts x_0 .. x_{n_b - 1}, target rows 0 .. n_b and draft rows 0 .. n_b - 1:
//   p_j = softmax(target[b,j] / T_b), q_j = softmax(draft[b,j] / T_b)  (no draft logits: q_j = 1 at x_j, 0 elsewhere)
//   accept[b,j] = min(1, p_j(x_j) / q_j(x_j));  x_j is accepted iff u_{b,j} q_j(x_j) < p_j(x_j) and all before it are
//   n = the number accepted; the token behind them is the first i with sum_{<=i} r > u_{b,K} sum r,
//       r = max(0, p_n - q_n) when a draft was rejected, r = p_n behind the last draft
// T_b not above 0: greedy (x_j is accepted iff it is the first arg-max of its row; the token behind is the arg-max).
// Exponentials, sums and the cumulative sum are fp64: the outcome is a whole number decided by where a cumulative sum
// passes a border, and one step of a flat distribution is 1/V.
#include "vx_dtype.h"
#include "vx_profile.h"

struct vx_verify_args {
    const void *target, *draft;
    long long t_seq, t_row, d_seq, d_row;         // strides in elements
    const long long *tokens;                      // [B, K]
    const int *lens;                              // [B] or nullptr
    const float *uniforms;                        // [B, K + 1]
    const float *temperature;                     // [B]
    int B, K, V;
};

struct vx_row_stat {                              // of one row of logits
    double z;                                     // sum of exp((x - m) / T)
    float m;                                      // largest logit
    int best;                                     // its first index
    int status;
    int pad;
};

__device__ __forceinline__ int vx_verify_len(const vx_verify_args &a, int b) {
    return a.lens ? vx_clamp_count(a.lens[b], a.K) : a.K;
}

// weight of a logit against the row's largest one; T > 0.  A masked (-inf) logit weighs 0 whatever T is.
__device__ __forceinline__ double vx_weight(float x, float m, double inv_t) {
    return x == -INFINITY ? 0.0 : exp(((double)x - (double)m) * inv_t);
}

// One workgroup per (sequence, row): target rows 0..K, then draft rows 0..K-1.
template <int DT>
__global__ __launch_bounds__(256) void vx_k_verify_stats(vx_verify_args a, vx_row_stat *__restrict__ stats) {
    typedef typename vx_elem<DT>::type E;
    __shared__ float s_m[4];
    __shared__ int s_i[4], s_bad[4];
    __shared__ double s_z[4];
    const int rows = 2 * a.K + 1, b = blockIdx.x / rows, j = blockIdx.x % rows, n = vx_verify_len(a, b);
    const bool is_draft = j > a.K;
    const float T = a.temperature[b];
    if (is_draft ? (!a.draft || j - a.K - 1 >= n || !(T > 0.f)) : j > n) return;
    const E *row = is_draft ? (const E *)a.draft + b * a.d_seq + (j - a.K - 1) * a.d_row : (const E *)a.target + b * a.t_seq + j * a.t_row;
    const int lane = vx_lane(), wave = threadIdx.x >> 6;
    float m = -INFINITY;
    int best = 0x7fffffff;
    bool bad = false;
    for (int i = threadIdx.x; i < a.V; i += 256) {
        const float x = (float)row[i];
        bad |= !(x < INFINITY);
        if (x > m) { m = x; best = i; }
    }
    for (int k = 32; k >= 1; k >>= 1) {
        const float om = __shfl_xor(m, k, VX_WAVE);
        const int oi = __shfl_xor(best, k, VX_WAVE);
        if (om > m || (om == m && oi < best)) { m = om; best = oi; }
    }
    const bool wbad = __any(bad);
    if (lane == 0) { s_m[wave] = m; s_i[wave] = best; s_bad[wave] = wbad; }
    __syncthreads();
    m = s_m[0]; best = s_i[0]; bad = s_bad[0];
    for (int w = 1; w < 4; ++w) {
        if (s_m[w] > m || (s_m[w] == m && s_i[w] < best)) { m = s_m[w]; best = s_i[w]; }
        bad |= s_bad[w];
    }
    const int status = bad ? VX_STATUS_NAN : (m == -INFINITY ? VX_STATUS_EMPTY_ROW : 0);
    double z = 0.0;
    if (!status && T > 0.f) {
        const double inv_t = 1.0 / (double)T;
        for (int i = threadIdx.x; i < a.V; i += 256) z += vx_weight((float)row[i], m, inv_t);
    }
    for (int k = 32; k >= 1; k >>= 1) z += __shfl_xor(z, k, VX_WAVE);
    if (lane == 0) s_z[wave] = z;
    __syncthreads();
    if (threadIdx.x == 0) {
        vx_row_stat r;
        r.z = (s_z[0] + s_z[1]) + (s_z[2] + s_z[3]);
        r.m = m; r.best = best; r.status = status; r.pad = 0;
        stats[blockIdx.x] = r;
    }
}

struct vx_choice {                                // what is left to do for a sequence
    int row;                                      // number of accepted drafts = the row that is drawn from
    int residual;                                 // 1: from max(0, p - q)
    int token;                                    // >= 0: known already (greedy); -1: draw; -2: none (invalid row)
};

// One thread per sequence.
template <int DT>
__global__ __launch_bounds__(64) void vx_k_verify_accept(vx_verify_args a, const vx_row_stat *__restrict__ stats,
                                                         vx_choice *__restrict__ choice, long long *__restrict__ out,
                                                         int *__restrict__ counts, float *__restrict__ accept,
                                                         int *__restrict__ status) {
    typedef typename vx_elem<DT>::type E;
    const int b = blockIdx.x * 64 + threadIdx.x;
    if (b >= a.B) return;
    const int n = vx_verify_len(a, b), K = a.K;
    const float T = a.temperature[b];
    const bool greedy = !(T > 0.f);
    const double inv_t = 1.0 / (double)T;
    const vx_row_stat *ts = stats + (long long)b * (2 * K + 1), *ds = ts + K + 1;
    int st = 0, acc = 0;
    bool going = true;
    for (int j = 0; j < n; ++j) {
        const long long x = a.tokens[(long long)b * K + j];
        const bool in = x >= 0 && x < a.V;
        double ratio = 0.0;
        bool ok = false;
        st |= ts[j].status | (in ? 0 : VX_STATUS_BAD_TOKEN);
        if (greedy) {
            ok = !ts[j].status && x == ts[j].best;
            ratio = ok ? 1.0 : 0.0;
        } else {
            const int dst = a.draft ? ds[j].status : 0;
            st |= dst;
            if (in && !ts[j].status && !dst) {
                const double p = vx_weight((float)((const E *)a.target)[b * a.t_seq + j * a.t_row + x], ts[j].m, inv_t) / ts[j].z;
                const double q = a.draft ? vx_weight((float)((const E *)a.draft)[b * a.d_seq + j * a.d_row + x], ds[j].m, inv_t) / ds[j].z : 1.0;
                ok = (double)a.uniforms[(long long)b * (K + 1) + j] * q < p;
                ratio = p >= q ? (p > 0.0 ? 1.0 : 0.0) : p / q;
            }
        }
        accept[(long long)b * K + j] = (float)ratio;
        going = going && ok;
        if (going) ++acc;
    }
    st |= ts[n].status;
    for (int j = n; j < K; ++j) accept[(long long)b * K + j] = 0.f;
    vx_choice c;
    c.row = acc;
    c.residual = acc < n;
    c.token = -1;
    if (ts[acc].status || (!greedy && acc < n && a.draft && ds[acc].status)) c.token = -2;
    else if (greedy) c.token = ts[acc].best;
    choice[b] = c;
    for (int j = 0; j <= K; ++j) out[(long long)b * (K + 1) + j] = j < acc ? a.tokens[(long long)b * K + j] : -1;
    if (c.token >= 0) out[(long long)b * (K + 1) + acc] = c.token;
    counts[b] = acc + 1;
    status[b] = st;
}

// One workgroup per sequence that still draws: the sum of the weights, then the place where the cumulative sum passes.
template <int DT>
__global__ __launch_bounds__(256) void vx_k_verify_draw(vx_verify_args a, const vx_row_stat *__restrict__ stats,
                                                        const vx_choice *__restrict__ choice, long long *__restrict__ out) {
    typedef typename vx_elem<DT>::type E;
    __shared__ double s_sum[257];
    __shared__ int s_last[256];
    const int b = blockIdx.x, K = a.K, tid = threadIdx.x;
    const vx_choice c = choice[b];
    if (c.token != -1) return;
    const int j = c.row;
    const vx_row_stat tr = stats[(long long)b * (2 * K + 1) + j];
    const E *row = (const E *)a.target + b * a.t_seq + j * a.t_row;
    const bool minus = c.residual && a.draft;
    const vx_row_stat dr = minus ? stats[(long long)b * (2 * K + 1) + K + 1 + j] : tr;
    const E *drow = minus ? (const E *)a.draft + b * a.d_seq + j * a.d_row : row;
    const long long drop = c.residual && !a.draft ? a.tokens[(long long)b * K + j] : -1;
    const double inv_t = 1.0 / (double)a.temperature[b];
    // each thread owns one contiguous piece of the row
    const int per = (a.V + 255) / 256, lo = min(a.V, tid * per), hi = min(a.V, lo + per);
    for (int only_p = 0; only_p < 2; ++only_p) {
        auto weight = [&](int i) -> double {
            if (i == drop && !only_p) return 0.0;
            const double p = vx_weight((float)row[i], tr.m, inv_t) / tr.z;
            if (!minus || only_p) return p;
            const double r = p - vx_weight((float)drow[i], dr.m, inv_t) / dr.z;
            return r > 0.0 ? r : 0.0;
        };
        double sum = 0.0;
        int last = -1;
        for (int i = lo; i < hi; ++i) {
            const double r = weight(i);
            sum += r;
            if (r > 0.0) last = i;
        }
        s_sum[tid] = sum;
        s_last[tid] = last;
        __syncthreads();
        if (tid == 0) {
            double run = 0.0;
            int l = -1;
            for (int t = 0; t < 256; ++t) {
                const double v = s_sum[t];
                s_sum[t] = run;
                run += v;
                l = max(l, s_last[t]);
            }
            s_sum[256] = run;
            s_last[0] = l;
        }
        __syncthreads();
        const double total = s_sum[256];
        if (!(total > 0.0)) { __syncthreads(); continue; }   // p and q alike to the last bit: draw from p
        const double goal = (double)a.uniforms[(long long)b * (K + 1) + K] * total;
        const bool none = !(goal < total);                    // a uniform of 1, or rounding: the last token with weight
        if (none) {
            if (tid == 0) out[(long long)b * (K + 1) + j] = s_last[0];
        } else if (hi > lo && s_sum[tid] <= goal && goal < s_sum[tid + 1]) {
            double run = s_sum[tid];
            int pick = -1;
            for (int i = lo; i < hi && pick < 0; ++i) {
                run += weight(i);
                if (run > goal) pick = i;
            }
            out[(long long)b * (K + 1) + j] = pick < 0 ? last : pick;
        }
        return;
    }
}

extern "C" size_t vx_verify_drafts_workspace_bytes(int B, int K, int V) {
    if (B <= 0 || K < 0 || V <= 0 || B > VX_MAX_VERIFY_BATCH || K > VX_MAX_DRAFTS || V > VX_MAX_VOCAB) return 0;
    return (((size_t)B * (2 * K + 1) * sizeof(vx_row_stat) + 255) & ~(size_t)255) + (((size_t)B * sizeof(vx_choice) + 255) & ~(size_t)255);
}

extern "C" int vx_verify_drafts(const void *d_target, int64_t target_seq_stride, int64_t target_row_stride, const void *d_draft,
                                int64_t draft_seq_stride, int64_t draft_row_stride, int dtype, const int64_t *d_draft_tokens,
                                const int32_t *d_draft_lens, const float *d_uniforms, const float *d_temperature, int B, int K,
                                int V, int64_t *d_tokens, int32_t *d_counts, float *d_accept, int32_t *d_status,
                                void *d_workspace, size_t workspace_bytes, void *stream) {
    if (!d_target || !d_uniforms || !d_temperature || !d_tokens || !d_counts || !d_status || !d_workspace || B <= 0 || K < 0 || V <= 0) return VX_ERR_INVALID_ARG;
    if ((K > 0 && (!d_draft_tokens || !d_accept)) || !vx_dtype_ok(dtype)) return VX_ERR_INVALID_ARG;
    if (target_row_stride < 0 || target_seq_stride < 0 || draft_row_stride < 0 || draft_seq_stride < 0) return VX_ERR_INVALID_ARG;
    if (B > VX_MAX_VERIFY_BATCH || K > VX_MAX_DRAFTS || V > VX_MAX_VOCAB) return VX_ERR_UNSUPPORTED;
    const int es = vx_elem_size(dtype);
    if ((((uintptr_t)d_target | (uintptr_t)d_draft) & (es - 1)) || (((uintptr_t)d_draft_tokens | (uintptr_t)d_tokens) & 7) ||
        (((uintptr_t)d_draft_lens | (uintptr_t)d_uniforms | (uintptr_t)d_temperature | (uintptr_t)d_counts | (uintptr_t)d_accept | (uintptr_t)d_status) & 3) ||
        ((uintptr_t)d_workspace & 255))
        return VX_ERR_ALIGNMENT;
    if (workspace_bytes < vx_verify_drafts_workspace_bytes(B, K, V)) return VX_ERR_WORKSPACE;
    vx_verify_args a = {d_target, d_draft, target_seq_stride, target_row_stride, draft_seq_stride, draft_row_stride,
                        (const long long *)d_draft_tokens, d_draft_lens, d_uniforms, d_temperature, B, K, V};
    vx_row_stat *stats = (vx_row_stat *)d_workspace;
    vx_choice *choice = (vx_choice *)((char *)d_workspace + (((size_t)B * (2 * K + 1) * sizeof(vx_row_stat) + 255) & ~(size_t)255));
    hipStream_t st = (hipStream_t)stream;
    vx_prof_begin(VX_PROF_VERIFY, st);
    VX_DISPATCH_DTYPE(dtype, {
        hipLaunchKernelGGL((vx_k_verify_stats<DT>), dim3((unsigned)(B * (2 * K + 1))), dim3(256), 0, st, a, stats);
        hipLaunchKernelGGL((vx_k_verify_accept<DT>), dim3((unsigned)((B + 63) / 64)), dim3(64), 0, st, a, stats, choice,
                           (long long *)d_tokens, d_counts, d_accept, d_status);
        hipLaunchKernelGGL((vx_k_verify_draw<DT>), dim3((unsigned)B), dim3(256), 0, st, a, stats, choice, (long long *)d_tokens);
    });
    vx_prof_end(VX_PROF_VERIFY, st);
    return hipGetLastError() == hipSuccess ? VX_OK : VX_ERR_LAUNCH;
}
