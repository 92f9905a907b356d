// Verification of drafted tokens against the target's distribution, from given uniform numbers.
// For sequence b with n_b drafts x_0 .. x_{n_b - 1}, target rows 0 .. n_b and draft rows 0 .. n_b - 1:
//   p_j = softmax(target[b,j] / T_b), q_j = softmax(draft[b,j] / T_b)  (no draft logits: q_j = 1 at x_j, 0 elsewhere)
//   accept[b,j] = min(1, p_j(x_j) / q_j(x_j));  x_j is accepted iff u_{b,j} q_j(x_j) < p_j(x_j) and all before it are
//   n = the number accepted; the token behind them is the first i with sum_{<=i} r > u_{b,K} sum r,
//       r = max(0, p_n - q_n) when a draft was rejected, r = p_n behind the last draft
// T_b not above 0: greedy (x_j is accepted iff it is the first arg-max of its row; the token behind is the arg-max).
//
// Launches over chunks of the vocabulary:
//   stats   every used row: largest logit and fp32 sum of exponentials of each quarter of a chunk (bound by the one read of the logits;
//           fp64 exponentials here would take twice the time of the read)
//   choose  the accepted drafts and the row to draw from; that row's (and the draft row's) sums again in fp64, of each quarter
//   rest    (with draft logits) that row's sums of max(0, p - q), fp64, of each quarter
//   draw    the token, one workgroup a sequence
// The token that is drawn is a whole number, decided by where a cumulative sum passes a border, and one step of a flat
// distribution is 1/V: everything it depends on is fp64.  How far the sums of the first launch are off, u = 2^-24:
//   a weight is the product of two exponentials (of its wave's largest logit against the row's, of its own against the
//   wave's), each off by 2 u (the instruction) + ln2 |t| 3 u (difference, factor, product), t its exponent to base 2;
//   weighted with the distribution the two |t| together average at most log2 V (the entropy less log2 of the sum);
//   the product 1 u, and 16 fp32 additions that follow one another (the rest are fp64):  (21 + 2.1 log2 V) u
// So a test u q < p, with two such sums, is taken from them unless its sides are within (42 + 4.2 log2 V) u of each other
// (6.8e-6 at V = 131072); then both rows are summed in fp64.
#include "vx_dtype.h"
#include "vx_profile.h"

struct vx_verify_args {
    const void *target, *draft;
    long long t_seq, t_row, d_seq, d_row;         // strides in elements
    const long long *tokens;                      // [B, K]
    const int *lens;                              // [B] or nullptr
    const float *uniforms;                        // [B, K + 1]
    const float *temperature;                     // [B] or nullptr: one_temperature
    float one_temperature;
    int B, K, V, chunks;
    // workspace
    float2 *stats;                                // [B][2 K + 1][4 chunks], for each wave: largest logit (NaN: an invalid one), sum (greedy: its index)
    double2 *z;                                   // [B][4 chunks]: sums of the row that is drawn from, target and draft, of each quarter of a chunk
    double *r;                                    // [B][4 chunks]: sums of max(0, p - q)
    struct vx_choice *choice;                     // [B]
    // outputs
    long long *out;                               // [B, K + 1]
    int *counts, *status;
    float *accept;
};

struct vx_choice {                                // what is left to do for a sequence
    int row;                                      // number of accepted drafts = the row that is drawn from
    int mode;                                     // 0: the token is known or there is none; 1: from p; 2: from p without `drop`; 3: from max(0, p - q)
    float mp, mq;                                 // largest logits of the two rows
    long long drop;
};

// chunk of a row: 256 threads x U pieces of 16 bytes
#define VX_VERIFY_U 4
// (256 threads x one piece in the draw: a quarter of it)
template <int DT> __host__ __device__ constexpr int vx_verify_chunk() { return 256 * VX_VERIFY_U * 16 / (int)sizeof(typename vx_elem<DT>::type); }

__device__ __forceinline__ int vx_verify_len(const vx_verify_args &a, int b) {
    return a.lens ? vx_clamp_count(a.lens[b], a.K) : a.K;
}
__device__ __forceinline__ float vx_verify_t(const vx_verify_args &a, int b) { return a.temperature ? a.temperature[b] : a.one_temperature; }
template <int DT>
__device__ __forceinline__ const typename vx_elem<DT>::type *vx_verify_target(const vx_verify_args &a, int b, int j) {
    return (const typename vx_elem<DT>::type *)a.target + b * a.t_seq + j * a.t_row;
}
template <int DT>
__device__ __forceinline__ const typename vx_elem<DT>::type *vx_verify_draft(const vx_verify_args &a, int b, int j) {
    return (const typename vx_elem<DT>::type *)a.draft + b * a.d_seq + j * a.d_row;
}

// 2^t for t <= 0: t = n + f, |f| <= 1/2, and the series of e^(f ln 2) up to its 12th term (the 13th is below 2e-16).
// 0 from t = -1023 down, and for the NaN of -inf * 0 (a masked logit at an infinite temperature).
__device__ __forceinline__ double vx_exp2_64(double t) {
    constexpr double L = 0.69314718055994530942;
    // 1.5 * 2^52 moves t's integer part into the low bits of the sum (the conversions and ldexp run at a quarter of the rate)
    constexpr double SHIFT = 6755399441055744.0;
    const double moved = fmax(t, -1100.0) + SHIFT, f = fmax(t, -1100.0) - (moved - SHIFT);
    const int n = __double2loint(moved);
    double p = L * L * L * L * L * L * L * L * L * L * L * L / 479001600.0;
    p = __builtin_fma(p, f, L * L * L * L * L * L * L * L * L * L * L / 39916800.0);
    p = __builtin_fma(p, f, L * L * L * L * L * L * L * L * L * L / 3628800.0);
    p = __builtin_fma(p, f, L * L * L * L * L * L * L * L * L / 362880.0);
    p = __builtin_fma(p, f, L * L * L * L * L * L * L * L / 40320.0);
    p = __builtin_fma(p, f, L * L * L * L * L * L * L / 5040.0);
    p = __builtin_fma(p, f, L * L * L * L * L * L / 720.0);
    p = __builtin_fma(p, f, L * L * L * L * L / 120.0);
    p = __builtin_fma(p, f, L * L * L * L / 24.0);
    p = __builtin_fma(p, f, L * L * L / 6.0);
    p = __builtin_fma(p, f, L * L * 0.5);
    p = __builtin_fma(p, f, L);
    p = __builtin_fma(p, f, 1.0);
    return p * __hiloint2double(max(n + 1023, 0) << 20, 0);        // 2^n, and 0 from n = -1023 down
}
// weight of a logit against the row's largest one; c = log2(e) / T
__device__ __forceinline__ double vx_weight(float x, float m, double c) {
    return vx_exp2_64(((double)x - (double)m) * c);
}
__device__ __forceinline__ double vx_verify_c(float T) { return 1.44269504088896340736 / (double)T; }

// the same in fp32; finite and not 0, so that the product with a masked logit is -inf at any temperature
__device__ __forceinline__ float vx_verify_c32(float T) { return fminf(fmaxf((float)vx_verify_c(T), 1e-45f), 3e38f); }

// the thread's values of a chunk, -inf where the row has ended: pieces of 16 bytes, the lanes side by side.  QUARTERS: each wave has
// its own quarter of the chunk; otherwise the waves' pieces alternate (statistics of 185 MB: 37 against 32 us)
template <bool QUARTERS>
__device__ __forceinline__ int vx_verify_piece(int u) {
    return QUARTERS ? ((int)(threadIdx.x >> 6) * VX_VERIFY_U + u) * 64 + vx_lane() : u * 256 + (int)threadIdx.x;
}
template <int DT, bool QUARTERS>
__device__ __forceinline__ void vx_verify_load(const typename vx_elem<DT>::type *row, int c0, int V,
                                               float x[VX_VERIFY_U * 16 / sizeof(typename vx_elem<DT>::type)]) {
    constexpr int VEC = 16 / sizeof(typename vx_elem<DT>::type);
    vx_vec<DT> v[VX_VERIFY_U];
    if (c0 + vx_verify_chunk<DT>() <= V) {
#pragma unroll
        for (int u = 0; u < VX_VERIFY_U; ++u) v[u].raw = vx_load16<DT>(row + c0 + vx_verify_piece<QUARTERS>(u) * VEC);
#pragma unroll
        for (int u = 0; u < VX_VERIFY_U; ++u)
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[u * VEC + k] = (float)v[u].e[k];
    } else {
#pragma unroll
        for (int u = 0; u < VX_VERIFY_U; ++u) {
            const int at = c0 + vx_verify_piece<QUARTERS>(u) * VEC;
            v[u] = vx_load_vec<DT>(row + at, V - at);
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[u * VEC + k] = at + k < V ? (float)v[u].e[k] : -INFINITY;
        }
    }
}

// One workgroup per (sequence, row, chunk): target rows 0..K, then draft rows 0..K-1.  Each wave leaves its own statistics: no
// barrier between a workgroup's loads and its end (185 MB in 32 us at 64 x 11 rows of 131072 bf16).
template <int DT>
__global__ __launch_bounds__(256) void vx_k_verify_stats(vx_verify_args a) {
    constexpr int VEC = 16 / sizeof(typename vx_elem<DT>::type), PER = VX_VERIFY_U * VEC;
    const int rows = a.draft ? 2 * a.K + 1 : a.K + 1;
    const int item = vx_block() / a.chunks, chunk = vx_block() - item * a.chunks;
    const int b = item / rows, j = item - b * rows;
    if (b >= a.B) return;
    const int n = vx_verify_len(a, b);
    const bool is_draft = j > a.K;
    const float T = vx_verify_t(a, b);
    const bool greedy = !(T > 0.f);
    if (is_draft ? (j - a.K - 1 >= n || greedy) : j > n) return;
    float x[PER];
    const int c0 = chunk * vx_verify_chunk<DT>();
    vx_verify_load<DT, false>(is_draft ? vx_verify_draft<DT>(a, b, j - a.K - 1) : vx_verify_target<DT>(a, b, j), c0, a.V, x);
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < PER; ++k) m = fmaxf(m, x[k]);
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) m = fmaxf(m, __shfl_xor(m, k, VX_WAVE));
    bool bad = false;
    float z = 0.f;
    int best = 0x7fffffff;
    if (greedy) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int i = c0 + vx_verify_piece<false>(k / VEC) * VEC + k % VEC;
            bad |= !(x[k] < INFINITY);
            if (x[k] == m) best = min(best, i);
        }
        bad = __any(bad);
#pragma unroll
        for (int k = 32; k >= 1; k >>= 1) best = min(best, __shfl_xor(best, k, VX_WAVE));
    } else {
        // A NaN or +inf makes the sum NaN by itself, and nothing else does: the subtrahend is finite.
        const float c = vx_verify_c32(T), top = m == -INFINITY ? 0.f : m;
        float part[4] = {};
#pragma unroll
        for (int k = 0; k < PER; ++k) part[k & 3] += __builtin_amdgcn_exp2f((x[k] - top) * c);
        z = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
        for (int k = 32; k >= 1; k >>= 1) z += __shfl_xor(z, k, VX_WAVE);
        bad = z != z;
    }
    if (vx_lane() == 0)
        a.stats[(((long long)b * (2 * a.K + 1) + j) * a.chunks + chunk) * 4 + (threadIdx.x >> 6)] =
            float2{bad ? __builtin_nanf("") : m, greedy ? __int_as_float(best) : z};
}

__device__ __forceinline__ double vx_verify_wave_sum(double v) {
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) v += __shfl_xor(v, k, VX_WAVE);
    return v;
}
// sum over the workgroup's 256 threads, in one order; every thread gets it
__device__ __forceinline__ double vx_verify_sum(double v, double *s_sum) {
    v = vx_verify_wave_sum(v);
    __syncthreads();
    if (vx_lane() == 0) s_sum[threadIdx.x >> 6] = v;
    __syncthreads();
    return (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
}

// this thread's part of a chunk's sum of weights
template <int DT>
__device__ __forceinline__ double vx_verify_chunk_sum(const typename vx_elem<DT>::type *row, int chunk, int V, float m, double c) {
    constexpr int PER = VX_VERIFY_U * 16 / sizeof(typename vx_elem<DT>::type);
    float x[PER];
    vx_verify_load<DT, true>(row, chunk * vx_verify_chunk<DT>(), V, x);
    double z = 0.0;
#pragma unroll
    for (int k = 0; k < PER; ++k) z += vx_weight(x[k], m, c);
    return z;
}

// One workgroup per (sequence, chunk).  Each takes the decision of its sequence by itself (a few KB of statistics); the first
// one of a sequence also writes it down.
template <int DT>
__global__ __launch_bounds__(256) void vx_k_verify_choose(vx_verify_args a) {
    __shared__ double s_z[2 * VX_MAX_DRAFTS + 1], s_sum[4];
    __shared__ float s_m[2 * VX_MAX_DRAFTS + 1];
    __shared__ int s_best[VX_MAX_DRAFTS + 1];
    __shared__ u64 s_ok, s_unsure;
    const int b = vx_block() / a.chunks, chunk = vx_block() - b * a.chunks, K = a.K;
    if (b >= a.B) return;
    const int n = vx_verify_len(a, b);
    const int lane = vx_lane(), w = threadIdx.x >> 6;
    const float T = vx_verify_t(a, b);
    const bool greedy = !(T > 0.f), has_q = a.draft && !greedy;
    const double c = vx_verify_c(T);
    // lane j of the first wave decides on draft j; what it needs is on its way while the rows are summed
    long long x = 0;
    float tx = 0.f, dx = 0.f, un = 0.f;
    bool in = false;
    if (w == 0 && lane < n) {
        x = a.tokens[(long long)b * K + lane];
        un = a.uniforms[(long long)b * (K + 1) + lane];
        in = x >= 0 && x < a.V;
        if (in) tx = (float)vx_verify_target<DT>(a, b, lane)[x];
        if (in && has_q) dx = (float)vx_verify_draft<DT>(a, b, lane)[x];
    }
    // largest logit and sum of each row: 16 lanes a row, over its chunks
    for (int i0 = 0; i0 < (has_q ? 2 * n + 1 : n + 1); i0 += 16) {
        const int i = i0 + (threadIdx.x >> 4), sub = lane & 15;
        const bool row = i < (has_q ? 2 * n + 1 : n + 1);
        const int j = i <= n ? i : K + 1 + (i - n - 1);           // row of the statistics
        const float2 *st = a.stats + ((long long)b * (2 * K + 1) + j) * a.chunks * 4;
        float m = -INFINITY;
        bool bad = false;
        float2 v[4];                                              // the first 64 of the row's statistics
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = row && sub + 16 * k < a.chunks * 4 ? st[sub + 16 * k] : float2{-INFINITY, 0.f};
        auto look = [&](float x) {
            bad |= x != x;
            m = fmaxf(m, x);
        };
#pragma unroll
        for (int k = 0; k < 4; ++k) look(v[k].x);
        if (row)
            for (int k = sub + 64; k < a.chunks * 4; k += 16) look(st[k].x);
#pragma unroll
        for (int k = 8; k >= 1; k >>= 1) m = fmaxf(m, __shfl_xor(m, k, VX_WAVE));
        bad = (__ballot(bad) >> (lane & 48)) & 0xffff;
        double z = 0.0;
        int best = 0x7fffffff;
        const float c32 = vx_verify_c32(T), top = m == -INFINITY ? 0.f : m;
        auto join = [&](float2 x) {
            if (greedy) best = x.x == m ? min(best, __float_as_int(x.y)) : best;
            else z += (double)(x.y * __builtin_amdgcn_exp2f((x.x - top) * c32));
        };
#pragma unroll
        for (int k = 0; k < 4; ++k) join(v[k]);
        if (row)
            for (int k = sub + 64; k < a.chunks * 4; k += 16) join(st[k]);
#pragma unroll
        for (int k = 8; k >= 1; k >>= 1) {
            z += __shfl_xor(z, k, VX_WAVE);
            best = min(best, __shfl_xor(best, k, VX_WAVE));
        }
        if (row && sub == 0) {
            const int at = i <= n ? i : VX_MAX_DRAFTS + 1 + (i - n - 1);
            s_m[at] = bad ? __builtin_nanf("") : m;
            s_z[at] = z;
            if (i <= n) s_best[i] = best;
        }
    }
    __syncthreads();
    auto invalid = [](float m) { return m != m ? VX_STATUS_NAN : (m == -INFINITY ? VX_STATUS_EMPTY_ROW : 0); };
    double ratio = 0.0, p = 0.0, q = 1.0;
    auto accept = [&] { return p >= q ? (p > 0.0 ? 1.0 : 0.0) : p / q; };
    int st = 0;
    if (w == 0) {
        bool ok = false, unsure = false;
        if (lane < n) {
            const int t_bad = invalid(s_m[lane]), q_bad = has_q ? invalid(s_m[VX_MAX_DRAFTS + 1 + lane]) : 0;
            st = t_bad | q_bad | (in ? 0 : VX_STATUS_BAD_TOKEN);
            if (in && !t_bad && !q_bad) {
                if (greedy) {
                    ok = s_best[lane] == x;
                    ratio = ok ? 1.0 : 0.0;
                } else {
                    p = vx_weight(tx, s_m[lane], c) / s_z[lane];
                    if (has_q) q = vx_weight(dx, s_m[VX_MAX_DRAFTS + 1 + lane], c) / s_z[VX_MAX_DRAFTS + 1 + lane];
                    const double uq = (double)un * q;
                    ok = uq < p;
                    unsure = p > 0.0 && fabs(uq - p) <= p * ((42.0 + 4.2 * (32 - __clz(a.V))) * 0x1p-24);
                    ratio = accept();
                }
            }
        }
        const u64 oks = __ballot(ok), maybe = __ballot(unsure), sure_no = __ballot(lane < n && !ok && !unsure);
        if (lane == 0) {
            s_ok = oks;
            s_unsure = maybe & (sure_no ? (sure_no & (0 - sure_no)) - 1 : ~0ull);     // those in front of the first certain rejection
        }
    }
    __syncthreads();
    for (u64 left = s_unsure; left; left &= left - 1) {
        const int j = __builtin_ctzll(left);
        double zp = 0.0, zq = 0.0;
        for (int k = 0; k < a.chunks; ++k) zp += vx_verify_chunk_sum<DT>(vx_verify_target<DT>(a, b, j), k, a.V, s_m[j], c);
        if (has_q)
            for (int k = 0; k < a.chunks; ++k) zq += vx_verify_chunk_sum<DT>(vx_verify_draft<DT>(a, b, j), k, a.V, s_m[VX_MAX_DRAFTS + 1 + j], c);
        zp = vx_verify_sum(zp, s_sum);
        zq = vx_verify_sum(zq, s_sum);
        if (threadIdx.x == j) {                                   // p and q from the exact sums
            p = p * s_z[j] / zp;
            if (has_q) q = q * s_z[VX_MAX_DRAFTS + 1 + j] / zq;
            s_ok = (double)un * q < p ? s_ok | (1ull << j) : s_ok & ~(1ull << j);
            ratio = accept();
        }
        __syncthreads();
    }
    const u64 no = ~s_ok;
    const int acc = min(n, no ? (int)__builtin_ctzll(no) : 64);
    const int row_bad = invalid(s_m[acc]), q_bad = has_q && acc < n ? invalid(s_m[VX_MAX_DRAFTS + 1 + acc]) : 0;
    const int mode = row_bad || q_bad || greedy ? 0 : (acc == n ? 1 : (a.draft ? 3 : 2));
    const int known = greedy && !row_bad ? s_best[acc] : -1;      // the drawn token comes with the next launch
    if (chunk == 0 && w == 0) {
        if (lane < K) {
            a.accept[(long long)b * K + lane] = lane < n ? (float)ratio : 0.f;
            a.out[(long long)b * (K + 1) + lane] = lane < acc ? x : (lane == acc ? known : -1);
        }
#pragma unroll
        for (int k = 32; k >= 1; k >>= 1) st |= __shfl_xor(st, k, VX_WAVE);
        if (lane == 0) {
            vx_choice ch;
            ch.row = acc; ch.mode = mode; ch.mp = s_m[acc];
            ch.mq = mode == 3 ? s_m[VX_MAX_DRAFTS + 1 + acc] : 0.f;
            ch.drop = mode == 2 ? a.tokens[(long long)b * K + acc] : -1;
            a.choice[b] = ch;
            a.counts[b] = acc + 1;
            a.status[b] = st | invalid(s_m[n]);
            a.out[(long long)b * (K + 1) + K] = acc == K ? known : -1;
        }
    }
    if (mode == 0) return;
    const double zp = vx_verify_wave_sum(vx_verify_chunk_sum<DT>(vx_verify_target<DT>(a, b, acc), chunk, a.V, s_m[acc], c));
    const double zq = mode == 3 ? vx_verify_wave_sum(vx_verify_chunk_sum<DT>(vx_verify_draft<DT>(a, b, acc), chunk, a.V, s_m[VX_MAX_DRAFTS + 1 + acc], c)) : 0.0;
    if (lane == 0) a.z[((long long)b * a.chunks + chunk) * 4 + w] = double2{zp, zq};
}

struct vx_pick_smem {
    double run[4], before;
    int first, last;
};

// Thread t holds the weight `sum` of the t-th of up to 256 parts: the first part with a weight at which the running weight, from
// `base` on, passes `goal`, and the weight in front of it; -1 where none does.  `last`: the last part with a weight (-1: none).
// Each running weight has its own order of additions, so one may pass that only adds nothing to the one before it, which did not:
// parts without a weight are never taken.
__device__ __forceinline__ int vx_pick_part(double sum, double base, double goal, vx_pick_smem &S, double &before, int &last) {
    const int lane = vx_lane(), w = threadIdx.x >> 6;
    double run = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(run, d, VX_WAVE);
        if (lane >= d) run += o;
    }
    __syncthreads();
    if (lane == 63) S.run[w] = run;
    if (threadIdx.x == 0) { S.first = 256; S.last = -1; }
    __syncthreads();
    double front = base;
    for (int i = 0; i < w; ++i) front += S.run[i];
    run += front;
    const double prev = __shfl_up(run, 1, VX_WAVE);
    const u64 passed = __ballot(run > goal && sum > 0.0), any = __ballot(sum > 0.0);
    if (lane == 0) {
        if (passed) atomicMin(&S.first, w * 64 + __builtin_ctzll(passed));
        if (any) atomicMax(&S.last, w * 64 + 63 - __builtin_clzll(any));
    }
    __syncthreads();
    const int first = S.first;
    last = S.last;
    if ((int)threadIdx.x == first) S.before = lane ? prev : front;
    __syncthreads();
    before = S.before;
    return first < 256 ? first : -1;
}

// The first i whose cumulative weight passes u * total; `sums(k)` the weight of the k-th run of RUN tokens, `weight(i)` of one
// token, `part(i)` of the RUN / 256 tokens from i on.  One workgroup: first the run, then the 1/256 of it, then the token; where
// rounding leaves none, the last one with a weight.  -1 where no token has a weight.
template <int RUN, class S, class P, class W>
__device__ __forceinline__ int vx_verify_pick(int runs, int V, float u, S sums, P part_weight, W weight, vx_pick_smem &sm, double *s_sum) {
    constexpr int PART = RUN / 256;
    const int tid = threadIdx.x, per = (runs + 255) / 256;        // runs of one thread
    double mine = 0.0, before;
    int last;
    for (int k = tid * per; k < min(runs, (tid + 1) * per); ++k) mine += sums(k);
    // a uniform of 1 and above (or NaN) is behind all running sums, whatever they are rounded to
    double goal = u < 1.f ? (double)u * vx_verify_sum(mine, s_sum) : INFINITY;
    int part = vx_pick_part(mine, 0.0, goal, sm, before, last);
    if (last < 0) return -1;
    if (part < 0) { part = last; goal = INFINITY; before = 0.0; }
    int run = part * per;
    if (per > 1) {                                                // more than 256 runs: on through this thread's
        bool passed = false;
        for (int k = part * per; k < min(runs, (part + 1) * per) && !passed; ++k) {
            const double v = sums(k);
            if (!(v > 0.0)) continue;
            run = k;
            passed = before + v > goal;
            if (!passed) before += v;
        }
        if (!passed) goal = INFINITY;                             // rounding: `before` holds the last run already
    }
    mine = part_weight(run * RUN + tid * PART);
    part = vx_pick_part(mine, before, goal, sm, before, last);
    if (part < 0) { part = max(last, 0); goal = INFINITY; }
    const int i = run * RUN + part * PART + tid;
    part = vx_pick_part(tid < PART && i < V ? weight(i) : 0.0, before, goal, sm, before, last);
    return i - tid + (part < 0 ? max(last, 0) : part);
}

// r of one token from its two logits; ip, iq: the inverse sums of the rows
__device__ __forceinline__ double vx_verify_rest(float x, float y, const vx_choice &ch, double c, double ip, double iq) {
    const double r = vx_weight(x, ch.mp, c) * ip - vx_weight(y, ch.mq, c) * iq;
    return r > 0.0 ? r : 0.0;
}
// sums of the two rows over all chunks, in the same order wherever they are needed
__device__ __forceinline__ double2 vx_verify_totals(const vx_verify_args &a, int b, double *s_sum) {
    double zp = 0.0, zq = 0.0;
    for (int k = threadIdx.x; k < a.chunks * 4; k += 256) {
        const double2 v = a.z[(long long)b * a.chunks * 4 + k];
        zp += v.x;
        zq += v.y;
    }
    zp = vx_verify_sum(zp, s_sum);
    return double2{zp, vx_verify_sum(zq, s_sum)};
}

// Sums of max(0, p - q): one workgroup per (sequence, chunk).
template <int DT>
__global__ __launch_bounds__(256) void vx_k_verify_rest(vx_verify_args a) {
    constexpr int CHUNK = vx_verify_chunk<DT>(), PER = VX_VERIFY_U * 16 / sizeof(typename vx_elem<DT>::type);
    __shared__ double s_sum[4];
    const int b = vx_block() / a.chunks, chunk = vx_block() - b * a.chunks;
    if (b >= a.B) return;
    const vx_choice ch = a.choice[b];
    if (ch.mode != 3) return;
    float x[PER], y[PER];
    vx_verify_load<DT, true>(vx_verify_target<DT>(a, b, ch.row), chunk * CHUNK, a.V, x);
    vx_verify_load<DT, true>(vx_verify_draft<DT>(a, b, ch.row), chunk * CHUNK, a.V, y);
    const double c = vx_verify_c(vx_verify_t(a, b));
    const double2 z = vx_verify_totals(a, b, s_sum);
    const double ip = 1.0 / z.x, iq = 1.0 / z.y;
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < PER; ++k) sum += vx_verify_rest(x[k], y[k], ch, c, ip, iq);
    sum = vx_verify_wave_sum(sum);
    if (vx_lane() == 0) a.r[((long long)b * a.chunks + chunk) * 4 + (threadIdx.x >> 6)] = sum;
}

// The drawn token: one workgroup per sequence.
template <int DT>
__global__ __launch_bounds__(256) void vx_k_verify_draw(vx_verify_args a) {
    constexpr int RUN = vx_verify_chunk<DT>() / 4, PER = RUN / 256;
    __shared__ double s_sum[4];
    __shared__ vx_pick_smem sm;
    const int b = blockIdx.x, runs = a.chunks * 4;
    const vx_choice ch = a.choice[b];
    const float u = a.uniforms[(long long)b * (a.K + 1) + a.K];
    const double c = vx_verify_c(vx_verify_t(a, b));
    if (ch.mode == 0) return;
    const typename vx_elem<DT>::type *trow = vx_verify_target<DT>(a, b, ch.row);
    const double2 *z = a.z + (long long)b * runs;
    auto from_p = [&](long long drop) {
        auto one = [&](int i) { return i == drop ? 0.0 : vx_weight((float)trow[i], ch.mp, c); };
        auto part = [&](int i) {                                  // the PER tokens from i on
            const vx_vec<DT> x = vx_load_vec<DT>(trow + i, a.V - i);
            double sum = 0.0;
#pragma unroll
            for (int k = 0; k < PER; ++k) sum += i + k >= a.V || i + k == drop ? 0.0 : vx_weight((float)x.e[k], ch.mp, c);
            return sum;
        };
        // a run that loses a token is summed again: its sum less the token's weight could be all rounding
        const int drop_run = drop >= 0 && drop < a.V ? (int)(drop / RUN) : -1;
        const double again = drop_run >= 0 ? vx_verify_sum(part(drop_run * RUN + threadIdx.x * PER), s_sum) : 0.0;
        return vx_verify_pick<RUN>(runs, a.V, u, [&](int k) { return k == drop_run ? again : z[k].x; }, part, one, sm, s_sum);
    };
    int i;
    if (ch.mode == 3) {
        const typename vx_elem<DT>::type *drow = vx_verify_draft<DT>(a, b, ch.row);
        const double2 t = vx_verify_totals(a, b, s_sum);
        const double ip = 1.0 / t.x, iq = 1.0 / t.y, *r = a.r + (long long)b * runs;
        auto one = [&](int k) { return vx_verify_rest((float)trow[k], (float)drow[k], ch, c, ip, iq); };
        auto part = [&](int i) {
            const vx_vec<DT> x = vx_load_vec<DT>(trow + i, a.V - i), y = vx_load_vec<DT>(drow + i, a.V - i);
            double sum = 0.0;
#pragma unroll
            for (int k = 0; k < PER; ++k) sum += i + k >= a.V ? 0.0 : vx_verify_rest((float)x.e[k], (float)y.e[k], ch, c, ip, iq);
            return sum;
        };
        i = vx_verify_pick<RUN>(runs, a.V, u, [&](int k) { return r[k]; }, part, one, sm, s_sum);
    } else {
        i = from_p(ch.drop);
    }
    if (i < 0) i = from_p(-1);                                    // p and q alike to the last bit; nothing but the rejected token
    if (threadIdx.x == 0) a.out[(long long)b * (a.K + 1) + ch.row] = i;
}

struct vx_verify_plan {
    int chunks;
    size_t stats, z, r, choice, total;
};

static vx_verify_plan vx_verify_make_plan(int B, int K, int V, int chunk) {
    vx_verify_plan p;
    p.chunks = (V + chunk - 1) / chunk;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += (n + 255) & ~(size_t)255; return o; };
    p.stats = take((size_t)B * (2 * K + 1) * p.chunks * 4 * sizeof(float2));
    p.z = take((size_t)B * p.chunks * 4 * sizeof(double2));
    p.r = take((size_t)B * p.chunks * 4 * sizeof(double));
    p.choice = take((size_t)B * sizeof(vx_choice));
    p.total = at;
    return p;
}

extern "C" size_t vx_verify_drafts_workspace_bytes(int B, int K, int V) {
    if (B <= 0 || K < 0 || V <= 0 || B > VX_MAX_VERIFY_BATCH || K > VX_MAX_DRAFTS || V > VX_MAX_VOCAB) return 0;
    return vx_verify_make_plan(B, K, V, vx_verify_chunk<VX_DTYPE_F32>()).total;      // the smallest chunk
}

extern "C" int vx_verify_drafts(const void *d_target, int64_t target_seq_stride, int64_t target_row_stride, const void *d_draft,
                                int64_t draft_seq_stride, int64_t draft_row_stride, int dtype, const int64_t *d_draft_tokens,
                                const int32_t *d_draft_lens, const float *d_uniforms, const float *d_temperature, float temperature,
                                int B, int K, int V, int64_t *d_tokens, int32_t *d_counts, float *d_accept, int32_t *d_status,
                                void *d_workspace, size_t workspace_bytes, void *stream) {
    if (!d_target || !d_uniforms || !d_tokens || !d_counts || !d_status || !d_workspace || B <= 0 || K < 0 || V <= 0) return VX_ERR_INVALID_ARG;
    if ((K > 0 && (!d_draft_tokens || !d_accept)) || !vx_dtype_ok(dtype)) return VX_ERR_INVALID_ARG;
    if (target_row_stride < 0 || target_seq_stride < 0 || draft_row_stride < 0 || draft_seq_stride < 0) return VX_ERR_INVALID_ARG;
    if (B > VX_MAX_VERIFY_BATCH || K > VX_MAX_DRAFTS || V > VX_MAX_VOCAB) return VX_ERR_UNSUPPORTED;
    const int es = vx_elem_size(dtype);
    if ((((uintptr_t)d_target | (uintptr_t)d_draft) & (es - 1)) || (((uintptr_t)d_draft_tokens | (uintptr_t)d_tokens) & 7) ||
        (((uintptr_t)d_draft_lens | (uintptr_t)d_uniforms | (uintptr_t)d_temperature | (uintptr_t)d_counts | (uintptr_t)d_accept | (uintptr_t)d_status) & 3) ||
        ((uintptr_t)d_workspace & 255))
        return VX_ERR_ALIGNMENT;
    if (workspace_bytes < vx_verify_drafts_workspace_bytes(B, K, V)) return VX_ERR_WORKSPACE;
    if (K == 0) d_draft = nullptr;
    const vx_verify_plan p = vx_verify_make_plan(B, K, V, es == 4 ? vx_verify_chunk<VX_DTYPE_F32>() : vx_verify_chunk<VX_DTYPE_F16>());
    const int64_t blocks = (int64_t)B * (d_draft ? 2 * K + 1 : K + 1) * p.chunks;
    if (blocks > 2147483647LL) return VX_ERR_UNSUPPORTED;
    char *ws = (char *)d_workspace;
    const vx_verify_args a = {d_target, d_draft, target_seq_stride, target_row_stride, draft_seq_stride, draft_row_stride,
                              (const long long *)d_draft_tokens, d_draft_lens, d_uniforms, d_temperature, temperature, B, K, V, p.chunks,
                              (float2 *)(ws + p.stats), (double2 *)(ws + p.z), (double *)(ws + p.r), (vx_choice *)(ws + p.choice),
                              (long long *)d_tokens, d_counts, d_status, d_accept};
    hipStream_t st = (hipStream_t)stream;
    vx_prof_begin(VX_PROF_VERIFY, st);
    VX_DISPATCH_DTYPE(dtype, {
        hipLaunchKernelGGL((vx_k_verify_stats<DT>), vx_grid(blocks), dim3(256), 0, st, a);
        hipLaunchKernelGGL((vx_k_verify_choose<DT>), vx_grid((int64_t)B * p.chunks), dim3(256), 0, st, a);
        if (d_draft) hipLaunchKernelGGL((vx_k_verify_rest<DT>), vx_grid((int64_t)B * p.chunks), dim3(256), 0, st, a);
        hipLaunchKernelGGL((vx_k_verify_draw<DT>), dim3((unsigned)B), dim3(256), 0, st, a);
    });
    vx_prof_end(VX_PROF_VERIFY, st);
    return hipGetLastError() == hipSuccess ? VX_OK : VX_ERR_LAUNCH;
}
