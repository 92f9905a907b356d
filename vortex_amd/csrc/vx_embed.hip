// Embedding lookup with scaling and its gradient.
//   out[t,:]     = scale * table[ids[t],:]                        (id < 0: padding, a row of zeros)
//   d_table[v,:] = scale * sum over t with ids[t] == v of grad_out[t,:]
#include "vx_dtype.h"
#include "vx_profile.h"

__device__ __forceinline__ long long vx_id_at(const void *ids, int id_bytes, long long t) {
    return id_bytes == 8 ? ((const long long *)ids)[t] : (long long)((const int *)ids)[t];
}

// ------------------------------------------------------------------------------------------------ lookup
// One wave per slice of one token's row, U 16-byte pieces for each lane, all loads issued before the first store.
template <int DT, int U, bool TINY, bool NT>
__global__ __launch_bounds__(256) void vx_k_embed(const void *__restrict__ ids, int id_bytes, long long T,
                                                  const void *__restrict__ table, long long n_rows, int D, int slices,
                                                  long long stride, float scale, void *__restrict__ out,
                                                  int *__restrict__ status) {
    typedef typename vx_elem<DT>::type E;
    constexpr int VEC = 16 / sizeof(E);
    const long long item = (long long)vx_block() * 4 + (threadIdx.x >> 6);
    if (item >= T * slices) return;
    const long long t = item / slices;
    const int slice = (int)(item - t * slices), lane = vx_lane();
    const long long id = vx_id_at(ids, id_bytes, t);
    const bool ok = id >= 0 && id < n_rows;
    if (id >= n_rows && status && lane == 0 && slice == 0) atomicOr(status, VX_STATUS_BAD_TOKEN);
    const E *src = (const E *)table + (ok ? id * stride : 0);
    E *dst = (E *)out + t * D;
    const int c0 = slice * 64 * VEC * U + lane * VEC;
    vx_vec<DT> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = vx_cols<DT>(c0 + u * 64 * VEC, D).template load<TINY>(src, D);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float f[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) f[k] = ok ? (float)v[u].e[k] * scale : 0.f;
        vx_cols<DT>(c0 + u * 64 * VEC, D).template store<NT>(dst, f, D);
    }
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
    // few tokens: short slices, so that the row of one token is spread over several waves
    const int vec = 16 / es;
    const bool wide = n_tokens * (int64_t)D > 1 << 20;
    const int slices = (D + 64 * vec * (wide ? 4 : 1) - 1) / (64 * vec * (wide ? 4 : 1));
    const int64_t blocks = (n_tokens * slices + 3) / 4;
    if (blocks > 2147483647LL) return VX_ERR_UNSUPPORTED;
    vx_prof_begin(VX_PROF_EMBED, st);
#define VX_EMBED_GO(...)                                                                                                       \
    hipLaunchKernelGGL((vx_k_embed<__VA_ARGS__>), vx_grid(blocks), dim3(256), 0, st, d_ids, id_bytes, (long long)n_tokens, d_table, \
                       (long long)n_rows, D, slices, (long long)table_stride, scale, d_out, d_status)
    VX_DISPATCH_DTYPE(dtype, {
        if (D < vec) VX_EMBED_GO(DT, 1, true, false);
        else if (vx_past_caches(d_out, n_tokens, D, dtype)) VX_EMBED_GO(DT, 4, false, true);
        else if (wide) VX_EMBED_GO(DT, 4, false, false);
        else VX_EMBED_GO(DT, 1, false, false);
    });
#undef VX_EMBED_GO
    vx_prof_end(VX_PROF_EMBED, st);
    return hipGetLastError() == hipSuccess ? VX_OK : VX_ERR_LAUNCH;
}

// ------------------------------------------------------------------------------------------------ gradient
// 1. The tokens are sorted by id, stably, so the tokens of a table row lie next to each other in their own order: the sums
//    have one order whatever the launch does.  Up to 16384 tokens by counting, for each token, the tokens in front of it
//    (T^2 / 64 compares of a wave: 14 us of the chip's issue at 16384, 3.5 at 8192; measured 8.5 us at 2048, 13 at 5001),
//    beyond by a radix sort (38 us at 65536).
// 2. Beyond 64 tokens every full chunk of 16 sorted tokens of one id is summed once, and (from 8192 tokens) every full chunk
//    of 16 such chunks: a frequent token's row costs at most 30 rows of grad_out, 30 chunks and one row for each further
//    256 tokens, instead of all its tokens on one wave (chunks of 32 / 16 / 8: 49 / 42 / 41 us at 2048 x 1024 fp32, whose end is
//    the longest such chain, 380 / 383 / 394 at 65536 x 4096 bf16).
// 3. Each table row is written once, from its chunks and the tokens at their ends; or, with few tokens, the rows without any are
//    cleared while the tokens are sorted.
#define VX_EG_COUNT_MAX 16384     // tokens sorted by counting
#define VX_EG_SUB 2048            // tokens one workgroup of the radix sort ranks at a time: 256 threads x 8
#define VX_EG_TILES 256           // workgroups of a sorting pass at most
#define VX_EG_BINS 512            // 9 bits of the id for each pass at most
#define VX_EG_CHUNK 16
#define VX_EG_CHUNK_MIN 64
#define VX_EG_CHUNK2_MIN 8192
#define VX_EG_ROWS 8              // table rows of one workgroup

// Columns of one wave's slice: U pieces of 64 lanes x 16 bytes of grad_out, 512 columns in every type (fp32 with one piece:
// 27 instead of 24 us at 2048 x 1024; 16-bit types with two: 33 instead of 24 us at 5001 x 1000 fp16, no gain at 4096 columns).
#define VX_EG_SLICE 512
template <int GT> __host__ __device__ constexpr int vx_eg_u() { return GT == VX_DTYPE_F32 ? 2 : 1; }

// Which tables are cleared beside the sort and then written only where there are tokens (us, this / every row once):
//   2048 x 32000 x 1024 fp32 34/39, 5001 x 50021 x 1000 fp16 27/37, 64 x 32000 24/30, 16000 x 32000 63/69, 2000 x 4096 23/23;
//   as many tokens as rows 93/86; beyond the 256 MB of the last cache the zeros are still on their way when the rows come
//   (16384 x 131072 x 4096 bf16 312/261, 5000 x 223/223, 2048 x 200/211).  Added to a given gradient: 2048 x 32000 20/24,
//   16000 x 57/59, 65536 x 129/121.
#define VX_EG_CLEAR_MAX (256LL << 20)
#define VX_EG_CLEAR_BLOCKS 1024   // 512 / 2048: 35 / 34 instead of 34 us at 2048 x 32000 x 1024 fp32
#define VX_EG_SPLIT 65536         // up to so many (token, slice) pairs there is a wave for each

struct vx_eg_plan {
    int bits, passes, tiles;
    long long tile;               // tokens of one tile, a multiple of VX_EG_SUB
    int chunks, chunks2;
    long long pitch;              // columns of a row of partial sums
    size_t key[2], pos[2], hist, part1, part2, total;
};

static vx_eg_plan vx_eg_make_plan(int64_t T, int64_t n_rows, int D) {
    vx_eg_plan p;
    int kb = 1;
    while (kb < 31 && (n_rows >> kb)) ++kb;                       // keys 0 .. n_rows (n_rows: no row)
    p.passes = (kb + 8) / 9;
    p.bits = (kb + p.passes - 1) / p.passes;
    const int64_t subs = (T + VX_EG_SUB - 1) / VX_EG_SUB, per = (subs + VX_EG_TILES - 1) / VX_EG_TILES;
    p.tile = per * VX_EG_SUB;
    p.tiles = (int)((T + p.tile - 1) / p.tile);
    p.chunks = T > VX_EG_CHUNK_MIN ? (int)(T / VX_EG_CHUNK) : 0;
    p.chunks2 = T >= VX_EG_CHUNK2_MIN ? p.chunks / VX_EG_CHUNK : 0;
    const bool radix = T > VX_EG_COUNT_MAX;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += (n + 255) & ~(size_t)255; return o; };
    for (int i = 0; i < 2; ++i) {
        p.key[i] = take(i == 0 || radix ? (size_t)T * 4 : 0);
        p.pos[i] = take(i == 0 || radix ? (size_t)T * 4 : 0);
    }
    p.hist = take(radix ? (size_t)p.tiles * VX_EG_BINS * 4 : 0);
    p.pitch = (D + VX_EG_SLICE - 1) / VX_EG_SLICE * VX_EG_SLICE;
    p.part1 = take((size_t)p.chunks * p.pitch * 4);
    p.part2 = take((size_t)p.chunks2 * p.pitch * 4);
    p.total = at;
    return p;
}

// Zeros for the table, written by the workgroups behind those that sort: `pieces` of 16 bytes at the aligned address `base`, and a
// few elements (2 bytes each) in front of and behind them.  A contiguous range for each workgroup, ordinary stores: 131 MB in
// 17.5 us (all workgroups side by side 21, past the caches 24).
struct vx_eg_zero {
    char *base;
    long long pieces;
    unsigned short *head, *tail;
    int heads, tails;
};
__device__ __forceinline__ void vx_eg_fill(const vx_eg_zero &z, int block, int blocks) {
    if (block == 0) {
        if ((int)threadIdx.x < z.heads) z.head[threadIdx.x] = 0;
        if ((int)threadIdx.x < z.tails) z.tail[threadIdx.x] = 0;
    }
    const long long per = (z.pieces + blocks - 1) / blocks, a = block * per, e = min(z.pieces, a + per);
    for (long long i = a + threadIdx.x; i < e; i += blockDim.x) ((vx_v4 *)z.base)[i] = vx_v4{0.f, 0.f, 0.f, 0.f};
}

__device__ __forceinline__ unsigned vx_eg_key(const void *ids, int id_bytes, long long t, long long n_rows, int *status) {
    const long long id = vx_id_at(ids, id_bytes, t);
    if (id >= n_rows && status) atomicOr(status, VX_STATUS_BAD_TOKEN);
    return (unsigned)(id >= 0 && id < n_rows ? id : n_rows);
}

// Stable sort by counting: a workgroup places 64 tokens, one for each lane; its 16 waves share the scan of all keys, four
// to an LDS read, a compare and an add-with-carry each.  Keys behind a token count when they are smaller, keys in front of
// it also when they are equal.  Workgroups from `own` on clear the table instead.
__global__ __launch_bounds__(1024) void vx_k_eg_count_sort(const void *__restrict__ ids, int id_bytes, int T, long long n_rows,
                                                           unsigned *__restrict__ key_out, int *__restrict__ pos_out,
                                                           int *__restrict__ status, int own, vx_eg_zero zero) {
    __shared__ __attribute__((aligned(16))) unsigned s_key[VX_EG_COUNT_MAX];
    __shared__ int s_count[64];
    if ((int)blockIdx.x >= own) { vx_eg_fill(zero, blockIdx.x - own, gridDim.x - own); return; }
    const int lane = vx_lane(), w = threadIdx.x >> 6;
    const int groups = (T + 3) >> 2;                              // of four keys
    for (int i = threadIdx.x; i < groups * 4; i += 1024)
        s_key[i] = i < T ? vx_eg_key(ids, id_bytes, i, n_rows, blockIdx.x == 0 ? status : nullptr) : ~0u;
    if (threadIdx.x < 64) s_count[threadIdx.x] = 0;
    __syncthreads();
    const int t0 = blockIdx.x * 64, t = min(t0 + lane, T - 1);
    const unsigned k = s_key[t];
    const int per = (groups + 15) / 16, g0 = min(groups, w * per), g1 = min(groups, g0 + per);
    int n = 0;
    auto below = [&](int from, int to, unsigned limit) {          // keys below `limit` in groups from .. to
        int g = from;
        for (; g + 8 <= to; g += 8) {
            uint4 q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = *(const uint4 *)&s_key[4 * (g + i)];
#pragma unroll
            for (int i = 0; i < 8; ++i) n += (q[i].x < limit) + (q[i].y < limit) + (q[i].z < limit) + (q[i].w < limit);
        }
        for (; g < to; ++g) {
            const uint4 q = *(const uint4 *)&s_key[4 * g];
            n += (q.x < limit) + (q.y < limit) + (q.z < limit) + (q.w < limit);
        }
    };
    const int mid0 = min(max(g0, t0 / 4), g1), mid1 = min(max(g0, t0 / 4 + 16), g1);    // the groups of the 64 tokens themselves
    below(g0, mid0, k + 1);
    for (int i = 4 * mid0; i < 4 * mid1; ++i) n += s_key[i] < k || (s_key[i] == k && i < t);
    below(mid1, g1, k);
    atomicAdd(&s_count[lane], n);
    __syncthreads();
    if (w == 0 && t0 + lane < T) {
        const int at = s_count[lane];
        key_out[at] = k;
        pos_out[at] = t;
    }
}

// Histogram of one digit of each tile.  Pass 0 reads the ids, the others the keys of the pass before.
__global__ __launch_bounds__(256) void vx_k_eg_hist(const void *__restrict__ ids, int id_bytes, const unsigned *__restrict__ key_in,
                                                    long long T, long long n_rows, int bits, int pass, long long tile,
                                                    int *__restrict__ hist, int *__restrict__ status) {
    __shared__ int s_h[VX_EG_BINS];
    const int bins = 1 << bits;
    for (int i = threadIdx.x; i < bins; i += 256) s_h[i] = 0;
    __syncthreads();
    const long long lo = blockIdx.x * tile, hi = min(T, lo + tile);
    for (long long t = lo + threadIdx.x; t < hi; t += 256) {
        const unsigned k = pass ? key_in[t] : vx_eg_key(ids, id_bytes, t, n_rows, status);
        atomicAdd(&s_h[(k >> (pass * bits)) & (bins - 1)], 1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += 256) hist[(size_t)blockIdx.x * VX_EG_BINS + i] = s_h[i];
}

// One radix sorting pass: each workgroup places the tokens of its tile, 2048 at a time, in order.
__global__ __launch_bounds__(256) void vx_k_eg_pass(const void *__restrict__ ids, int id_bytes, long long T, long long n_rows,
                                                    int bits, int pass, long long tile, const int *__restrict__ hist,
                                                    const unsigned *__restrict__ key_in, const int *__restrict__ pos_in,
                                                    unsigned *__restrict__ key_out, int *__restrict__ pos_out) {
    __shared__ int s_wave[4][VX_EG_BINS];     // digits seen by each wave: counts, then the wave's first place of each digit
    __shared__ int s_base[VX_EG_BINS];        // next place of each digit
    __shared__ int s_scan[4];
    const int bins = 1 << bits, tiles = gridDim.x, shift = pass * bits, lane = vx_lane(), w = threadIdx.x >> 6;
    // digits 2 tid and 2 tid + 1: how often in all tiles, how often in the tiles before this one
    int total[2] = {}, before[2] = {};
#pragma unroll 8
    for (int t = 0; t < tiles; ++t) {
        const int2 c = 2 * (int)threadIdx.x < bins ? *(const int2 *)&hist[(size_t)t * VX_EG_BINS + 2 * threadIdx.x] : int2{0, 0};
        total[0] += c.x; total[1] += c.y;
        if (t < (int)blockIdx.x) { before[0] += c.x; before[1] += c.y; }
    }
    int run = total[0] + total[1];
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(run, d, VX_WAVE);
        if (lane >= d) run += o;
    }
    if (lane == 63) s_scan[w] = run;
    __syncthreads();
    run -= total[0] + total[1];
    for (int i = 0; i < w; ++i) run += s_scan[i];
    if (2 * (int)threadIdx.x < bins) {
        s_base[2 * threadIdx.x] = run + before[0];
        s_base[2 * threadIdx.x + 1] = run + total[0] + before[1];
    }
    const long long lo = blockIdx.x * tile, hi = min(T, lo + tile);
    for (long long t0 = lo; t0 < hi; t0 += VX_EG_SUB) {
        const int n = (int)min((long long)VX_EG_SUB, hi - t0);
        unsigned key[8];
        int pos[8], place[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {                             // wave w holds tokens w*512 + r*64 + lane: its own in order
            const int i = w * 512 + r * 64 + lane;
            key[r] = 0;
            pos[r] = (int)(t0 + i);
            if (i < n) {
                if (pass) { key[r] = key_in[t0 + i]; pos[r] = pos_in[t0 + i]; }
                else key[r] = vx_eg_key(ids, id_bytes, t0 + i, n_rows, nullptr);
            }
        }
        for (int i = lane; i < bins; i += 64) s_wave[w][i] = 0;   // the wave's own counters: LDS keeps a wave's order
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const bool in = w * 512 + r * 64 + lane < n;
            const int d = (key[r] >> shift) & (bins - 1);
            u64 same = __ballot(in);
            for (int b = 0; b < bits; ++b) {
                const u64 one = __ballot((d >> b) & 1);
                same &= ((d >> b) & 1) ? one : ~one;
            }
            place[r] = 0;
            if (in) {
                place[r] = s_wave[w][d] + vx_mbcnt(same);
                if (vx_mbcnt(same) == 0) s_wave[w][d] += __popcll(same);
            }
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        for (int i = threadIdx.x; i < bins; i += 256) {
            int at = s_base[i];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = s_wave[q][i];
                s_wave[q][i] = at;
                at += c;
            }
            s_base[i] = at;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (w * 512 + r * 64 + lane < n) {
                const int at = place[r] + s_wave[w][(key[r] >> shift) & (bins - 1)];
                key_out[at] = key[r];
                pos_out[at] = pos[r];
            }
        __syncthreads();
    }
}

// sum[] += N rows of grad_out at pos(0..N-1), all of them in flight together, added in that order
template <int GT, int U, bool TINY, int N, class P>
__device__ __forceinline__ void vx_eg_add_n(const typename vx_elem<GT>::type *__restrict__ grad, P pos, int D, int c, float *sum) {
    constexpr int VEC = 16 / sizeof(typename vx_elem<GT>::type);
    vx_vec<GT> v[N][U];
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
        for (int q = 0; q < U; ++q) v[u][q] = vx_cols<GT>(c + q * 64 * VEC, D).template load<TINY>(grad + (long long)pos(u) * D, D);
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
        for (int q = 0; q < U; ++q)
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[q * VEC + k] += (float)v[u][q].e[k];
}

// sum[] += rows of grad_out at pos[a..b), in that order.  The positions are scalar loads: as vector loads they wait for the
// stores of the rows before (355 instead of 268 us for the rows of 65536 tokens x 4096 columns bf16).
template <int GT, int U, bool TINY>
__device__ __forceinline__ void vx_eg_add_tokens(const typename vx_elem<GT>::type *__restrict__ grad, const int *__restrict__ pos,
                                                 int a, int b, int D, int c, float *sum) {
    auto at = [&](int u) { return pos[a + u]; };
    for (; b - a >= 4; a += 4) vx_eg_add_n<GT, U, TINY, 4>(grad, at, D, c, sum);
    if ((b - a) & 2) { vx_eg_add_n<GT, U, TINY, 2>(grad, at, D, c, sum); a += 2; }
    if ((b - a) & 1) vx_eg_add_n<GT, U, TINY, 1>(grad, at, D, c, sum);
}

// sum[] += rows a..b of fp32 partial sums.  Their rows are padded to VX_EG_SLICE columns (pitch), so no column sticks out: a
// lane keeps the columns of its sums, those of vx_cols.
template <int GT, int U>
__device__ __forceinline__ void vx_eg_add_partials(const float *__restrict__ part, long long a, long long b, long long pitch, int c, float *sum) {
    constexpr int VEC = 16 / sizeof(typename vx_elem<GT>::type);
#pragma unroll 4
    for (long long i = a; i < b; ++i)
#pragma unroll
        for (int q = 0; q < U; ++q)
#pragma unroll
            for (int k = 0; k < VEC; k += 4) {
                const vx_f4 v = *(const vx_f4 *)(part + i * pitch + c + q * 64 * VEC + k);
                sum[q * VEC + k] += v.x; sum[q * VEC + k + 1] += v.y; sum[q * VEC + k + 2] += v.z; sum[q * VEC + k + 3] += v.w;
            }
}

// One wave per (chunk of 16 sorted tokens, slice of columns); chunks of several ids have no sum of their own.
template <int GT, int U, bool TINY>
__global__ __launch_bounds__(256) void vx_k_eg_chunks(const unsigned *__restrict__ key, const int *__restrict__ pos, int chunks,
                                                      unsigned n_rows, const void *__restrict__ grad, int D, int slices,
                                                      long long pitch, float *__restrict__ part1) {
    typedef typename vx_elem<GT>::type G;
    constexpr int VEC = 16 / sizeof(G);
    const long long item = (long long)vx_block() * 4 + (threadIdx.x >> 6);
    const long long c1 = item / slices;
    if (c1 >= chunks) return;
    const int a = (int)c1 * VX_EG_CHUNK, c = (int)(item - c1 * slices) * VX_EG_SLICE + vx_lane() * VEC;
    const unsigned k0 = key[a];
    if (k0 >= n_rows || key[a + VX_EG_CHUNK - 1] != k0) return;
    float sum[U * VEC] = {};
    const int mine = pos[a + (vx_lane() & (VX_EG_CHUNK - 1))];
#pragma unroll
    for (int i = 0; i < VX_EG_CHUNK; i += 4)
        vx_eg_add_n<GT, U, TINY, 4>((const G *)grad, [&](int u) { return __builtin_amdgcn_readlane(mine, i + u); }, D, c, sum);
#pragma unroll
    for (int q = 0; q < U; ++q)
#pragma unroll
        for (int k = 0; k < VEC; k += 4)
            *(vx_f4 *)(part1 + c1 * pitch + c + q * 64 * VEC + k) = vx_f4{sum[q * VEC + k], sum[q * VEC + k + 1], sum[q * VEC + k + 2], sum[q * VEC + k + 3]};
}

// The same over 16 chunks; 256 columns for each wave.
__global__ __launch_bounds__(256) void vx_k_eg_chunks2(const unsigned *__restrict__ key, int chunks, unsigned n_rows, int slices,
                                                       long long pitch, const float *__restrict__ part1, float *__restrict__ part2) {
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long long c2 = item / slices;
    if (c2 >= chunks) return;
    const int a = (int)c2 * VX_EG_CHUNK * VX_EG_CHUNK, c = (int)(item - c2 * slices) * 256 + vx_lane() * 4;
    const unsigned k0 = key[a];
    if (k0 >= n_rows || key[a + VX_EG_CHUNK * VX_EG_CHUNK - 1] != k0) return;
    float sum[4] = {};
    vx_eg_add_partials<VX_DTYPE_F32, 1>(part1, c2 * VX_EG_CHUNK, (c2 + 1) * VX_EG_CHUNK, pitch, c, sum);
    *(vx_f4 *)(part2 + c2 * pitch + c) = vx_f4{sum[0], sum[1], sum[2], sum[3]};
}

// first i in [0, n] with key[i] >= target, by the 16 lanes of a quarter wave: a sixteenth of the range is left each step
__device__ __forceinline__ int vx_eg_lower_bound(const unsigned *__restrict__ key, int n, unsigned target) {
    const int lane = vx_lane(), sub = lane & 15, at = lane & 48;
    int lo = 0, hi = n;
    while (__any(hi > lo)) {
        const int step = (hi - lo + 15) >> 4;
        const long long p = (long long)lo + (long long)(sub + 1) * step - 1;
        const bool less = p < hi && key[p] < target;
        const int c = __popc((unsigned)(__ballot(less) >> at) & 0xffffu);
        const long long top = (long long)lo + (long long)(c + 1) * step - 1;
        lo = (int)min((long long)hi, (long long)lo + (long long)c * step);
        hi = (int)min((long long)hi, top);
        hi = max(hi, lo);
    }
    return lo;
}

struct vx_eg_sums {                                               // what a table row is summed from
    const unsigned *key;
    const int *pos;
    const void *grad;
    long long pitch, n_rows;
    const float *part1, *part2;
    int T, D, slices, levels;                                     // levels: of chunks (0, 1, 2)
    float scale;
    void *out;
    int accumulate;
};

// Columns c .. of row v from the sorted tokens s .. e - 1 and their chunks.
template <int GT, int TT, int U, bool TINY, bool NT>
__device__ __forceinline__ void vx_eg_row(const vx_eg_sums &a, long long v, int s, int e, int c) {
    typedef typename vx_elem<GT>::type G;
    typedef typename vx_elem<TT>::type E;
    constexpr int VEC = 16 / sizeof(G);
    const int D = a.D;
    float sum[U * VEC] = {};
    const int a1 = (s + VX_EG_CHUNK - 1) / VX_EG_CHUNK, b1 = e / VX_EG_CHUNK;
    if (a.levels == 0 || a1 >= b1) {
        vx_eg_add_tokens<GT, U, TINY>((const G *)a.grad, a.pos, s, e, D, c, sum);
    } else {
        vx_eg_add_tokens<GT, U, TINY>((const G *)a.grad, a.pos, s, a1 * VX_EG_CHUNK, D, c, sum);
        const int a2 = (a1 + VX_EG_CHUNK - 1) / VX_EG_CHUNK, b2 = b1 / VX_EG_CHUNK;
        if (a.levels == 1 || a2 >= b2) {
            vx_eg_add_partials<GT, U>(a.part1, a1, b1, a.pitch, c, sum);
        } else {
            vx_eg_add_partials<GT, U>(a.part1, a1, (long long)a2 * VX_EG_CHUNK, a.pitch, c, sum);
            vx_eg_add_partials<GT, U>(a.part2, a2, b2, a.pitch, c, sum);
            vx_eg_add_partials<GT, U>(a.part1, (long long)b2 * VX_EG_CHUNK, b1, a.pitch, c, sum);
        }
        vx_eg_add_tokens<GT, U, TINY>((const G *)a.grad, a.pos, b1 * VX_EG_CHUNK, e, D, c, sum);
    }
    if (c >= D) return;
    E *dst = (E *)a.out + v * D;
    const float scale = s == e ? 0.f : a.scale;                   // zeros without a token, whatever the scale
#pragma unroll
    for (int k = 0; k < U * VEC; ++k) sum[k] *= scale;
    // columns at .. at + VEC of the sums, from c on to be stored; the table's pieces are VEC wide, or half of it where a
    // 16-bit gradient is summed into fp32
    constexpr int W = 16 / sizeof(E);
#pragma unroll
    for (int q = 0; q < U; ++q) {
        const vx_cols<GT> col(c + q * 64 * VEC, D);
        if (col.c >= D) continue;
#pragma unroll
        for (int k = 0; k < VEC; k += W) {
            vx_cols<TT> part(0, D);
            part.c = max(col.c, col.at + k);
            part.at = col.at + k;
            float *f = sum + q * VEC + k;
            if (a.accumulate) {
                vx_vec<TT> old;
                if (!TINY) {
                    old.raw = vx_load16<TT>(dst + part.at);
                } else {
#pragma unroll
                    for (int j = 0; j < W; ++j) old.e[j] = part.at + j < D ? dst[part.at + j] : (E)0.0f;
                }
#pragma unroll
                for (int j = 0; j < W; ++j) f[j] = (float)old.e[j] + f[j];
            }
            part.template store<NT>(dst, f, D);
        }
    }
}

// Every table row: block + i * blocks (i < 8), as frequent ids lie next to each other and go to different workgroups.
// A wave sums one slice of one row.  Bound by the write of the table: few registers, so that many waves have their loads and
// stores on the way (a version that split long rows over the waves of a workgroup held 94 instead of 62 registers: 292
// instead of 265 us for the rows of 65536 tokens x 4096 columns bf16 over 131072).
template <int GT, int TT, int U, bool TINY, bool NT>
__global__ __launch_bounds__(256) void vx_k_eg_rows(vx_eg_sums a) {
    constexpr int VEC = 16 / sizeof(typename vx_elem<GT>::type);
    __shared__ int s_at[2 * VX_EG_ROWS];
    const int lane = vx_lane(), w = threadIdx.x >> 6;
    const long long block = vx_block(), blocks = (a.n_rows + VX_EG_ROWS - 1) / VX_EG_ROWS;
    if (block >= blocks) return;
    {
        const int q = threadIdx.x >> 4;                           // 16 searches: the beginning and the end of 8 rows
        const long long v = block + (q >> 1) * blocks + (q & 1);
        const int at = vx_eg_lower_bound(a.key, a.T, (unsigned)min(v, a.n_rows));
        if ((lane & 15) == 0) s_at[q] = at;
    }
    __syncthreads();
    for (int item = w; item < VX_EG_ROWS * a.slices; item += 4) {
        const int i = item / a.slices, c = (item - i * a.slices) * VX_EG_SLICE + lane * VEC;
        const long long v = block + i * blocks;
        const int s = __builtin_amdgcn_readfirstlane(s_at[2 * i]), e = __builtin_amdgcn_readfirstlane(s_at[2 * i + 1]);
        if (v >= a.n_rows || (a.accumulate && s == e)) continue;
        vx_eg_row<GT, TT, U, TINY, NT>(a, v, s, e, c);
    }
}

// The rows that have tokens: one wave (or, with few tokens, one for each slice) where a sorted token's id differs from the one
// before it.
template <int GT, int TT, int U, bool TINY>
__global__ __launch_bounds__(256) void vx_k_eg_runs(vx_eg_sums a, int split) {
    constexpr int VEC = 16 / sizeof(typename vx_elem<GT>::type);
    const int lane = vx_lane();
    const long long item = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), s_ = item / split;
    if (s_ >= a.T) return;
    const int s = (int)s_, part = (int)(item - s_ * split);
    const unsigned k = a.key[s];
    if (k >= a.n_rows || (s > 0 && a.key[s - 1] == k)) return;
    int e = s + 1;
    while (true) {                                                // 64 tokens at a time as far as the id is the same
        const u64 other = __ballot(e + lane >= a.T || a.key[min(e + lane, a.T - 1)] != k);
        if (other) { e += __builtin_ctzll(other); break; }
        e += 64;
    }
    for (int i = part; i < a.slices; i += split) vx_eg_row<GT, TT, U, TINY, false>(a, k, s, e, i * VX_EG_SLICE + lane * VEC);
}

extern "C" size_t vx_embed_tokens_grad_workspace_bytes(int64_t n_tokens, int64_t n_rows, int D) {
    if (n_tokens <= 0 || n_rows <= 0 || D <= 0 || n_tokens > VX_MAX_TOKENS || n_rows > VX_MAX_VOCAB || D > VX_MAX_TOKEN_WIDTH) return 0;
    return vx_eg_make_plan(n_tokens, n_rows, D).total;
}

// steps 2 and 3, once the tokens are sorted (key, pos)
template <int GT, int TT, bool TINY>
static void vx_eg_sum(const vx_eg_plan &p, const unsigned *key, const int *pos, int T, const void *grad, long long n_rows, int D,
                      float scale, void *out, int accumulate, bool runs, float *part1, float *part2, hipStream_t st) {
    constexpr int U = vx_eg_u<GT>();
    const int slices = (int)(p.pitch / VX_EG_SLICE), slices2 = (int)(p.pitch / 256);
    if (p.chunks)
        hipLaunchKernelGGL((vx_k_eg_chunks<GT, U, TINY>), vx_grid(((int64_t)p.chunks * slices + 3) / 4), dim3(256), 0, st, key,
                           pos, p.chunks, (unsigned)n_rows, grad, D, slices, p.pitch, part1);
    if (p.chunks2)
        hipLaunchKernelGGL(vx_k_eg_chunks2, dim3((unsigned)(((int64_t)p.chunks2 * slices2 + 3) / 4)), dim3(256), 0, st, key, p.chunks2,
                           (unsigned)n_rows, slices2, p.pitch, part1, part2);
    const vx_eg_sums a = {key, pos, grad, p.pitch, n_rows, part1, part2, T, D, slices, p.chunks2 ? 2 : (p.chunks ? 1 : 0), scale, out, accumulate};
    if (runs) {
        const int split = (int64_t)T * slices <= VX_EG_SPLIT ? slices : 1;
        hipLaunchKernelGGL((vx_k_eg_runs<GT, TT, U, TINY>), dim3((unsigned)(((int64_t)T * split + 3) / 4)), dim3(256), 0, st, a, split);
        return;
    }
    const dim3 grid = vx_grid((n_rows + VX_EG_ROWS - 1) / VX_EG_ROWS);
    if (!TINY && !accumulate && vx_past_caches(out, n_rows, D, TT))
        hipLaunchKernelGGL((vx_k_eg_rows<GT, TT, U, TINY, !TINY>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((vx_k_eg_rows<GT, TT, U, TINY, false>), grid, dim3(256), 0, st, a);
}

extern "C" int vx_embed_tokens_grad(const void *d_ids, int id_bytes, int64_t n_tokens, const void *d_grad_out,
                                    int grad_dtype, int64_t n_rows, int D, float scale, void *d_grad_table,
                                    int table_dtype, int accumulate, int32_t *d_status, void *d_workspace,
                                    size_t workspace_bytes, void *stream) {
    if (!d_ids || !d_grad_out || !d_grad_table || !d_workspace || n_tokens <= 0 || n_rows <= 0 || D <= 0) return VX_ERR_INVALID_ARG;
    if ((id_bytes != 4 && id_bytes != 8) || !vx_dtype_ok(grad_dtype) || !vx_dtype_ok(table_dtype)) return VX_ERR_INVALID_ARG;
    if (n_tokens > VX_MAX_TOKENS || n_rows > VX_MAX_VOCAB || D > VX_MAX_TOKEN_WIDTH) return VX_ERR_UNSUPPORTED;
    if (table_dtype != grad_dtype && table_dtype != VX_DTYPE_F32) return VX_ERR_UNSUPPORTED;
    const vx_eg_plan p = vx_eg_make_plan(n_tokens, n_rows, D);
    if (workspace_bytes < p.total) return VX_ERR_WORKSPACE;
    if (((uintptr_t)d_grad_out & (vx_elem_size(grad_dtype) - 1)) || ((uintptr_t)d_grad_table & (vx_elem_size(table_dtype) - 1)) ||
        ((uintptr_t)d_ids & (id_bytes - 1)) || ((uintptr_t)d_status & 3) || ((uintptr_t)d_workspace & 255))
        return VX_ERR_ALIGNMENT;
    const int T = (int)n_tokens;
    if ((int64_t)p.chunks * (p.pitch / VX_EG_SLICE) > 4LL * 2147483647 || (int64_t)p.chunks2 * (p.pitch / 256) > 4LL * 2147483647)
        return VX_ERR_UNSUPPORTED;
    char *ws = (char *)d_workspace;
    unsigned *key[2] = {(unsigned *)(ws + p.key[0]), (unsigned *)(ws + p.key[1])};
    int *pos[2] = {(int *)(ws + p.pos[0]), (int *)(ws + p.pos[1])}, *hist = (int *)(ws + p.hist);
    float *part1 = (float *)(ws + p.part1), *part2 = (float *)(ws + p.part2);
    hipStream_t st = (hipStream_t)stream;
    vx_prof_begin(VX_PROF_EMBED_GRAD, st);
    const int es = vx_elem_size(table_dtype);
    const int64_t bytes = n_rows * D * es;
    const bool runs = T <= VX_EG_COUNT_MAX && 2 * n_tokens <= n_rows && (accumulate || bytes <= VX_EG_CLEAR_MAX || 64 * n_tokens <= n_rows);
    int at = 0;                                                   // the buffers that hold the sorted tokens
    if (T <= VX_EG_COUNT_MAX) {
        vx_eg_zero z = {};
        int own = (T + 63) / 64, clear = 0;
        if (runs && !accumulate) {
            char *const first = (char *)d_grad_table, *const last = first + bytes;
            char *const base = (char *)(((uintptr_t)first + 15) & ~(uintptr_t)15), *const mid = base < last ? base : last;
            const int64_t pieces = (last - mid) / 16;
            z = vx_eg_zero{mid, pieces, (unsigned short *)first, (unsigned short *)(mid + pieces * 16), (int)((mid - first) / 2),
                           (int)((last - mid - pieces * 16) / 2)};
            clear = (int)min((int64_t)VX_EG_CLEAR_BLOCKS, pieces / 1024 + 1);
        }
        hipLaunchKernelGGL(vx_k_eg_count_sort, dim3(own + clear), dim3(1024), 0, st, d_ids, id_bytes, T, (long long)n_rows, key[0],
                           pos[0], d_status, own, z);
    } else {
        for (int i = 0; i < p.passes; ++i) {
            at = i & 1;
            hipLaunchKernelGGL(vx_k_eg_hist, dim3(p.tiles), dim3(256), 0, st, d_ids, id_bytes, key[at ^ 1], (long long)T,
                               (long long)n_rows, p.bits, i, p.tile, hist, d_status);
            hipLaunchKernelGGL(vx_k_eg_pass, dim3(p.tiles), dim3(256), 0, st, d_ids, id_bytes, (long long)T, (long long)n_rows, p.bits,
                               i, p.tile, hist, key[at ^ 1], pos[at ^ 1], key[at], pos[at]);
        }
    }
    VX_DISPATCH_DTYPE(grad_dtype, {
        if (D < 16 / vx_elem_size(DT)) {
            if (table_dtype == DT) vx_eg_sum<DT, DT, true>(p, key[at], pos[at], T, d_grad_out, n_rows, D, scale, d_grad_table, accumulate, runs, part1, part2, st);
            else vx_eg_sum<DT, VX_DTYPE_F32, true>(p, key[at], pos[at], T, d_grad_out, n_rows, D, scale, d_grad_table, accumulate, runs, part1,
                                                    part2, st);
        } else {
            if (table_dtype == DT) vx_eg_sum<DT, DT, false>(p, key[at], pos[at], T, d_grad_out, n_rows, D, scale, d_grad_table, accumulate, runs, part1, part2, st);
            else vx_eg_sum<DT, VX_DTYPE_F32, false>(p, key[at], pos[at], T, d_grad_out, n_rows, D, scale, d_grad_table, accumulate, runs, part1,
                                                     part2, st);
        }
    });
    vx_prof_end(VX_PROF_EMBED_GRAD, st);
    return hipGetLastError() == hipSuccess ? VX_OK : VX_ERR_LAUNCH;
}
