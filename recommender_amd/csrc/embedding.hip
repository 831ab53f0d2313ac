// embedding.hip - lookup of a batch of table rows with scaling, and its gradient by sorted tokens (gfx950, MI355X).
//
//   out[t] = scale * table[ids[t]]                       dtable[v] = scale * sum_{t: ids[t] = v} grad[t]
//
// The gradient sorts the batch's positions by id (stable: equal ids stay in the order of t), so that a table row's tokens
// are one stretch of the sorted list; a row is then summed by one group of lanes in fp32, in the order of t, and written
// once.  No atomics: the same inputs give the same bits.
#include <algorithm>
#include <math.h>
#include "rows.h"

namespace {

// ------------------------------------------------------------------ lookup
// A thread moves V elements (one access); the V-element pieces of the output are numbered through.
template <typename T, int V>
__global__ __launch_bounds__(256) void k_embedding(const T *__restrict__ table, int64_t stride, int64_t n_rows, int32_t d,
                                                   const int32_t *__restrict__ ids, int64_t n, float scale, T *__restrict__ out)
{
    const int32_t per = d / V;
    const int64_t total = n * per;
    for (int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x; p < total; p += (int64_t)gridDim.x * 256) {
        const int64_t t = p / per;
        const int32_t c = (int32_t)(p - t * per) * V;
        const int32_t id = ids[t];
        float v[V];
        if (id >= 0 && id < n_rows) {
            load_vec<V>(table + (int64_t)id * stride + c, v);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] *= scale;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = id < 0 ? 0.f : NAN;
        }
        store_vec<V>(out + p * V, v);
    }
}

template <typename T>
int launch_embedding(const T *table, int64_t stride, int64_t n_rows, int32_t d, const int32_t *ids, int64_t n, float scale,
                     T *out, hipStream_t st)
{
    const int v = vec_elems(sizeof(T), d, stride, d, table, out);
    const unsigned grid = (unsigned)std::min<int64_t>((n * (d / v) + 255) / 256, 1 << 20);
#define MF_EMB(V_) hipLaunchKernelGGL((k_embedding<T, V_>), dim3(grid), dim3(256), 0, st, table, stride, n_rows, d, ids, n, scale, out)
    if constexpr (sizeof(T) == 2) {
        if (v == 8) { MF_EMB(8); MF_LAUNCH_CHECK(); return MFSGD_OK; }
    }
    if (v == 4) MF_EMB(4);
    else if (v == 2) MF_EMB(2);
    else MF_EMB(1);
#undef MF_EMB
    MF_LAUNCH_CHECK();
    return MFSGD_OK;
}

// ------------------------------------------------------------------ positions sorted by id
// Keys: an id inside the table, or n_rows for everything else (padding, ids behind the table), which sorts to the end.
__device__ __forceinline__ uint32_t sort_key(int32_t id, int64_t n_rows)
{
    return (uint32_t)id < (uint64_t)n_rows ? (uint32_t)id : (uint32_t)n_rows;
}

// Small batches: the rank of position t is the number of smaller keys plus the number of equal keys in front of it.  A wave
// ranks 64 positions against all keys, held in LDS; one launch, no passes.
constexpr int RANK_MAX = 4096;
__global__ __launch_bounds__(64) void k_rank(const int32_t *__restrict__ ids, int32_t n, int64_t n_rows,
                                             uint32_t *__restrict__ key_out, int32_t *__restrict__ pos_out)
{
    __shared__ __attribute__((aligned(16))) uint32_t keys[RANK_MAX];
    const int lane = threadIdx.x;
    const int n4 = (n + 3) & ~3;
    for (int i = lane; i < n4; i += 64) keys[i] = i < n ? sort_key(ids[i], n_rows) : 0xffffffffu;
    __syncthreads();
    const int t = blockIdx.x * 64 + lane;
    const uint32_t mine = keys[t < n ? t : 0];
    int32_t rank = 0;
    for (int i = 0; i < n4; i += 4) {
        const uint4 k = *(const uint4 *)(keys + i);
        rank += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
        rank += (k.x == mine && i < t) + (k.y == mine && i + 1 < t) + (k.z == mine && i + 2 < t) + (k.w == mine && i + 3 < t);
    }
    if (t < n) { key_out[rank] = mine; pos_out[rank] = t; }
}

// Large batches: least significant digit first, DIGIT bits a pass, stable.  A tile is SORT_TILE consecutive entries of one
// workgroup; a pass counts every tile's digits, turns the counts into first places and moves the entries.
constexpr int SORT_TILE = 4096, SORT_BINS = 1024, SORT_PER = SORT_TILE / 256;

__global__ __launch_bounds__(256) void k_sort_count(const uint32_t *__restrict__ key, const int32_t *__restrict__ ids, int32_t n,
                                                    int64_t n_rows, int shift, int bins, int32_t *__restrict__ counts)
{
    __shared__ int32_t cnt[SORT_BINS];
    for (int b = threadIdx.x; b < bins; b += 256) cnt[b] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * SORT_TILE;
    for (int i = 0; i < SORT_PER; ++i) {
        const int64_t t = base + i * 256 + threadIdx.x;
        if (t < n) {
            const uint32_t k = ids ? sort_key(ids[t], n_rows) : key[t];
            atomicAdd(&cnt[(k >> shift) & (bins - 1)], 1);          // whole numbers: any order gives the same count
        }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += 256) counts[(int64_t)b * gridDim.x + blockIdx.x] = cnt[b];
}

// counts[bin][tile] -> exclusive sums over the tiles of a bin, totals[bin]; one wave per bin
__global__ __launch_bounds__(64) void k_sort_tiles(int32_t *__restrict__ counts, int32_t tiles, int32_t *__restrict__ totals)
{
    const int lane = threadIdx.x;
    int32_t *row = counts + (int64_t)blockIdx.x * tiles;
    int32_t carry = 0;
    for (int a = 0; a < tiles; a += 64) {
        const int i = a + lane;
        const int32_t c = i < tiles ? row[i] : 0;
        int32_t s = c;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int32_t up = __shfl_up(s, m, 64);
            if (lane >= m) s += up;
        }
        if (i < tiles) row[i] = carry + s - c;
        carry += __shfl(s, 63, 64);
    }
    if (lane == 0) totals[blockIdx.x] = carry;
}

__global__ __launch_bounds__(256) void k_sort_move(const uint32_t *__restrict__ key, const int32_t *__restrict__ pos,
                                                   const int32_t *__restrict__ ids, int32_t n, int64_t n_rows, int shift, int bits,
                                                   const int32_t *__restrict__ counts, const int32_t *__restrict__ totals,
                                                   uint32_t *__restrict__ key_out, int32_t *__restrict__ pos_out)
{
    __shared__ int32_t cnt[4][SORT_BINS];
    __shared__ int32_t first[SORT_BINS];
    __shared__ int32_t part[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bins = 1 << bits;
    for (int b = tid; b < 4 * SORT_BINS; b += 256) (&cnt[0][0])[b] = 0;
    // first place of every bin: exclusive sums of the totals, four bins a thread
    {
        int32_t c[4], s = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) { c[i] = 4 * tid + i < bins ? totals[4 * tid + i] : 0; s += c[i]; }
        int32_t incl = s;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int32_t up = __shfl_up(incl, m, 64);
            if (lane >= m) incl += up;
        }
        if (lane == 63) part[wave] = incl;
        __syncthreads();
        int32_t at = incl - s;
        for (int w = 0; w < wave; ++w) at += part[w];
#pragma unroll
        for (int i = 0; i < 4; ++i) { if (4 * tid + i < bins) first[4 * tid + i] = at; at += c[i]; }
    }
    __syncthreads();
    // a wave takes SORT_TILE / 4 consecutive entries, 64 at a time: a lane's place among the wave's entries of its bin
    const int64_t base = (int64_t)blockIdx.x * SORT_TILE + wave * (SORT_TILE / 4);
    uint32_t k[SORT_PER];
    int32_t p[SORT_PER], r[SORT_PER];
#pragma unroll
    for (int i = 0; i < SORT_PER; ++i) {
        const int64_t t = base + i * 64 + lane;
        const bool live = t < n;
        k[i] = live ? (ids ? sort_key(ids[t], n_rows) : key[t]) : 0;
        p[i] = live ? (ids ? (int32_t)t : pos[t]) : -1;
    }
#pragma unroll
    for (int i = 0; i < SORT_PER; ++i) {
        const uint32_t bin = (k[i] >> shift) & (bins - 1);
        uint64_t same = __ballot(p[i] >= 0);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot((bin >> b) & 1);
            same &= ((bin >> b) & 1) ? set : ~set;
        }
        if (p[i] >= 0) {
            const int before = __popcll(same & ((1ull << lane) - 1));
            const int32_t had = cnt[wave][bin];
            r[i] = had + before;
            // the last of the equal lanes writes the new count; the wave's other lanes have read the old one by then
            if ((same >> lane) == 1) cnt[wave][bin] = had + before + 1;
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    for (int b = tid; b < bins; b += 256) {
        int32_t at = first[b] + counts[(int64_t)b * gridDim.x + blockIdx.x];
#pragma unroll
        for (int w = 0; w < 4; ++w) { const int32_t c = cnt[w][b]; cnt[w][b] = at; at += c; }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SORT_PER; ++i)
        if (p[i] >= 0) {
            const int32_t at = cnt[wave][(k[i] >> shift) & (bins - 1)] + r[i];
            key_out[at] = k[i];
            pos_out[at] = p[i];
        }
}

// first[v] = number of sorted keys below v, v = 0 .. n_rows
__global__ __launch_bounds__(256) void k_row_first(const uint32_t *__restrict__ key, int32_t n, int64_t n_rows, int32_t *__restrict__ first)
{
    const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (v > n_rows) return;
    int32_t lo = 0, hi = n;
    while (lo < hi) { const int32_t mid = lo + ((hi - lo) >> 1); if (key[mid] < (uint32_t)v) lo = mid + 1; else hi = mid; }
    first[v] = lo;
}

// ------------------------------------------------------------------ sums
// A row with more than HEAVY tokens is summed in stretches that start at multiples of HEAVY of the sorted list, so that many
// groups share a popular row.  Such a row crosses a multiple of HEAVY, so a stretch holds at most two of them: the one it
// starts with (slot 0) and another it ends with (slot 1).
constexpr int HEAVY = 256;

// Sum of grad[pos[s .. e)], columns c .. c + V of this lane; the group's L lanes read L positions at once and hand them round
template <typename T, int V, int L>
__device__ __forceinline__ void sum_rows(const T *__restrict__ grad, int64_t stride, const int32_t *__restrict__ pos, int32_t s,
                                         int32_t e, int32_t c, int32_t d, int gl, float (&acc)[V])
{
    const bool in = c < d;
    for (int32_t a = s; a < e; a += L) {
        const int m = std::min<int32_t>(L, e - a);
        const int32_t mine = pos[a + (gl < m ? gl : 0)];
        int j = 0;
        for (; j + 4 <= m; j += 4) {
            float v[4][V];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int32_t p = __shfl(mine, j + i, L);
                load_vec<V>(grad + (int64_t)p * stride + (in ? c : 0), v[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int q = 0; q < V; ++q) acc[q] += v[i][q];
        }
        for (; j < m; ++j) {
            float v[V];
            const int32_t p = __shfl(mine, j, L);
            load_vec<V>(grad + (int64_t)p * stride + (in ? c : 0), v);
#pragma unroll
            for (int q = 0; q < V; ++q) acc[q] += v[q];
        }
    }
}

__device__ __forceinline__ int32_t first_of(const uint32_t *__restrict__ key, int32_t n, uint32_t v)
{
    int32_t lo = 0, hi = n;
    while (lo < hi) { const int32_t mid = lo + ((hi - lo) >> 1); if (key[mid] < v) lo = mid + 1; else hi = mid; }
    return lo;
}

template <typename T, int V, int L>
__global__ __launch_bounds__(256) void k_heavy_parts(const T *__restrict__ grad, int64_t stride, const uint32_t *__restrict__ key,
                                                     const int32_t *__restrict__ pos, int32_t n, int64_t n_rows, int32_t d,
                                                     const int32_t *__restrict__ first, float *__restrict__ parts)
{
    const int gl = threadIdx.x % L;
    const int32_t chunk = (int32_t)((int64_t)blockIdx.x * (256 / L) + threadIdx.x / L);
    const int64_t lo = (int64_t)chunk * HEAVY;
    if (lo >= n) return;
    const int32_t a = (int32_t)lo, z = (int32_t)std::min<int64_t>(n, lo + HEAVY);
    const uint32_t kf = key[a], kl = key[z - 1];
#pragma unroll 1
    for (int slot = 0; slot < 2; ++slot) {
        const uint32_t kk = slot ? kl : kf;
        if ((slot && kl == kf) || kk >= (uint64_t)n_rows) continue;
        const int32_t s = first ? first[kk] : first_of(key, n, kk), e = first ? first[kk + 1] : first_of(key, n, kk + 1);
        if (e - s <= HEAVY) continue;
        for (int32_t c0 = 0; c0 < d; c0 += V * L) {
            const int32_t c = c0 + gl * V;
            float acc[V] = {};
            sum_rows<T, V, L>(grad, stride, pos, std::max(s, a), std::min(e, z), c, d, gl, acc);
            if (c < d) {
                float *dst = parts + ((int64_t)chunk * 2 + slot) * d + c;
#pragma unroll
                for (int q = 0; q < V; ++q) dst[q] = acc[q];
            }
        }
    }
}

template <typename T, int V, int L>
__global__ __launch_bounds__(256) void k_row_sums(const T *__restrict__ grad, int64_t stride, const uint32_t *__restrict__ key,
                                                  const int32_t *__restrict__ pos, int32_t n, int64_t n_rows, int32_t d, float scale,
                                                  const int32_t *__restrict__ first, const float *__restrict__ parts, int accumulate,
                                                  T *__restrict__ out, int64_t out_stride)
{
    const int gl = threadIdx.x % L;
    const int64_t v = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (v >= n_rows) return;
    const int32_t s = first ? first[v] : first_of(key, n, (uint32_t)v), e = first ? first[v + 1] : first_of(key, n, (uint32_t)v + 1);
    if (s == e && accumulate) return;
    for (int32_t c0 = 0; c0 < d; c0 += V * L) {
        const int32_t c = c0 + gl * V;
        float acc[V] = {};
        if (e - s <= HEAVY) sum_rows<T, V, L>(grad, stride, pos, s, e, c, d, gl, acc);
        else if (c < d)
            for (int32_t k = s / HEAVY; k <= (e - 1) / HEAVY; ++k) {
                const float *src = parts + ((int64_t)k * 2 + ((int64_t)k * HEAVY < s)) * d + c;
#pragma unroll
                for (int q = 0; q < V; ++q) acc[q] += src[q];
            }
        if (c < d) {
            T *dst = out + v * out_stride + c;
            float was[V] = {};
            if (accumulate) load_vec<V>(dst, was);
#pragma unroll
            for (int q = 0; q < V; ++q) acc[q] = fmaf(acc[q], scale, was[q]);
            store_vec<V>(dst, acc);
        }
    }
}

// what a gradient call keeps in its workspace
struct GradPlan {
    int passes, bits, tiles;
    int64_t key[2], pos[2], counts, totals, first, parts, bytes;
};

GradPlan grad_plan(int64_t n, int64_t n_rows, int32_t d)
{
    GradPlan p = {};
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t o = at; at += align_up(bytes, 256); return o; };
    const bool small = n <= RANK_MAX;
    for (int i = 0; i < (small ? 1 : 2); ++i) { p.key[i] = take(n * 4); p.pos[i] = take(n * 4); }
    if (!small) {
        int bits = 1;
        while (bits < 31 && (n_rows >> bits)) ++bits;       // keys are 0 .. n_rows
        p.passes = (bits + 9) / 10;
        p.bits = (bits + p.passes - 1) / p.passes;
        p.tiles = (int)((n + SORT_TILE - 1) / SORT_TILE);
        p.counts = take((int64_t)(1 << p.bits) * p.tiles * 4);
        p.totals = take((int64_t)(1 << p.bits) * 4);
        p.first = take((n_rows + 1) * 4);
    }
    if (n > HEAVY) p.parts = take((n + HEAVY - 1) / HEAVY * 2 * (int64_t)d * 4);
    p.bytes = std::max<int64_t>(at, 256);
    return p;
}

template <typename T, int V, int L>
int launch_sums(const T *grad, int64_t stride, const uint32_t *key, const int32_t *pos, int32_t n, int64_t n_rows, int32_t d,
                float scale, int accumulate, const int32_t *first, float *parts, T *out, int64_t out_stride, hipStream_t st)
{
    constexpr int G = 256 / L;
    if (n > HEAVY) {
        const int64_t chunks = ((int64_t)n + HEAVY - 1) / HEAVY;
        hipLaunchKernelGGL((k_heavy_parts<T, V, L>), dim3((unsigned)((chunks + G - 1) / G)), dim3(256), 0, st, grad, stride, key, pos, n, n_rows, d,
                           first, parts);
    }
    hipLaunchKernelGGL((k_row_sums<T, V, L>), dim3((unsigned)((n_rows + G - 1) / G)), dim3(256), 0, st, grad, stride, key, pos, n, n_rows, d, scale,
                       first, parts, accumulate, out, out_stride);
    MF_LAUNCH_CHECK();
    return MFSGD_OK;
}

template <typename T, int V>
int launch_sums_v(int lanes, const T *grad, int64_t stride, const uint32_t *key, const int32_t *pos, int32_t n, int64_t n_rows,
                  int32_t d, float scale, int accumulate, const int32_t *first, float *parts, T *out, int64_t out_stride, hipStream_t st)
{
#define MF_SUM(L_) return launch_sums<T, V, L_>(grad, stride, key, pos, n, n_rows, d, scale, accumulate, first, parts, out, out_stride, st)
    if (lanes <= 8) MF_SUM(8);
    if (lanes <= 16) MF_SUM(16);
    if (lanes <= 32) MF_SUM(32);
    MF_SUM(64);
#undef MF_SUM
}

template <typename T>
int grad_impl(const T *grad, int64_t stride, const int32_t *ids, int64_t n, int64_t n_rows, int32_t d, float scale, int accumulate,
              T *out, int64_t out_stride, char *ws, hipStream_t st)
{
    const GradPlan p = grad_plan(n, n_rows, d);
    uint32_t *key[2] = {(uint32_t *)(ws + p.key[0]), (uint32_t *)(ws + p.key[1])};
    int32_t *pos[2] = {(int32_t *)(ws + p.pos[0]), (int32_t *)(ws + p.pos[1])};
    int32_t *first = nullptr;
    const int32_t m = (int32_t)n;
    int at = 0;
    if (n <= RANK_MAX) {
        if (n) hipLaunchKernelGGL(k_rank, dim3((unsigned)((n + 63) / 64)), dim3(64), 0, st, ids, m, n_rows, key[0], pos[0]);
    } else {
        int32_t *counts = (int32_t *)(ws + p.counts), *totals = (int32_t *)(ws + p.totals);
        for (int pass = 0; pass < p.passes; ++pass) {
            const int shift = pass * p.bits, from = (pass + 1) & 1;
            at = pass & 1;
            const int32_t *src = pass ? nullptr : ids;
            hipLaunchKernelGGL(k_sort_count, dim3(p.tiles), dim3(256), 0, st, key[from], src, m, n_rows, shift, 1 << p.bits, counts);
            hipLaunchKernelGGL(k_sort_tiles, dim3(1 << p.bits), dim3(64), 0, st, counts, p.tiles, totals);
            hipLaunchKernelGGL(k_sort_move, dim3(p.tiles), dim3(256), 0, st, key[from], pos[from], src, m, n_rows, shift, p.bits, counts,
                               totals, key[at], pos[at]);
        }
        first = (int32_t *)(ws + p.first);
        hipLaunchKernelGGL(k_row_first, dim3((unsigned)((n_rows + 256) / 256)), dim3(256), 0, st, key[at], m, n_rows, first);
    }
    float *parts = (float *)(ws + p.parts);
    const int v = vec_elems(sizeof(T), d, stride, out_stride, grad, out);
    const int lanes = (d + v - 1) / v;
#define MF_GRAD(V_) return launch_sums_v<T, V_>(lanes, grad, stride, key[at], pos[at], m, n_rows, d, scale, accumulate, first, parts, out, out_stride, st)
    if constexpr (sizeof(T) == 2) {
        if (v == 8) MF_GRAD(8);
    }
    if (v == 4) MF_GRAD(4);
    if (v == 2) MF_GRAD(2);
    MF_GRAD(1);
#undef MF_GRAD
}

}  // namespace

extern "C" {

int mfsgd_hip_embedding(const void *table, int64_t table_stride, int64_t n_rows, int32_t d, const int32_t *ids, int64_t n,
                        float scale, int32_t dtype, void *out, void *stream)
{
    MF_ARG(n >= 0 && n_rows >= 0 && n_rows <= INT32_MAX && d >= 1 && table_stride >= d, "embedding: bad shape");
    MF_ARG(dtype == MFSGD_F32 || dtype == MFSGD_BF16, "embedding: unknown dtype %d", dtype);
    if (n == 0) return MFSGD_OK;
    MF_ARG(ids && out && (table || n_rows == 0), "embedding: null pointer");
    if (dtype == MFSGD_F32)
        return launch_embedding<float>((const float *)table, table_stride, n_rows, d, ids, n, scale, (float *)out, as_stream(stream));
    return launch_embedding<__bf16>((const __bf16 *)table, table_stride, n_rows, d, ids, n, scale, (__bf16 *)out, as_stream(stream));
}

int64_t mfsgd_embedding_grad_workspace(int64_t n, int64_t n_rows, int32_t d)
{
    if (n < 0 || n >= INT32_MAX || n_rows < 0 || n_rows >= INT32_MAX || d < 1) return -1;
    return grad_plan(n, n_rows, d).bytes;
}

int mfsgd_hip_embedding_grad(const void *grad, int64_t grad_stride, const int32_t *ids, int64_t n, int64_t n_rows, int32_t d,
                             float scale, int32_t dtype, int32_t accumulate, void *out, int64_t out_stride, void *workspace,
                             int64_t workspace_bytes, void *stream)
{
    MF_ARG(n >= 0 && n < INT32_MAX && n_rows >= 0 && n_rows < INT32_MAX && d >= 1 && grad_stride >= d && out_stride >= d,
           "embedding_grad: bad shape (n and the table below 2^31 - 1 rows)");
    MF_ARG(dtype == MFSGD_F32 || dtype == MFSGD_BF16, "embedding_grad: unknown dtype %d", dtype);
    if (n_rows == 0 || (n == 0 && accumulate)) return MFSGD_OK;
    MF_ARG(out && (n == 0 || (grad && ids)), "embedding_grad: null pointer");
    MF_ARG(workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= grad_plan(n, n_rows, d).bytes,
           "embedding_grad: needs a 16-byte aligned workspace of %lld bytes", (long long)grad_plan(n, n_rows, d).bytes);
    if (dtype == MFSGD_F32)
        return grad_impl<float>((const float *)grad, grad_stride, ids, n, n_rows, d, scale, accumulate, (float *)out, out_stride,
                                (char *)workspace, as_stream(stream));
    return grad_impl<__bf16>((const __bf16 *)grad, grad_stride, ids, n, n_rows, d, scale, accumulate, (__bf16 *)out, out_stride,
                             (char *)workspace, as_stream(stream));
}

}  // extern "C"
