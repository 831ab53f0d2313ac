// embedding.hip - lookup of a batch of table rows with scaling, and its gradient by sorted tokens (gfx950, MI355X).
//
//   out[t] = scale * table[ids[t]]                       dtable[v] = scale * sum_{t: ids[t] = v} grad[t]
//
// The gradient sorts the batch's positions by id (stable: equal ids stay in the order of t), so that a table row's tokens
// are one stretch of the sorted list; a row is then summed by one group of lanes in fp32, in the order of t, and written
// once.  A popular row is cut where the sorted list is at multiples of 16 or 32, summed by many groups and joined.  No floating-point atomics: the same inputs give the same bits.
//
// 2 M tokens of 512 bytes into 480189 rows: 373 us, of which the sums take 270 (1.28 GB: 4.7 TB/s, a copy reaches 5.1) and the
// sort and the rows' first places the rest.  131072 bf16 tokens of 256 bytes: 56 us, eight launches of 3 to 20 us that wait for
// each other; the sums would be 10 us at a copy's rate.  1000 tokens: 17 us, three launches.
#include <algorithm>
#include <math.h>
#include "rows.h"

namespace {

// a group's step behind the last token, or column, still fits 32 bits
constexpr int64_t MAX_TOKENS = ((int64_t)1 << 31) - 1024, MAX_ROW = (int64_t)1 << 30;

// ------------------------------------------------------------------ lookup
// A thread moves PIECES pieces of V elements (one access each), all of them asked for before
// the first one is used; the pieces of the output are numbered through.  A row's last piece ends with the row: where V does not
// divide the width it repeats some of the piece before, with the same values.  Bound by memory: 1 M bf16 rows of 200 bytes 42 us (5.1 TB/s, what a copy reaches; 96 us
// with one piece a thread); 32 rows: the launch, 8.4 us from Python.
constexpr int PIECES = 4;
template <typename T, int V, bool PAST>
__global__ __launch_bounds__(256) void k_embedding(const T *table, int64_t stride, int64_t n_rows, int32_t d,
                                                   const int32_t *__restrict__ ids, int64_t n, float scale, T *out)
{
    constexpr int U = PIECES;
    const int32_t per = (d + V - 1) / V;
    const int64_t p0 = group_id() * (256 * U), t0 = p0 / per;          // the same for all threads
    const int32_t skip = (int32_t)(p0 - t0 * per);
    int32_t id[U], c[U];
    uint32_t to[U];                     // behind the first row's start: at most two rows and 1024 pieces
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t x = skip + u * 256 + threadIdx.x;
        const uint32_t row = x / (uint32_t)per;
        c[u] = std::min((int32_t)(x - row * per) * V, d - V);
        to[u] = row * (uint32_t)d + c[u];
        id[u] = ids[std::min<int64_t>(t0 + row, n - 1)];
    }
    float v[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) load_vec<V>(table + (id[u] >= 0 && id[u] < n_rows ? id[u] * stride + c[u] : 0), v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t p = p0 + u * 256 + threadIdx.x;
#pragma unroll
        for (int i = 0; i < V; ++i) v[u][i] = id[u] < 0 ? 0.f : id[u] < n_rows ? v[u][i] * scale : NAN;
        if (p < n * per) {
            T *dst = out + t0 * d + to[u];
            if constexpr (PAST) store_past<V>(dst, v[u]);
            else store_vec<V>(dst, v[u]);
        }
    }
}

template <typename T>
int launch_embedding(const T *table, int64_t stride, int64_t n_rows, int32_t d, const int32_t *ids, int64_t n, float scale,
                     T *out, hipStream_t st)
{
    if (n_rows == 0) { table = out; stride = 0; }       // nothing is taken from it, but the first piece is always asked for
    constexpr int WIDE = 16 / sizeof(T), HALF = 8 / sizeof(T);
    // Pieces of 16 bytes where all of them are aligned, else of 8 (2 M bf16 rows of 254 bytes: 156 us by 8, 159 by 16 and 300 by
    // elements; of 264 bytes: 155 by 8, 163 by 16)
    const bool aligned = d % WIDE == 0 && stride % WIDE == 0 && (uintptr_t)table % 16 == 0 && (uintptr_t)out % 16 == 0;
    const int v = aligned ? WIDE : d >= HALF ? HALF : 1;
    // A large output goes past the caches, which then hold the table: into memory not written lately 1 M rows of 200 bytes take 42
    // us against 68, 2 M of 512 bytes 224 against 321.  One that fits the L2s twice stays there for whoever reads it next
    const bool past = n * d * (int64_t)sizeof(T) > ((int64_t)64 << 20);
    const dim3 grid = grid_of((n * ((d + v - 1) / v) + 256 * PIECES - 1) / (256 * PIECES));
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, table, stride, n_rows, d, ids, n, scale, out); };
    if (v == WIDE) go(past ? k_embedding<T, WIDE, true> : k_embedding<T, WIDE, false>);
    else if (v == HALF) go(past ? k_embedding<T, HALF, true> : k_embedding<T, HALF, false>);
    else go(past ? k_embedding<T, 1, true> : k_embedding<T, 1, false>);
    MF_LAUNCH_CHECK();
    return MFSGD_OK;
}

// ------------------------------------------------------------------ positions sorted by id
// Keys: an id inside the table, or n_rows for everything else (padding, ids behind the table), which sorts to the end.
__device__ __forceinline__ uint32_t sort_key(int32_t id, int64_t n_rows)
{
    return (uint32_t)id < (uint64_t)n_rows ? (uint32_t)id : (uint32_t)n_rows;
}

// Small batches: the rank of position t is the number of smaller keys plus the number of equal keys in front of it.  16 lanes
// rank one position, a sixteenth of the keys each, read from LDS four at a time; one launch, no passes.  With `first` the groups
// behind the positions' do the same for the table's rows: first[v] is the number of keys below v, v = 0 .. n_rows.
constexpr int RANK_MAX = 8192;
__global__ __launch_bounds__(256) void k_rank(const int32_t *__restrict__ ids, int32_t n, int64_t n_rows, uint2 *__restrict__ sorted,
                                              int32_t *__restrict__ first)
{
    __shared__ __attribute__((aligned(16))) uint32_t keys[RANK_MAX];
    const int n4 = (n + 3) & ~3, part = threadIdx.x & 15;
    for (int i = threadIdx.x; i < n4; i += 256) keys[i] = i < n ? sort_key(ids[i], n_rows) : 0xffffffffu;
    __syncthreads();
    const int t_groups = (n + 15) / 16, group = blockIdx.x;
    const bool of_row = group >= t_groups;
    const int t = of_row ? -1 : group * 16 + (threadIdx.x >> 4);            // of a row: no equal key counts
    const int64_t v = (int64_t)(group - t_groups) * 16 + (threadIdx.x >> 4);
    const uint32_t mine = of_row ? (uint32_t)v : keys[t < n ? t : 0];
    int32_t rank = 0;
    for (int i = 4 * part; i < n4; i += 64) {
        const uint4 k = *(const uint4 *)(keys + i);
        const uint32_t below = mine + (i + 3 < t);              // in front of t equal keys count as smaller
        rank += (k.x < below) + (k.y < below) + (k.z < below) + (k.w < below);
        if (i <= t && t <= i + 3) rank += (k.x == mine && i < t) + (k.y == mine && i + 1 < t) + (k.z == mine && i + 2 < t);
    }
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) rank += __shfl_xor(rank, m, 16);
    if (part) return;
    if (of_row) { if (v <= n_rows) first[v] = rank; }
    else if (t < n) sorted[rank] = make_uint2(mine, (uint32_t)t);
}

// Large batches: least significant digit first, up to ten bits a pass, stable.  A tile is 256 PER consecutive entries of one
// workgroup; a pass counts every tile's digits, turns the counts into first places and moves the entries.  An entry is (key,
// position).  Bound by latency and LDS atomics, not by the 16 to 32 MB that a pass over 2 M entries moves: 14 + 6 + 23 us.
constexpr int SORT_BINS = 1024;

template <int PER>
__global__ __launch_bounds__(256) void k_sort_count(const uint2 *__restrict__ in, const int32_t *__restrict__ ids, int32_t n,
                                                    int64_t n_rows, int shift, int bins, int32_t *__restrict__ counts)
{
    __shared__ int32_t cnt[SORT_BINS];
    for (int b = threadIdx.x; b < bins; b += 256) cnt[b] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * (256 * PER);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int64_t t = base + i * 256 + threadIdx.x;
        if (t < n) {
            const uint32_t k = ids ? sort_key(ids[t], n_rows) : in[t].x;
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

template <int PER>
__global__ __launch_bounds__(256) void k_sort_move(const uint2 *__restrict__ in, const int32_t *__restrict__ ids, int32_t n, int64_t n_rows,
                                                   int shift, int bits, const int32_t *__restrict__ counts,
                                                   const int32_t *__restrict__ totals, uint2 *__restrict__ out)
{
    __shared__ int32_t cnt[4][SORT_BINS];
    __shared__ uint64_t peers[4][SORT_BINS];
    __shared__ int32_t first[SORT_BINS];
    __shared__ int32_t part[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bins = 1 << bits;
    for (int b = tid; b < 4 * SORT_BINS; b += 256) { (&cnt[0][0])[b] = 0; (&peers[0][0])[b] = 0; }
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
    // a wave takes 64 PER consecutive entries, 64 at a time: a lane's place among the wave's entries of its bin
    const int64_t base = (int64_t)blockIdx.x * (256 * PER) + wave * (64 * PER);
    uint32_t k[PER];
    int32_t p[PER], r[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int64_t t = base + i * 64 + lane;
        const bool live = t < n;
        if (ids) {
            k[i] = live ? sort_key(ids[t], n_rows) : 0;
            p[i] = live ? (int32_t)t : -1;
        } else {
            const uint2 e = live ? in[t] : make_uint2(0u, ~0u);
            k[i] = e.x;
            p[i] = (int32_t)e.y;
        }
    }
    // The lanes of a bin find each other through a word in LDS that each sets its bit in (ten ballots of the digit's bits and
    // their logic took three times the instructions: a pass over 2 M entries 29 -> 23 us)
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const uint32_t bin = (k[i] >> shift) & (bins - 1);
        const bool live = p[i] >= 0;
        if (live) atomicOr((unsigned long long *)&peers[wave][bin], 1ull << lane);
        asm volatile("" ::: "memory");          // a wave's LDS operations keep their order; the compiler has to as well
        if (live) {
            const uint64_t same = peers[wave][bin];
            const int32_t had = cnt[wave][bin];
            const int before = __popcll(same & ((1ull << lane) - 1));
            r[i] = had + before;
            asm volatile("" ::: "memory");
            // the last of the equal lanes leaves the new count and a clear word; the others have read both by then
            if ((same >> lane) == 1) { cnt[wave][bin] = had + before + 1; peers[wave][bin] = 0; }
        }
        asm volatile("" ::: "memory");
    }
    __syncthreads();
    for (int b = tid; b < bins; b += 256) {
        int32_t at = first[b] + counts[(int64_t)b * gridDim.x + blockIdx.x];
#pragma unroll
        for (int w = 0; w < 4; ++w) { const int32_t c = cnt[w][b]; cnt[w][b] = at; at += c; }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (p[i] >= 0) {
            const int32_t at = cnt[wave][(k[i] >> shift) & (bins - 1)] + r[i];
            out[at] = make_uint2(k[i], (uint32_t)p[i]);
        }
}

// ------------------------------------------------------------------ sums
// A row with more than 2^hs tokens is summed in stretches that start at multiples of 2^hs of the sorted list, so that many
// groups of lanes share a popular row.  Such a row crosses a multiple of 2^hs, so a stretch holds at most two of them: the one
// it starts with (slot 0) and another it ends with (slot 1).  The same again, SUPER stretches at a time, for rows of more than
// SUPER stretches.
constexpr int SUPER = 32;

// Lane gl of a group of L takes V columns, from here on; a row's last lane takes its last V, some of them another lane's as well
__device__ __forceinline__ int32_t column(int32_t c, int32_t d, int V) { return std::min(c, d - V); }

// Sum of grad[positions s .. e), columns c .. c + V of this lane; the group's L lanes read L positions at once and hand them round
template <typename T, int V, int L>
__device__ __forceinline__ void sum_rows(const T *__restrict__ grad, int64_t stride, const uint2 *__restrict__ sorted, int32_t s,
                                         int32_t e, int32_t c, int gl, float (&acc)[V])
{
    const T *base = grad + c;
    for (int32_t a = s; a < e; a += L) {
        const int m = std::min<int32_t>(L, e - a);
        const int32_t mine = (int32_t)sorted[a + (gl < m ? gl : 0)].y;
        int j = 0;
        for (; j + 8 <= m; j += 8) {
            float v[8][V];
#pragma unroll
            for (int i = 0; i < 8; ++i) load_vec<V>(base + (int64_t)__shfl(mine, j + i, L) * stride, v[i]);
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int q = 0; q < V; ++q) acc[q] += v[i][q];
        }
        if (j < m) {                    // up to seven more, asked for at once
            float v[7][V];
#pragma unroll
            for (int i = 0; i < 7; ++i) {
                const int32_t p = __shfl(mine, j + i < m ? j + i : j, L);
#pragma unroll
                for (int q = 0; q < V; ++q) v[i][q] = 0.f;
                if (j + i < m) load_vec<V>(base + (int64_t)p * stride, v[i]);
            }
#pragma unroll
            for (int i = 0; i < 7; ++i)
#pragma unroll
                for (int q = 0; q < V; ++q) acc[q] += v[i][q];
        }
    }
}

// parts k0 + g, k0 + g + step, .. k1 of a row, of which the first, k0, is in slot 1 if the row starts inside it
template <int V>
__device__ __forceinline__ void sum_parts(const float *__restrict__ parts, int32_t k0, int32_t k1, int64_t start, int64_t width, int32_t c,
                                          int32_t d, float (&acc)[V], int g = 0, int step = 1)
{
    const int64_t inside = (int64_t)k0 * width < start;
    const float *src = parts + (int64_t)k0 * 2 * d + c;
    const int32_t m = k1 - k0;
#pragma unroll 8
    for (int32_t k = g; k <= m; k += step) {
        float v[V];
        load_vec<V>(src + (k ? (int64_t)k * 2 : inside) * d, v);
#pragma unroll
        for (int q = 0; q < V; ++q) acc[q] += v[q];
    }
}

// Two things the sums need, in one launch.  The first `heavy_groups` workgroups sum the heavy rows' stretches, a group of L lanes
// each; it finds what it has to know about its two rows in the keys around it: a row that holds a position of the stretch has
// more than 2^hs tokens exactly if more than 2^hs of them lie no farther than 2^hs from the stretch.  The other workgroups write
// first[v], the number of sorted keys below v, for v = 0 .. n_rows.
template <typename T, int V, int L>
__global__ __launch_bounds__(256) void k_spread(const T *__restrict__ grad, int64_t stride, const uint2 *__restrict__ sorted, int32_t n,
                                                int64_t n_rows, int32_t d, int hs, int heavy_groups, float *__restrict__ parts, int32_t *__restrict__ first)
{
    if (group_id() >= heavy_groups) {
        const int64_t v = (group_id() - heavy_groups) * 256 + threadIdx.x;
        if (v > n_rows) return;
        int32_t lo = 0, hi = n;
        while (lo < hi) { const int32_t mid = lo + ((hi - lo) >> 1); if (sorted[mid].x < (uint32_t)v) lo = mid + 1; else hi = mid; }
        first[v] = lo;
        return;
    }
    const int gl = threadIdx.x % L, width = 1 << hs;
    const int64_t lo = (group_id() * (256 / L) + threadIdx.x / L) << hs;
    if (lo >= n) return;
    const int32_t a = (int32_t)lo, z = (int32_t)std::min<int64_t>(n, lo + width);
    const uint32_t kf = sorted[a].x, kl = sorted[z - 1].x;
    uint32_t count = 0;                 // a byte each: tokens of kf near by, of kf in the stretch, of kl near by, of kl in the stretch
    for (int i = gl; i < 3 * width; i += L) {
        const int64_t t = lo - width + i;
        if (t < 0 || t >= n) continue;
        const uint32_t k = sorted[t].x, in = (t >= a && t < z) << 8 | 1;
        count += (k == kf ? in : 0) + (k == kl ? in << 16 : 0);
    }
#pragma unroll
    for (int m = 1; m < L; m <<= 1) count += __shfl_xor(count, m, L);
#pragma unroll 1
    for (int slot = 0; slot < 2; ++slot) {
        const uint32_t kk = slot ? kl : kf, c2 = count >> (16 * slot);
        if ((slot && kl == kf) || kk >= (uint64_t)n_rows || (int)(c2 & 255) <= width) continue;
        const int32_t m = (c2 >> 8) & 255, s = slot ? z - m : a, e = s + m;
        for (int32_t c0 = 0; c0 < d; c0 += V * L) {
            const int32_t c = c0 + gl * V;
            float acc[V] = {};
            sum_rows<T, V, L>(grad, stride, sorted, s, e, column(c, d, V), gl, acc);
            if (c < d) store_vec<V>(parts + ((lo >> hs) * 2 + slot) * d + column(c, d, V), acc);
        }
    }
}

__device__ __forceinline__ int32_t stretches(int32_t s, int32_t e, int hs) { return ((e - 1) >> hs) - (s >> hs) + 1; }

// one workgroup a super-stretch of SUPER parts; a thread a column
__global__ __launch_bounds__(256) void k_super_parts(const uint2 *__restrict__ sorted, int32_t n, int64_t n_rows, int32_t d,
                                                     const int32_t *__restrict__ first, int hs, const float *__restrict__ parts, float *__restrict__ supers)
{
    const int64_t lo = (int64_t)blockIdx.x * (SUPER << hs);
    const int32_t a = (int32_t)lo, z = (int32_t)std::min<int64_t>(n, lo + (SUPER << hs));
    const uint32_t kf = sorted[a].x, kl = sorted[z - 1].x;
    for (int slot = 0; slot < 2; ++slot) {
        const uint32_t kk = slot ? kl : kf;
        if ((slot && kl == kf) || kk >= (uint64_t)n_rows) continue;
        const int32_t s = first[kk], e = first[kk + 1];
        if (stretches(s, e, hs) <= SUPER) continue;
        for (int32_t c = threadIdx.x; c < d; c += 256) {
            float acc[1] = {};
            sum_parts<1>(parts, std::max(s, a) >> hs, (std::min(e, z) - 1) >> hs, s, 1 << hs, c, d, acc);
            supers[((int64_t)blockIdx.x * 2 + slot) * d + c] = acc[0];
        }
    }
}

// The rows' sums.  The first `joins` workgroups join the parts of the heavy rows: a group of L lanes a stretch, for the heavy
// row that starts in it (there is one at most: it goes on behind the stretch); a row of more than SUPER stretches, of which a
// workgroup starts one at most, by all its groups, or (supers) from the sums of SUPER stretches.  The others sum the light rows: a group takes R
// neighbouring rows, whose tokens are neighbours in the sorted list - one wait for the rows' first places, one for the tokens'
// positions and one for every eight gradient rows, whichever row they belong to.  A table row has two or three tokens where the
// batch is as long as the table, and a wait a step and row would be most of the time.
template <typename T, int V, int L, int R>
__global__ __launch_bounds__(256) void k_row_sums(const T *__restrict__ grad, int64_t stride, const uint2 *__restrict__ sorted, int32_t n,
                                                  int64_t n_rows, int32_t d, float scale, const int32_t *__restrict__ first, int hs, int joins,
                                                  const float *__restrict__ parts, const float *__restrict__ supers, int accumulate,
                                                  T *__restrict__ out, int64_t out_stride)
{
    const int gl = threadIdx.x % L;
    auto put = [&](float (&acc)[V], int64_t v, int32_t c, bool any) {
        if (c < d && (any || !accumulate)) {
            const int32_t c1 = column(c, d, V);
            T *dst = out + v * out_stride + c1;
            float was[V] = {};
            if (accumulate) load_vec<V>(dst, was);
            const float f = any ? scale : 0.f;  // a row without tokens is zero whatever the scale is
#pragma unroll
            for (int q = 0; q < V; ++q) was[q] = fmaf(acc[q], f, was[q]);
            if (accumulate && c1 < c) {         // the columns of another lane: not a second time
#pragma unroll
                for (int q = 0; q < V; ++q) if (c1 + q >= c) store_f32(dst + q, was[q]);
            } else store_vec<V>(dst, was);
        }
#pragma unroll
        for (int q = 0; q < V; ++q) acc[q] = 0.f;
    };
    const int64_t group = group_id();
    if (group < joins) {
        __shared__ int32_t big[3];
        __shared__ float sums[256 / L][V * L];
        if (threadIdx.x == 0) big[2] = -1;
        __syncthreads();
        const int64_t a = (group * (256 / L) + threadIdx.x / L) << hs;
        const uint32_t v = a < n ? sorted[std::min<int64_t>(n, a + (1 << hs)) - 1].x : ~0u;
        if (v < (uint64_t)n_rows) {
            const int32_t s = first[v], e = first[v + 1];
            if (e - s > 1 << hs && s >= a) {
                const bool many = stretches(s, e, hs) > SUPER;
                if (many && !supers) { if (gl == 0) { big[0] = s; big[1] = e; big[2] = (int32_t)v; } }
                else
                    for (int32_t c = gl * V; c < d; c += V * L) {
                        float acc[V] = {};
                        if (!many) sum_parts<V>(parts, s >> hs, (e - 1) >> hs, s, 1 << hs, column(c, d, V), d, acc);
                        else sum_parts<V>(supers, s / (SUPER << hs), (e - 1) / (SUPER << hs), s, SUPER << hs, column(c, d, V), d, acc);
                        put(acc, v, c, true);
                    }
            }
        }
        __syncthreads();
        const int32_t s = big[0], e = big[1], row = big[2];
        if (row < 0) return;
        const int g = threadIdx.x / L;
        for (int32_t c0 = 0; c0 < d; c0 += V * L) {
            const int32_t c = c0 + gl * V;
            float acc[V] = {};
            if (c < d) sum_parts<V>(parts, s >> hs, (e - 1) >> hs, s, 1 << hs, column(c, d, V), d, acc, g, 256 / L);
#pragma unroll
            for (int q = 0; q < V; ++q) sums[g][gl * V + q] = acc[q];
            __syncthreads();
            if (g == 0) {
#pragma unroll 1
                for (int k = 1; k < 256 / L; ++k)
#pragma unroll
                    for (int q = 0; q < V; ++q) acc[q] += sums[k][gl * V + q];
                put(acc, row, c, true);
            }
            __syncthreads();
        }
        return;
    }
    const int64_t v0 = ((group - joins) * (256 / L) + threadIdx.x / L) * R;
    if (v0 >= n_rows) return;
    const int rows = (int)std::min<int64_t>(R, n_rows - v0);
    const int64_t vf = v0 + std::min(gl, rows);
    const int32_t f = first[vf];
    const int32_t f_next = __shfl(f, gl < R ? gl + 1 : R, L);
    const int lead = (threadIdx.x & 63) / L * L;         // the group's first lane
    const uint32_t heavy = (uint32_t)(__ballot(gl < rows && f_next - f > 1 << hs) >> lead) & ((1u << R) - 1);
    for (int32_t c0 = 0; c0 < d; c0 += V * L) {
        const int32_t c = c0 + gl * V;
        float acc[V] = {};
        const T *base = grad + column(c, d, V);
        for (int r = 0; r < rows; ++r) {
            if ((heavy >> r) & 1) continue;
            const int stop = std::min(rows, r + __builtin_ctz((heavy >> r) | 1u << R));     // rows r .. stop: none of them heavy
            int32_t s = __shfl(f, r, L), e = __shfl(f, r + 1, L);        // of the row in work
            const int32_t e0 = __shfl(f, stop, L);
            for (int32_t a = s; a < e0; a += L) {
                const int m = std::min<int32_t>(L, e0 - a);
                const int32_t mine = (int32_t)sorted[a + (gl < m ? gl : 0)].y;
                for (int j = 0; j < m; j += 8) {
                    float v[8][V];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int32_t p = __shfl(mine, j + i < m ? j + i : j, L);
                        if (j + i < m) load_vec<V>(base + (int64_t)p * stride, v[i]);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (j + i < m) {
                            while (a + j + i >= e) {             // behind the row: it is done, and so are empty ones after it
                                put(acc, v0 + r, c, e > s);
                                ++r;
                                s = e;
                                e = __shfl(f, r + 1, L);
                            }
#pragma unroll
                            for (int q = 0; q < V; ++q) acc[q] += v[i][q];
                        }
                }
            }
            for (; r < stop; ++r) {
                put(acc, v0 + r, c, e > s);
                s = e;
                e = __shfl(f, r + 2 <= rows ? r + 2 : rows, L);
            }
            --r;                                                 // the loop's own step
        }
    }
}

// what a gradient call keeps in its workspace
struct GradPlan {
    int passes, bits, per, tiles, hs;
    bool use_supers;
    int64_t sorted[2], counts, totals, first, parts, supers, bytes;
};

GradPlan grad_plan(int64_t n, int64_t n_rows, int32_t d)
{
    GradPlan p = {};
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t o = at; at += align_up(bytes, 256); return o; };
    const bool small = n <= RANK_MAX;
    for (int i = 0; i < (small ? 1 : 2); ++i) p.sorted[i] = take(n * 8);
    if (!small) {
        int bits = 1;
        while (bits < 31 && (n_rows >> bits)) ++bits;       // keys are 0 .. n_rows
        p.passes = (bits + 9) / 10;
        p.bits = (bits + p.passes - 1) / p.passes;
        // small tiles fill the chip, large ones keep the table of counts short: the change is where either has a tile a CU
        p.per = n <= 256 * 1024 ? 4 : 16;
        p.tiles = (int)((n + 256 * p.per - 1) / (256 * p.per));
        p.counts = take((int64_t)(1 << p.bits) * p.tiles * 4);
        p.totals = take((int64_t)(1 << p.bits) * 4);
    }
    p.first = take((n_rows + 1) * 4);
    // Short stretches keep the wait for a popular row short (131072 tokens of bf16, d = 128: 74 us with 16, 85 with 32, 102
    // with 64), long ones write and read fewer parts (2 M tokens of fp32: 432, 405 and 402 us)
    p.hs = n <= RANK_MAX || n > 256 * 1024 ? 5 : 4;
    if (n > 1 << p.hs) p.parts = take(((n + (1 << p.hs) - 1) >> p.hs) * 2 * (int64_t)d * 4);
    // A row's parts joined by one workgroup, or first 32 and 32 of them in a launch of their own, which costs 2 to 6 us whatever the
    // batch is and pays where one row has most of it; the host does not see how long the longest row is.  The bound is where a
    // batch of one row alone would take more than twice an ordinary one's time without that launch.  Popular items of 59047, and
    // all tokens of one row, d = 128, us without / with it:
    //    65536 tokens  fp32 41 / 44 and  63 / 46    bf16 47 / 49 and  54 / 46
    //   131072         fp32 49 / 54 and  98 / 61    bf16 56 / 62 and  76 / 61
    //   196608         fp32 57 / 62 and 133 / 74    bf16 62 / 67 and  98 / 74
    //   262144         fp32 66 / 71 and 167 / 88    bf16 67 / 72 and 124 / 90
    p.use_supers = n > 128 * 1024;
    if (p.use_supers) p.supers = take((n + (SUPER << p.hs) - 1) / (SUPER << p.hs) * 2 * (int64_t)d * 4);
    p.bytes = std::max<int64_t>(at, 256);
    return p;
}

template <typename T> struct SumArgs {
    const T *grad;
    int64_t stride;
    const uint2 *sorted;
    int32_t n;
    int64_t n_rows;
    int32_t d;
    float scale;
    int accumulate;
    int32_t *first;
    bool has_first;                     // else it is to be found
    int hs;
    float *parts, *supers;              // supers NULL: not used
    T *out;
    int64_t out_stride;
};

template <typename T, int V, int L>
int launch_sums(const SumArgs<T> &a, hipStream_t st)
{
    constexpr int G = 256 / L;
    const int64_t chunks = a.n > 1 << a.hs ? ((int64_t)a.n + (1 << a.hs) - 1) >> a.hs : 0;
    const int joins = (int)((chunks + G - 1) / G);
    const int64_t spread = joins + (a.has_first ? 0 : (a.n_rows + 256) / 256);
    if (spread)
        hipLaunchKernelGGL((k_spread<T, V, L>), grid_of(spread), dim3(256), 0, st, a.grad, a.stride, a.sorted, a.n, a.n_rows, a.d, a.hs, joins,
                           a.parts, a.first);
    if (chunks && a.supers)
        hipLaunchKernelGGL(k_super_parts, dim3((unsigned)((chunks + SUPER - 1) / SUPER)), dim3(256), 0, st, a.sorted, a.n, a.n_rows, a.d,
                           (const int32_t *)a.first, a.hs, (const float *)a.parts, a.supers);
    constexpr int R = 4, per_group = G * R;           // rows a group (131072 tokens, 59047 rows: 66 us with 2 or 4, 74 with 8), rows a workgroup
    hipLaunchKernelGGL((k_row_sums<T, V, L, R>), grid_of(joins + (a.n_rows + per_group - 1) / per_group), dim3(256), 0, st, a.grad,
                       a.stride, a.sorted, a.n, a.n_rows, a.d, a.scale, (const int32_t *)a.first, a.hs, joins, (const float *)a.parts, (const float *)a.supers, a.accumulate, a.out,
                       a.out_stride);
    MF_LAUNCH_CHECK();
    return MFSGD_OK;
}

// Rows shorter than 16 bytes go by elements, others by pieces of 16 bytes
template <typename T>
int launch_sums_d(const SumArgs<T> &a, hipStream_t st)
{
    constexpr int V = 16 / sizeof(T);
    if (a.d < V) return launch_sums<T, 1, 8>(a, st);
    const int lanes = (a.d + V - 1) / V;
    if (lanes <= 8) return launch_sums<T, V, 8>(a, st);
    if (lanes <= 16) return launch_sums<T, V, 16>(a, st);
    if (lanes <= 32) return launch_sums<T, V, 32>(a, st);
    return launch_sums<T, V, 64>(a, st);
}

template <typename T>
int grad_impl(const T *grad, int64_t stride, const int32_t *ids, int64_t n, int64_t n_rows, int32_t d, float scale, int accumulate,
              T *out, int64_t out_stride, char *ws, hipStream_t st)
{
    const GradPlan p = grad_plan(n, n_rows, d);
    uint2 *sorted[2] = {(uint2 *)(ws + p.sorted[0]), (uint2 *)(ws + p.sorted[1])};
    const int32_t m = (int32_t)n;
    int32_t *first = (int32_t *)(ws + p.first);
    int at = 0;
    bool has_first = false;
    if (n <= RANK_MAX) {
        // The rows' first places by ranking while that is less than a launch (32 tokens of a 17770-row table 18.5 -> 14.9 us, 1000
        // of 1682 rows 19.5 -> 18.0; 8000 of 16000 rows would take 57 instead of 42)
        has_first = n && n_rows <= 65536 && n * n_rows <= 1 << 25;
        if (n) hipLaunchKernelGGL(k_rank, dim3((unsigned)((n + 15) / 16 + (has_first ? (n_rows + 16) / 16 : 0))), dim3(256), 0, st, ids, m, n_rows,
                                  sorted[0], first);
    } else {
        int32_t *counts = (int32_t *)(ws + p.counts), *totals = (int32_t *)(ws + p.totals);
        for (int pass = 0; pass < p.passes; ++pass) {
            const int shift = pass * p.bits;
            const uint2 *in = sorted[(pass + 1) & 1];
            at = pass & 1;
            const int32_t *src = pass ? nullptr : ids;
            if (p.per == 4) hipLaunchKernelGGL(k_sort_count<4>, dim3(p.tiles), dim3(256), 0, st, in, src, m, n_rows, shift, 1 << p.bits, counts);
            else hipLaunchKernelGGL(k_sort_count<16>, dim3(p.tiles), dim3(256), 0, st, in, src, m, n_rows, shift, 1 << p.bits, counts);
            hipLaunchKernelGGL(k_sort_tiles, dim3(1 << p.bits), dim3(64), 0, st, counts, p.tiles, totals);
            if (p.per == 4) hipLaunchKernelGGL(k_sort_move<4>, dim3(p.tiles), dim3(256), 0, st, in, src, m, n_rows, shift, p.bits,
                                               (const int32_t *)counts, (const int32_t *)totals, sorted[at]);
            else hipLaunchKernelGGL(k_sort_move<16>, dim3(p.tiles), dim3(256), 0, st, in, src, m, n_rows, shift, p.bits,
                                    (const int32_t *)counts, (const int32_t *)totals, sorted[at]);
        }
    }
    const SumArgs<T> a = {grad, stride, sorted[at], m, n_rows, d, scale, accumulate, first, has_first, p.hs, (float *)(ws + p.parts),
                          p.use_supers ? (float *)(ws + p.supers) : nullptr, out, out_stride};
    return launch_sums_d(a, st);
}

}  // namespace

extern "C" {

int mfsgd_hip_embedding(const void *table, int64_t table_stride, int64_t n_rows, int32_t d, const int32_t *ids, int64_t n,
                        float scale, int32_t dtype, void *out, void *stream)
{
    MF_ARG(n >= 0 && n_rows >= 0 && n_rows <= INT32_MAX && d >= 1 && d <= MAX_ROW && table_stride >= d, "embedding: bad shape");
    MF_ARG(dtype == MFSGD_F32 || dtype == MFSGD_BF16, "embedding: unknown dtype %d", dtype);
    if (n == 0) return MFSGD_OK;
    MF_ARG(n <= ((int64_t)1 << 40) / d, "embedding: more than 2^40 elements");
    MF_ARG(ids && out && (table || n_rows == 0), "embedding: null pointer");
    if (dtype == MFSGD_F32)
        return launch_embedding<float>((const float *)table, table_stride, n_rows, d, ids, n, scale, (float *)out, as_stream(stream));
    return launch_embedding<__bf16>((const __bf16 *)table, table_stride, n_rows, d, ids, n, scale, (__bf16 *)out, as_stream(stream));
}

int64_t mfsgd_embedding_grad_workspace(int64_t n, int64_t n_rows, int32_t d)
{
    if (n < 0 || n > MAX_TOKENS || n_rows < 0 || n_rows >= INT32_MAX || d < 1 || d > MAX_ROW) return -1;
    return grad_plan(n, n_rows, d).bytes;
}

int mfsgd_hip_embedding_grad(const void *grad, int64_t grad_stride, const int32_t *ids, int64_t n, int64_t n_rows, int32_t d,
                             float scale, int32_t dtype, int32_t accumulate, void *out, int64_t out_stride, void *workspace,
                             int64_t workspace_bytes, void *stream)
{
    MF_ARG(n >= 0 && n <= MAX_TOKENS && n_rows >= 0 && n_rows < INT32_MAX && d >= 1 && d <= MAX_ROW && grad_stride >= d && out_stride >= d,
           "embedding_grad: bad shape (n at most 2^31 - 1024, the table below 2^31 - 1 rows, rows of at most 2^30 elements)");
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
