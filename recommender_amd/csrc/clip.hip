// clip.hip - the global norm of a set of gradients and their clipping (gfx950, MI355X).
//
//   norm = sqrt(sum_i sum g_i^2)          g_i <- g_i * min(1, max_norm / norm)
//
// Two launches: a workgroup per piece of at most `piece` elements writes the piece's sum of squares (float64, so that no
// square overflows or vanishes); in the second launch every workgroup adds all the partial sums in the same order by itself
// - which saves a launch and any waiting between workgroups - and scales its piece.  The set's pointers travel as kernel
// arguments (nothing is copied to the device, so the calls can be captured), CLIP_MAX tensors a launch.
// Bound by memory where the set is large (64 M fp32: 40 us for the sums, 6.4 TB/s, and 77 for the scaling, 6.6 TB/s with some
// of its reads out of the last-level cache), by two launches where it is small (624 K fp32: 16 us from Python).
#include <algorithm>
#include <math.h>
#include <stdlib.h>
#include "rows.h"

namespace {

// Tensors a launch: 28 bytes each of the 4 KB of kernel arguments.  The host writes all of them for every launch, so a set of a
// few tensors goes in a short list.
constexpr int CLIP_MAX = 128, CLIP_FEW = 8;
constexpr int64_t PIECE_MIN = 4096;    // elements
constexpr int PIECES = 1024;           // pieces a large set is cut into: four workgroups a CU

template <int MAX> struct ClipSet {
    const void *in[MAX];
    void *out[MAX];
    int64_t size[MAX];
    int32_t first[MAX];                // first piece of a tensor, counted from this launch's first; bit 31: bf16
    int32_t n_tensors;
};

// piece -> tensor: the last one whose first piece is not behind it (empty tensors have no piece)
template <int MAX>
__device__ __forceinline__ int tensor_of(const ClipSet<MAX> &set, int piece)
{
    int lo = 0, hi = set.n_tensors - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((set.first[mid] & 0x7fffffff) <= piece) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double block_sum(double v, double *red)
{
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    const double s = (red[0] + red[1]) + (red[2] + red[3]);
    __syncthreads();
    return s;
}

// Eight loads in flight a thread: the sums alone would wait for every load (64 M fp32, both launches: 162 -> 151 us)
template <typename T>
__device__ __forceinline__ double piece_squares(const T *__restrict__ p, int64_t n)
{
    constexpr int V = 16 / sizeof(T), U = 8;
    double s[U] = {};
    int64_t done = 0;
    if ((uintptr_t)p % 16 == 0) {
        const int64_t nv = n / V;
        int64_t i = threadIdx.x;
        for (; i + 256 * (U - 1) < nv; i += 256 * U) {
            float v[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) load_vec<V>(p + (i + 256 * u) * V, v[u]);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int q = 0; q < V; ++q) s[u] += (double)v[u][q] * v[u][q];
        }
        for (; i < nv; i += 256) {
            float v[V];
            load_vec<V>(p + i * V, v);
#pragma unroll
            for (int q = 0; q < V; ++q) s[0] += (double)v[q] * v[q];
        }
        done = nv * V;
    }
    for (int64_t i = done + threadIdx.x; i < n; i += 256) { const float v = load_f32(p + i); s[0] += (double)v * v; }
#pragma unroll
    for (int u = 1; u < U; ++u) s[0] += s[u];
    return s[0];
}

template <int MAX>
__global__ __launch_bounds__(256) void k_squares(const ClipSet<MAX> set, int64_t piece, double *__restrict__ partial)
{
    __shared__ double red[4];
    const int t = tensor_of(set, (int)blockIdx.x);
    const int64_t at = (int64_t)(blockIdx.x - (set.first[t] & 0x7fffffff)) * piece;
    const int64_t n = std::min<int64_t>(piece, set.size[t] - at);
    const double s = set.first[t] < 0 ? piece_squares((const __bf16 *)set.in[t] + at, n) : piece_squares((const float *)set.in[t] + at, n);
    const double sum = block_sum(s, red);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// every workgroup: the same sum in the same order
__device__ __forceinline__ float norm_of(const double *__restrict__ partial, int32_t n_partial, double *red)
{
    double s = 0;
    for (int i = threadIdx.x; i < n_partial; i += 256) s += partial[i];
    return (float)sqrt(block_sum(s, red));
}

__global__ __launch_bounds__(256) void k_norm(const double *__restrict__ partial, int32_t n_partial, float *__restrict__ norm)
{
    __shared__ double red[4];
    const float v = norm_of(partial, n_partial, red);
    if (threadIdx.x == 0) *norm = v;
}

// From the piece's end to its start, and past the caches on the way out: the set's last quarter gigabyte, read by the launch
// before, still lies in the last-level cache then, and what is written does not push it out (64 M fp32, out of place: 151 us
// forwards through the caches, 144 backwards, 125 past them, 120 both; 772 MB in all, of which 515 MB cannot be avoided)
template <typename T>
__device__ __forceinline__ void piece_scale(const T *p, T *o, int64_t n, float factor)
{
    constexpr int V = 16 / sizeof(T), U = 4;
    const bool wide = (uintptr_t)p % 16 == 0 && (uintptr_t)o % 16 == 0;
    const int64_t nv = wide ? n / V : 0, blocks = nv / (256 * U);
    for (int64_t i = nv * V + threadIdx.x; i < n; i += 256) store_f32(o + i, load_f32(p + i) * factor);
    auto scaled = [&](float (&v)[V], int64_t i) {
#pragma unroll
        for (int q = 0; q < V; ++q) v[q] *= factor;
        store_past<V>(o + i * V, v);
    };
    for (int64_t i = blocks * 256 * U + threadIdx.x; i < nv; i += 256) {
        float v[V];
        load_vec<V>(p + i * V, v);
        scaled(v, i);
    }
    for (int64_t b = 0; b < blocks; ++b) {
        const int64_t i = (blocks - 1 - b) * 256 * U + threadIdx.x;
        float v[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) load_vec<V>(p + (i + 256 * u) * V, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) scaled(v[u], i + 256 * u);
    }
}

template <int MAX>
__global__ __launch_bounds__(256) void k_clip(const ClipSet<MAX> set, int64_t piece, const double *__restrict__ partial, int32_t n_partial,
                                              float max_norm, float *__restrict__ norm, int first_launch)
{
    __shared__ double red[4];
    const float v = norm_of(partial, n_partial, red);
    if (first_launch && blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
    const float ratio = max_norm / v;
    const float factor = ratio > 1.f ? 1.f : ratio;          // not a number stays not a number
    const int t = tensor_of(set, (int)blockIdx.x);
    if (factor == 1.f && set.out[t] == set.in[t]) return;
    const int64_t at = (int64_t)(blockIdx.x - (set.first[t] & 0x7fffffff)) * piece;
    const int64_t n = std::min<int64_t>(piece, set.size[t] - at);
    if (set.first[t] < 0) piece_scale((const __bf16 *)set.in[t] + at, (__bf16 *)set.out[t] + at, n, factor);
    else piece_scale((const float *)set.in[t] + at, (float *)set.out[t] + at, n, factor);
}

// The size of a piece: about PIECES of them, multiples of PIECE_MIN so that every piece of an aligned tensor is aligned
int64_t piece_size(const int64_t *sizes, int32_t n)
{
    int64_t total = 0;
    for (int i = 0; i < n; ++i) total += sizes[i];
    return std::max(PIECE_MIN, align_up((total + PIECES - 1) / PIECES, PIECE_MIN));
}

int64_t piece_count(const int64_t *sizes, int32_t n, int64_t piece)
{
    int64_t c = 0;
    for (int i = 0; i < n; ++i) c += (sizes[i] + piece - 1) / piece;
    return c;
}

template <int MAX, typename F>
int for_sets(const void *const *in, void *const *out, const int64_t *sizes, const int32_t *dtypes, int32_t n, int64_t piece, F &&launch)
{
    int64_t before = 0;
    for (int a = 0; a < n;) {
        ClipSet<MAX> set;
        int32_t pieces = 0;
        set.n_tensors = 0;
        for (; a < n && set.n_tensors < MAX; ++a) {
            if (sizes[a] == 0) continue;
            const int i = set.n_tensors++;
            set.in[i] = in[a];
            set.out[i] = out ? out[a] : const_cast<void *>(in[a]);
            set.size[i] = sizes[a];
            set.first[i] = pieces | (dtypes[a] == MFSGD_BF16 ? INT32_MIN : 0);
            pieces += (int32_t)((sizes[a] + piece - 1) / piece);
        }
        if (set.n_tensors) launch(set, pieces, before);
        before += pieces;
    }
    MF_LAUNCH_CHECK();
    return MFSGD_OK;
}

int check_set(const char *who, const void *const *in, void *const *out, const int64_t *sizes, const int32_t *dtypes, int32_t n,
              float *norm, void *ws, int64_t ws_bytes)
{
    MF_ARG(n >= 0 && (n == 0 || (in && sizes && dtypes)) && norm, "%s: null pointer", who);
    for (int i = 0; i < n; ++i) {
        MF_ARG(sizes[i] >= 0 && (sizes[i] == 0 || (in[i] && (!out || out[i]))), "%s: tensor %d has a negative size or a null pointer", who, i);
        MF_ARG(dtypes[i] == MFSGD_F32 || dtypes[i] == MFSGD_BF16, "%s: tensor %d has the unknown dtype %d", who, i, dtypes[i]);
    }
    const int64_t need = mfsgd_grad_norm_workspace(sizes, n);
    MF_ARG(need >= 0, "%s: too many pieces", who);
    MF_ARG(ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need, "%s: needs a 16-byte aligned workspace of %lld bytes", who, (long long)need);
    return MFSGD_OK;
}

// What a call writes must not be written, or read as something else, by another of its workgroups: no two written stretches
// may meet, and a written stretch may meet only the gradient it replaces, and that exactly.
int check_apart(const char *who, const void *const *in, void *const *out, const int64_t *sizes, const int32_t *dtypes, int32_t n)
{
    struct Stretch { uintptr_t a, z; int32_t tensor, written; };
    Stretch *s = (Stretch *)malloc(sizeof(Stretch) * 2 * (size_t)(n + 1));
    MF_ARG(s, "%s: out of host memory", who);
    int m = 0, met = -1;
    for (int i = 0; i < n; ++i) {
        if (!sizes[i]) continue;
        const uintptr_t bytes = (uintptr_t)sizes[i] * (dtypes[i] == MFSGD_BF16 ? 2 : 4), a = (uintptr_t)in[i], o = out ? (uintptr_t)out[i] : a;
        s[m++] = {o, o + bytes, i, 1};
        if (o != a) s[m++] = {a, a + bytes, i, 0};
    }
    std::sort(s, s + m, [](const Stretch &x, const Stretch &y) { return x.a < y.a; });
    uintptr_t written_to = 0, read_to = 0;      // ends of the written and of the read stretches seen so far
    for (int k = 0; k < m && met < 0; ++k) {
        if (s[k].a < written_to || (s[k].written && s[k].a < read_to)) met = s[k].tensor;
        (s[k].written ? written_to : read_to) = std::max(s[k].written ? written_to : read_to, s[k].z);
    }
    free(s);
    MF_ARG(met < 0, "%s: tensor %d shares memory with another one of the call", who, met);
    return MFSGD_OK;
}

template <int MAX>
int squares(const void *const *in, const int64_t *sizes, const int32_t *dtypes, int32_t n, int64_t piece, double *partial, hipStream_t st)
{
    return for_sets<MAX>(in, nullptr, sizes, dtypes, n, piece, [&](const ClipSet<MAX> &set, int32_t pieces, int64_t before) {
        hipLaunchKernelGGL(k_squares<MAX>, dim3(pieces), dim3(256), 0, st, set, piece, partial + before);
    });
}

template <int MAX>
int clip(const void *const *in, void *const *out, const int64_t *sizes, const int32_t *dtypes, int32_t n, int64_t piece, int32_t pieces,
         float max_norm, float *norm, double *partial, hipStream_t st)
{
    if (const int rc = squares<MAX>(in, sizes, dtypes, n, piece, partial, st)) return rc;
    int first = 1;
    return for_sets<MAX>(in, out, sizes, dtypes, n, piece, [&](const ClipSet<MAX> &set, int32_t count, int64_t) {
        hipLaunchKernelGGL(k_clip<MAX>, dim3(count), dim3(256), 0, st, set, piece, partial, pieces, max_norm, norm, first);
        first = 0;
    });
}

}  // namespace

extern "C" {

int64_t mfsgd_grad_norm_workspace(const int64_t *h_sizes, int32_t n_tensors)
{
    if (n_tensors < 0 || (n_tensors && !h_sizes)) return -1;
    for (int i = 0; i < n_tensors; ++i) if (h_sizes[i] < 0 || h_sizes[i] > ((int64_t)1 << 50)) return -1;
    return align_up(std::max<int64_t>(1, piece_count(h_sizes, n_tensors, piece_size(h_sizes, n_tensors))) * 8, 256);
}

int mfsgd_hip_grad_norm(const void *const *h_grads, const int64_t *h_sizes, const int32_t *h_dtypes, int32_t n_tensors, float *norm,
                        void *workspace, int64_t workspace_bytes, void *stream)
{
    if (const int rc = check_set("grad_norm", h_grads, nullptr, h_sizes, h_dtypes, n_tensors, norm, workspace, workspace_bytes)) return rc;
    const int64_t piece = piece_size(h_sizes, n_tensors);
    const int32_t pieces = (int32_t)piece_count(h_sizes, n_tensors, piece);
    const auto sum = n_tensors <= CLIP_FEW ? squares<CLIP_FEW> : squares<CLIP_MAX>;
    if (const int rc = sum(h_grads, h_sizes, h_dtypes, n_tensors, piece, (double *)workspace, as_stream(stream))) return rc;
    hipLaunchKernelGGL(k_norm, dim3(1), dim3(256), 0, as_stream(stream), (const double *)workspace, pieces, norm);
    MF_LAUNCH_CHECK();
    return MFSGD_OK;
}

int mfsgd_hip_clip_grads(const void *const *h_grads, void *const *h_out, const int64_t *h_sizes, const int32_t *h_dtypes,
                         int32_t n_tensors, float max_norm, float *norm, void *workspace, int64_t workspace_bytes, void *stream)
{
    if (const int rc = check_set("clip_grads", h_grads, h_out, h_sizes, h_dtypes, n_tensors, norm, workspace, workspace_bytes)) return rc;
    MF_ARG(max_norm > 0, "clip_grads: max_norm must be positive");
    if (const int rc = check_apart("clip_grads", h_grads, h_out, h_sizes, h_dtypes, n_tensors)) return rc;
    const int64_t piece = piece_size(h_sizes, n_tensors);
    const int32_t pieces = (int32_t)piece_count(h_sizes, n_tensors, piece);
    hipStream_t st = as_stream(stream);
    double *partial = (double *)workspace;
    if (pieces == 0) {
        hipLaunchKernelGGL(k_norm, dim3(1), dim3(256), 0, st, partial, 0, norm);
        MF_LAUNCH_CHECK();
        return MFSGD_OK;
    }
    const auto run = n_tensors <= CLIP_FEW ? clip<CLIP_FEW> : clip<CLIP_MAX>;
    return run(h_grads, h_out, h_sizes, h_dtypes, n_tensors, piece, pieces, max_norm, norm, partial, st);
}

}  // extern "C"
