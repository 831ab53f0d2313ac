// rows.h - what the minibatch operators share (embedding.hip, softmax_loss.hip, clip.hip): float32 and bfloat16 rows, moved
// a few elements at a time.
#pragma once
#include "common.h"

// ---- bf16 <-> fp32 for the minibatch operators (round to nearest even; v_cvt_pk_bf16_f32 on gfx950)
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ uint32_t pack_bf16(float a, float b)
{
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ __forceinline__ float load_f32(const float *p) { return *p; }
__device__ __forceinline__ float load_f32(const __bf16 *p) { return (float)*p; }
__device__ __forceinline__ void store_f32(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_f32(__bf16 *p, float v) { *p = (__bf16)v; }

// N consecutive elements starting at p: one load / store of up to 16 bytes.  p is aligned to an element, no more: the hardware
// takes vector accesses at any address, so rows of odd widths move in the same pieces as even ones.
template <int W, int ALIGN> struct Words { typedef uint32_t type __attribute__((ext_vector_type(W), aligned(ALIGN), may_alias)); };
template <> struct Words<1, 2> { typedef uint32_t type __attribute__((aligned(2), may_alias)); };
template <> struct Words<1, 4> { typedef uint32_t type __attribute__((may_alias)); };
template <int N, typename T> using words_of = typename Words<(N * sizeof(T) + 3) / 4, sizeof(T)>::type;

template <int N, typename T> __device__ __forceinline__ void load_vec(const T *p, float (&v)[N])
{
    constexpr int W = N * sizeof(T) / 4;
    if constexpr (W == 0) v[0] = load_f32(p);
    else {
        const words_of<N, T> t = *(const words_of<N, T> *)p;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            uint32_t w;
            if constexpr (W == 1) w = t; else w = t[i];
            if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(w);
            else { v[2 * i] = bf16_lo(w); v[2 * i + 1] = bf16_hi(w); }
        }
    }
}
template <int N, typename T> __device__ __forceinline__ words_of<N, T> words_from(const float (&v)[N])
{
    words_of<N, T> t;
#pragma unroll
    for (int i = 0; i < (int)(N * sizeof(T) / 4); ++i) {
        uint32_t w;
        if constexpr (sizeof(T) == 4) w = __float_as_uint(v[i]);
        else w = pack_bf16(v[2 * i], v[2 * i + 1]);
        if constexpr (N * sizeof(T) == 4) t = w; else t[i] = w;
    }
    return t;
}
template <int N, typename T> __device__ __forceinline__ void store_vec(T *p, const float (&v)[N])
{
    if constexpr (N * sizeof(T) < 4) store_f32(p, v[0]);
    else *(words_of<N, T> *)p = words_from<N, T>(v);
}
// ... past the caches (one bf16 element goes through them)
template <int N, typename T> __device__ __forceinline__ void store_past(T *p, const float (&v)[N])
{
    if constexpr (N * sizeof(T) < 4) store_f32(p, v[0]);
    else __builtin_nontemporal_store(words_from<N, T>(v), (words_of<N, T> *)p);
}

static inline int64_t align_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// A dimension of a grid holds fewer than 2^32 threads: workgroups from 2^22 on go on in the second dimension.  The last ones may
// be more than were asked for; every kernel launched like this looks at its own number.
static inline dim3 grid_of(int64_t groups)
{
    const int64_t x = (int64_t)1 << 22;
    return groups <= x ? dim3((unsigned)groups) : dim3((unsigned)x, (unsigned)((groups + x - 1) / x));
}
__device__ __forceinline__ int64_t group_id() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }
