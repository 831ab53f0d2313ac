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

// N consecutive elements starting at p, which is aligned to their size: one load / store of up to 16 bytes
template <int N> __device__ __forceinline__ void load_vec(const float *p, float (&v)[N])
{
    if constexpr (N == 4) { const float4 t = *(const float4 *)p; v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w; }
    else if constexpr (N == 2) { const float2 t = *(const float2 *)p; v[0] = t.x; v[1] = t.y; }
    else v[0] = *p;
}
template <int N> __device__ __forceinline__ void load_vec(const __bf16 *p, float (&v)[N])
{
    if constexpr (N == 1) v[0] = (float)*p;
    else {
        uint32_t w[N / 2];
        if constexpr (N == 8) { const uint4 t = *(const uint4 *)p; w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w; }
        else if constexpr (N == 4) { const uint2 t = *(const uint2 *)p; w[0] = t.x; w[1] = t.y; }
        else w[0] = *(const uint32_t *)p;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) { v[2 * i] = bf16_lo(w[i]); v[2 * i + 1] = bf16_hi(w[i]); }
    }
}
template <int N> __device__ __forceinline__ void store_vec(float *p, const float (&v)[N])
{
    if constexpr (N == 4) *(float4 *)p = make_float4(v[0], v[1], v[2], v[3]);
    else if constexpr (N == 2) *(float2 *)p = make_float2(v[0], v[1]);
    else *p = v[0];
}
template <int N> __device__ __forceinline__ void store_vec(__bf16 *p, const float (&v)[N])
{
    if constexpr (N == 1) *p = (__bf16)v[0];
    else {
        uint32_t w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
        if constexpr (N == 8) *(uint4 *)p = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (N == 4) *(uint2 *)p = make_uint2(w[0], w[1]);
        else *(uint32_t *)p = w[0];
    }
}

// ... past the caches (V elements are 4, 8 or 16 bytes; one bf16 element goes through them)
template <int N, typename T> __device__ __forceinline__ void store_past(T *p, const float (&v)[N])
{
    constexpr int W = N * sizeof(T) / 4;
    if constexpr (W == 0) store_vec<N>(p, v);
    else {
        uint32_t w[W];
#pragma unroll
        for (int i = 0; i < W; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
            else w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
        }
        typedef uint32_t words __attribute__((ext_vector_type(W)));
        words x;
        if constexpr (W == 1) x = (words)w[0];
        else {
#pragma unroll
            for (int i = 0; i < W; ++i) x[i] = w[i];
        }
        __builtin_nontemporal_store(x, (words *)p);
    }
}

// Elements one access may take when every row starts at `stride` elements behind the one before: the largest power of two
// that divides the row length, every stride and every pointer, at most 16 bytes.
static inline int vec_elems(int elem_size, int64_t row, int64_t stride_a, int64_t stride_b, const void *a, const void *b)
{
    int v = 16 / elem_size;
    while (v > 1 && (row % v || stride_a % v || stride_b % v || (uintptr_t)a % ((size_t)v * elem_size) ||
                     (uintptr_t)b % ((size_t)v * elem_size))) v /= 2;
    return v;
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
