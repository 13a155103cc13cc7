// Pieces that the row kernels (layer_norm.cu, stream_mix.cu) share.
#pragma once

#include <cstring>
#include <type_traits>

#include "mhc_common.cuh"
#include "mhc_proj.h"

namespace mhcp {

inline bool known_dtype(int dtype) { return dtype >= MHC_DTYPE_F32 && dtype <= MHC_DTYPE_F16; }

// Whether an array (which may be null) starts at one of its elements' addresses:
// a load from another one is a fault.
inline bool at_element(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <class... Pointers>
inline bool at_elements(int dtype, Pointers... p)
{
    return (at_element(p, dtype == MHC_DTYPE_F32 ? 4 : 2) && ...);
}

// Element i of an array whose type is known at run time only: the small
// operands (per-token coefficients, a norm's weight and bias).
__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype)
{
    switch (dtype) {
        case MHC_DTYPE_BF16: return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
        case MHC_DTYPE_F16: return to_f32(static_cast<const __half*>(p)[i]);
        default: return static_cast<const float*>(p)[i];
    }
}

__device__ __forceinline__ void store_any(void* p, int64_t i, int dtype, float v)
{
    switch (dtype) {
        case MHC_DTYPE_BF16: static_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v); break;
        case MHC_DTYPE_F16: static_cast<__half*>(p)[i] = from_f32<__half>(v); break;
        default: static_cast<float*>(p)[i] = v;
    }
}

// Two columns at a time: packed fp32 arithmetic, one instruction for two
// results (the row kernels have few instruction slots per byte).
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

// Holds values in registers: the compiler may otherwise load them again in
// each turn of a loop, as it can see that they do not change.
template <int kPairs>
__device__ __forceinline__ void keep(float2 (&v)[kPairs])
{
#pragma unroll
    for (int i = 0; i < kPairs; ++i) asm volatile("" : "+f"(v[i].x), "+f"(v[i].y));
}

// Elements 2 i and 2 i + 1 of a 16-byte piece.
template <class Elem>
__device__ __forceinline__ float2 pair_of(const uint4& q, int i)
{
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (sizeof(Elem) == 4) {
        return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    } else if constexpr (std::is_same<Elem, __nv_bfloat16>::value) {
        return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    } else {
        __half2 h;
        memcpy(&h, &w[i], 4);
        return __half22float2(h);
    }
}

// The 16-byte piece of K elements.
template <class Elem, int kPairs>
__device__ __forceinline__ uint4 piece_of(const float2 (&v)[kPairs])
{
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        if constexpr (sizeof(Elem) == 4) {
            w[2 * i] = __float_as_uint(v[i].x);
            w[2 * i + 1] = __float_as_uint(v[i].y);
        } else if constexpr (std::is_same<Elem, __nv_bfloat16>::value) {
            const __nv_bfloat162 h = __float22bfloat162_rn(v[i]);
            memcpy(&w[i], &h, 4);
        } else {
            const __half2 h = __float22half2_rn(v[i]);
            memcpy(&w[i], &h, 4);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Widths are ints in the kernels, rows a dimension of a grid.
constexpr int64_t kMaxWidth = int64_t{1} << 30, kMaxRows = (int64_t{1} << 31) - 1;

inline bool rows_ok(int64_t N, int64_t C) { return N >= 0 && N <= kMaxRows && C >= 1 && C <= kMaxWidth; }

// The threads that work on one row: 4, 8, 16 or 32 lanes of a warp, or several
// whole warps; a block may hold more than one such group, block (threads,
// groups), and each has a barrier of its own.
struct Group {
    int threads, t, id;
    unsigned lanes;  // of the warp, the group's

    __device__ __forceinline__ Group()
        : threads(blockDim.x), t(threadIdx.x), id(threadIdx.y),
          lanes(blockDim.x >= 32 ? 0xffffffffu
                                 : ((1u << blockDim.x) - 1) << (threadIdx.x + threadIdx.y * blockDim.x & 31 & ~(blockDim.x - 1)))
    {
    }
    __device__ __forceinline__ bool one_warp() const { return threads <= 32; }
    __device__ __forceinline__ int warps() const { return threads >> 5; }

    __device__ __forceinline__ void sync() const
    {
        if (threads <= 32)
            __syncwarp(lanes);
        else if (blockDim.y == 1)
            __syncthreads();
        else
            asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(threads) : "memory");
    }
    // Sums over the group's lanes of a warp.
    template <int K>
    __device__ __forceinline__ void lane_sum(float (&v)[K]) const
    {
        for (int m = min(threads, 32) >> 1; m > 0; m >>= 1) {
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(lanes, v[k], m);
        }
    }
};

// Sums of K values over a group's threads, in every thread, in an order fixed
// by the group's size.  `buf`: 32 K floats of the group at a 16-byte boundary
// that group_sum_init has seen; the caller keeps two calls with the same buf
// apart (by a barrier or by alternating buffers).
template <int K>
__device__ __forceinline__ void group_sum_init(const Group& g, float* buf)
{
    // parts of warps that the group does not have: added as zeros
    if (!g.one_warp() && g.t >= g.warps() && g.t < 32) {
#pragma unroll
        for (int k = 0; k < K; ++k) buf[k * 32 + g.t] = 0.0f;
    }
}

template <int K>
__device__ __forceinline__ void group_sum(const Group& g, float (&v)[K], float* buf)
{
    if (g.one_warp()) {
        g.lane_sum(v);
        return;
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], m);
    }
    if ((g.t & 31) == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) buf[k * 32 + (g.t >> 5)] = v[k];
    }
    g.sync();
    float4 f[K];
#pragma unroll
    for (int k = 0; k < K; ++k) f[k] = *reinterpret_cast<const float4*>(buf + k * 32);
    for (int w = 4; w < g.warps(); w += 4) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const float4 o = *reinterpret_cast<const float4*>(buf + k * 32 + w);
            f[k] = make_float4(f[k].x + o.x, f[k].y + o.y, f[k].z + o.z, f[k].w + o.w);
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = (f[k].x + f[k].y) + (f[k].z + f[k].w);
}

}  // namespace mhcp
