// Pieces that the row kernels (layer_norm.cu, stream_mix.cu) share.
#pragma once

#include "mhc_common.cuh"
#include "mhc_proj.h"

namespace mhcp {

inline bool known_dtype(int dtype) { return dtype >= MHC_DTYPE_F32 && dtype <= MHC_DTYPE_F16; }

inline int elem_bytes(int dtype) { return dtype == MHC_DTYPE_F32 ? 4 : 2; }

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

// A thread's columns of a row, K of them, as the kernels move them:
//   VecCols     one 16-byte piece of consecutive columns.  For rows whose
//               starts are 16-byte aligned and whose width is whole pieces.
//   LooseCols   K columns `step` apart, one by one, so that a warp's lanes
//               are next to each other in memory; each is in the row or not.
template <class Elem>
struct VecCols {
    static constexpr int K = 16 / sizeof(Elem);
    int c0;  // < 0: none

    __device__ __forceinline__ VecCols(int first, bool in) : c0(in ? first : -1) {}
    __device__ __forceinline__ bool has(int) const { return c0 >= 0; }
    __device__ __forceinline__ int col(int j) const { return c0 + j; }

    __device__ __forceinline__ void load(const Elem* __restrict__ row, float (&v)[K]) const
    {
        uint4 q = make_uint4(0, 0, 0, 0);
        if (c0 >= 0) q = __ldg(reinterpret_cast<const uint4*>(row + c0));
        const Elem* e = reinterpret_cast<const Elem*>(&q);
#pragma unroll
        for (int j = 0; j < K; ++j) v[j] = to_f32(e[j]);
    }

    __device__ __forceinline__ void store(Elem* __restrict__ row, const float (&v)[K]) const
    {
        uint4 q;
        Elem* e = reinterpret_cast<Elem*>(&q);
#pragma unroll
        for (int j = 0; j < K; ++j) e[j] = from_f32<Elem>(v[j]);
        if (c0 >= 0) *reinterpret_cast<uint4*>(row + c0) = q;
    }
};

template <class Elem, int kCols>
struct LooseCols {
    static constexpr int K = kCols;
    int c0, step, C;

    __device__ __forceinline__ LooseCols(int first, int stride, int width) : c0(first), step(stride), C(width) {}
    __device__ __forceinline__ int col(int j) const { return c0 + j * step; }
    __device__ __forceinline__ bool has(int j) const { return static_cast<unsigned>(col(j)) < static_cast<unsigned>(C); }

    __device__ __forceinline__ void load(const Elem* __restrict__ row, float (&v)[K]) const
    {
#pragma unroll
        for (int j = 0; j < K; ++j) v[j] = has(j) ? to_f32(row[col(j)]) : 0.0f;
    }

    __device__ __forceinline__ void store(Elem* __restrict__ row, const float (&v)[K]) const
    {
#pragma unroll
        for (int j = 0; j < K; ++j)
            if (has(j)) row[col(j)] = from_f32<Elem>(v[j]);
    }
};

// Widths are ints in the kernels.
constexpr int64_t kMaxWidth = int64_t{1} << 30;

// Sums of K values over the block's threads, in every thread, in an order
// fixed by the block's size.  `buf` holds K floats per warp; the caller keeps
// two calls with the same buf apart (by a barrier or by alternating buffers).
template <int K>
__device__ __forceinline__ void block_sum(float (&v)[K], float* buf)
{
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], m);
    }
    const int warps = blockDim.x >> 5;
    if (warps == 1) return;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) buf[(threadIdx.x >> 5) * K + k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = buf[k];
    for (int w = 1; w < warps; ++w) {
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += buf[w * K + k];
    }
}

}  // namespace mhcp
