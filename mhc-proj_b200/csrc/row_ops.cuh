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
