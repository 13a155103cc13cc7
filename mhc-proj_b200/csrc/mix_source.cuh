// What the mix kernels share.
#pragma once

#include "philox.cuh"
#include "row_ops.cuh"

namespace mhcp {

template <class Elem>
struct MixIn {
    const Elem* x;
    int64_t stride, stream_stride;
    const Elem* y;
    int64_t y_stride;
    const void *T, *h;
    int T_dtype, h_dtype;
};

// A token's coefficients.
struct MixCoef {
    float t[16], h[4];
};

// kWide: T and h are fp32 and 16-byte aligned.
template <bool kWide, class Elem>
__device__ __forceinline__ MixCoef mix_coef(const MixIn<Elem>& in, int64_t r)
{
    MixCoef k;
    if constexpr (kWide) {
        const float4* t = reinterpret_cast<const float4*>(in.T) + 4 * r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 f = __ldg(t + i);
            k.t[4 * i] = f.x;
            k.t[4 * i + 1] = f.y;
            k.t[4 * i + 2] = f.z;
            k.t[4 * i + 3] = f.w;
        }
        const float4 f = __ldg(reinterpret_cast<const float4*>(in.h) + r);
        k.h[0] = f.x;
        k.h[1] = f.y;
        k.h[2] = f.z;
        k.h[3] = f.w;
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) k.t[i] = load_any(in.T, 16 * r + i, in.T_dtype);
#pragma unroll
        for (int i = 0; i < 4; ++i) k.h[i] = load_any(in.h, 4 * r + i, in.h_dtype);
    }
    return k;
}

// The 20 sums of a token in one warp.  Instead of a butterfly per value, each
// step halves the values a lane holds: it keeps one half and hands the other
// to its partner.  Lane l ends with value `l` for l < 20 (slot order below).
__device__ __forceinline__ float warp_sum20(const float (&a)[20])
{
    const int lane = threadIdx.x & 31;
    float b[16], rest[4];
#pragma unroll
    for (int i = 0; i < 16; ++i) b[i] = a[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) rest[i] = a[16 + i];
    // 16 values over the lanes' bits 0..3, then bit 4: lane l has value l & 15
#pragma unroll
    for (int m = 8, bit = 8; m >= 1; m >>= 1, bit >>= 1) {
        const bool up = lane & bit;
#pragma unroll
        for (int i = 0; i < m; ++i) {
            const float give = up ? b[i] : b[i + m];
            const float mine = up ? b[i + m] : b[i];
            b[i] = mine + __shfl_xor_sync(0xffffffffu, give, bit);
        }
    }
    b[0] += __shfl_xor_sync(0xffffffffu, b[0], 16);
    // 4 values over bits 0..1, then bits 2..4: lane l has value l & 3
#pragma unroll
    for (int m = 2, bit = 2; m >= 1; m >>= 1, bit >>= 1) {
        const bool up = lane & bit;
#pragma unroll
        for (int i = 0; i < m; ++i) {
            const float give = up ? rest[i] : rest[i + m];
            const float mine = up ? rest[i + m] : rest[i];
            rest[i] = mine + __shfl_xor_sync(0xffffffffu, give, bit);
        }
    }
#pragma unroll
    for (int bit = 4; bit <= 16; bit <<= 1) rest[0] += __shfl_xor_sync(0xffffffffu, rest[0], bit);
    return lane < 16 ? b[0] : rest[0];
}

// A thread adds up a token's terms for its 20 sums in 32 bits over runs of so many
// columns' pairs; the runs are added up in 64 bits, so that the rounding of a
// token of 2^30 columns is that of a short one.
constexpr int kMixRun = 256;

// Sum number `mine` (warp_sum20's order) of a token.
template <class Elem>
__device__ __forceinline__ void put_token_sum(const MixIn<Elem>& in, int64_t r, int mine, float sum, void* dT, void* dh)
{
    if (mine < 16)
        store_any(dT, 16 * r + mine, in.T_dtype, sum);
    else if (mine < 20)
        store_any(dh, 4 * r + mine - 16, in.h_dtype, sum);
}

// Writes the sums of a token that `lanes` lanes share, from each lane's part
// (kLong: of the last run, and lane l has sum l of the runs before it).
template <bool kLong = false, class Elem>
__device__ __forceinline__ void put_token_sums(const MixIn<Elem>& in, int64_t r, bool live, int lane, int lanes,
                                               float (&v)[20], void* dT, void* dh, double before = 0.0)
{
    if (lanes == 32) {
        float sum = warp_sum20(v);
        if constexpr (kLong) sum = static_cast<float>(before + sum);
        if (live) put_token_sum(in, r, lane, sum, dT, dh);
        return;
    }
    for (int m = lanes >> 1; m > 0; m >>= 1) {
#pragma unroll
        for (int i = 0; i < 20; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
    }
    if (!live) return;
    const int mine = lane & (lanes - 1);
#pragma unroll
    for (int q = 0; q < 5; ++q) {
        if ((q & (lanes - 1)) != mine) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (q < 4)
                store_any(dT, 16 * r + 4 * q + i, in.T_dtype, v[4 * q + i]);
            else
                store_any(dh, 4 * r + i, in.h_dtype, v[16 + i]);
        }
    }
}

}  // namespace mhcp
