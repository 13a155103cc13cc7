// The residual update of an mHC layer with n = 4 streams, forward and
// backward: per token, with T its 4x4 mixing matrix (a projection's output),
// h its four output weights and y the sublayer's output,
//   X'[i] = sum_j T[i, j] X[j] + h[i] drop(y)
// and given G = dL/dX'
//   dX[j] = sum_i T[i, j] G[i]         dT[i, j] = sum_c G[i] X[j]
//   dy = drop(sum_i h[i] G[i])         dh[i] = sum_c G[i] drop(y)
// drop is dropout.cu's with the element's index in the (tokens, C) array y, so
// the fused form is the composition with dropout's output left unrounded.
// Arithmetic and sums are fp32; outputs are rounded once.
#include <algorithm>

#include "philox.cuh"
#include "row_ops.cuh"

namespace mhcp {

#ifndef MHC_MIXF_T
#define MHC_MIXF_T 256
#endif
constexpr int kMixBlock = 256;

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

template <class Elem>
__device__ __forceinline__ MixCoef mix_coef(const MixIn<Elem>& in, int64_t r)
{
    MixCoef k;
#pragma unroll
    for (int i = 0; i < 16; ++i) k.t[i] = load_any(in.T, 16 * r + i, in.T_dtype);
#pragma unroll
    for (int i = 0; i < 4; ++i) k.h[i] = load_any(in.h, 4 * r + i, in.h_dtype);
    return k;
}

// A thread's columns of a row, K of them, as the kernels move them:
//   MixVecCols     one 16-byte piece of consecutive columns.  For rows whose
//               starts are 16-byte aligned and whose width is whole pieces.
//   MixLooseCols   K columns `step` apart, one by one, so that a warp's lanes
//               are next to each other in memory; each is in the row or not.
template <class Elem>
struct MixVecCols {
    static constexpr int K = 16 / sizeof(Elem);
    int c0;  // < 0: none

    __device__ __forceinline__ MixVecCols(int first, bool in) : c0(in ? first : -1) {}
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
struct MixLooseCols {
    static constexpr int K = kCols;
    int c0, step, C;

    __device__ __forceinline__ MixLooseCols(int first, int stride, int width) : c0(first), step(stride), C(width) {}
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

// How a token's columns are spread over its threads, kLanes threads of a
// group at a time:
//   MixVec     16-byte pieces; piece v's draws are one half or the whole of a
//              group of eight elements, since a row of whole pieces starts at
//              a multiple of its length
//   MixLoose   any width and alignment: a warp takes 256 columns (K per lane
//              and step, 32 apart), counted from the last multiple of eight
//              elements before the row, so that lane l's one call of the
//              generator gives the draws of the warp's columns 8 l .. 8 l + 7,
//              which the lanes hand round
template <class Elem>
struct MixVec {
    using Cols = MixVecCols<Elem>;
    static constexpr int K = Cols::K;
    int64_t first;  // element index of the row's start in y
    int C, t, threads;

    __device__ __forceinline__ MixVec(int64_t r, int width, int thread, int of)
        : first(r * width), C(width), t(thread), threads(of)
    {
    }
    __device__ __forceinline__ int steps() const { return (C / K + threads - 1) / threads; }
    __device__ __forceinline__ Cols cols(int step) const
    {
        const int c = (step * threads + t) * K;
        return Cols(c, c < C);
    }
    // Bit j: column j of `cols(step)` is kept.
    __device__ __forceinline__ uint32_t keep(int step, const Dropout& d, uint2 key) const
    {
        const int64_t e = first + (step * threads + t) * K;
        return keep_bits(e >> 3, d.offset, key, d.limit) >> (e & 7);
    }
};

template <class Elem, int kCols>
struct MixLoose {
    using Cols = MixLooseCols<Elem, kCols>;
    static constexpr int K = Cols::K;
    static constexpr int kParts = 8 / K;  // steps to a warp's 256 columns
    int64_t group;                        // of eight elements, the row's first
    int shift, C, warp, lane, warps;
    uint32_t bits = 0;

    __device__ __forceinline__ MixLoose(int64_t r, int width, int thread, int of)
        : group(r * width >> 3), shift(static_cast<int>(r * width & 7)), C(width), warp(thread >> 5), lane(thread & 31),
          warps(of >> 5)
    {
    }
    __device__ __forceinline__ int steps() const { return (C + shift + 256 * warps - 1) / (256 * warps) * kParts; }
    __device__ __forceinline__ int chunk(int step) const { return (step / kParts * warps + warp) * 256; }
    __device__ __forceinline__ Cols cols(int step) const
    {
        return Cols(chunk(step) + step % kParts * (32 * K) + lane - shift, 32, C);
    }
    // All lanes of the warp call it, step by step.
    __device__ __forceinline__ uint32_t keep(int step, const Dropout& d, uint2 key)
    {
        if (step % kParts == 0) bits = keep_bits(group + (chunk(step) >> 3) + lane, d.offset, key, d.limit);
        uint32_t k = 0;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int from = 4 * (step % kParts * K + j) + (lane >> 3);
            k |= (__shfl_sync(0xffffffffu, bits, from) >> (lane & 7) & 1u) << j;
        }
        return k;
    }
};

// y with its dropped elements at zero.
template <int K>
__device__ __forceinline__ void drop(float (&y)[K], uint32_t keep, float scale)
{
#pragma unroll
    for (int j = 0; j < K; ++j) y[j] = (keep >> j & 1u) ? y[j] * scale : 0.0f;
}

// Block: (threads of a token, tokens).
template <class Elem, class Map>
__global__ void __launch_bounds__(kMixBlock)
mix_fwd_kernel(MixIn<Elem> in, Elem* __restrict__ out, Dropout d, int64_t N, int C)
{
    constexpr int K = Map::K;
    const int64_t r = blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y;
    if (r >= N) return;
    const uint2 key = dropout_key(d);
    const Elem* x = in.x + r * in.stride;
    const Elem* yr = in.y + r * in.y_stride;
    Elem* o = out + r * 4 * C;
    Map map(r, C, threadIdx.x, blockDim.x);
    const MixCoef k = mix_coef(in, r);
    const int steps = map.steps();
    for (int s = 0; s < steps; ++s) {
        const typename Map::Cols cols = map.cols(s);
        float v[4][K], y[K];
#pragma unroll
        for (int j = 0; j < 4; ++j) cols.load(x + j * in.stream_stride, v[j]);
        cols.load(yr, y);
        if (d.limit) drop(y, map.keep(s, d, key), d.scale);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a[K];
#pragma unroll
            for (int c = 0; c < K; ++c) {
                a[c] = k.h[i] * y[c];
#pragma unroll
                for (int j = 0; j < 4; ++j) a[c] = fmaf(k.t[4 * i + j], v[j][c], a[c]);
            }
            cols.store(o + static_cast<int64_t>(i) * C, a);
        }
    }
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

template <class Elem, class Map>
__global__ void __launch_bounds__(kMixBlock)
mix_bwd_kernel(const Elem* __restrict__ g, int64_t g_stride, int64_t g_stream_stride, MixIn<Elem> in,
               Elem* __restrict__ dx, void* __restrict__ dT, Elem* __restrict__ dy, void* __restrict__ dh, Dropout d,
               int64_t N, int C)
{
    constexpr int K = Map::K;
    __shared__ float part[kMixBlock / 32][20];
    const int64_t r = blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y;
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    float sum = 0.0f;
    if (r < N) {
        const uint2 key = dropout_key(d);
        const Elem* x = in.x + r * in.stride;
        const Elem* yr = in.y + r * in.y_stride;
        const Elem* gr = g + r * g_stride;
        Elem* dxr = dx + r * 4 * C;
        Map map(r, C, threadIdx.x, blockDim.x);
        const MixCoef k = mix_coef(in, r);
        float acc[20];
#pragma unroll
        for (int i = 0; i < 20; ++i) acc[i] = 0.0f;
        const int steps = map.steps();
        for (int s = 0; s < steps; ++s) {
            const typename Map::Cols cols = map.cols(s);
            float gv[4][K], v[4][K], y[K], b[K];
#pragma unroll
            for (int i = 0; i < 4; ++i) cols.load(gr + i * g_stream_stride, gv[i]);
            cols.load(yr, y);
#pragma unroll
            for (int j = 0; j < 4; ++j) cols.load(x + j * in.stream_stride, v[j]);
#pragma unroll
            for (int c = 0; c < K; ++c) {
                b[c] = k.h[0] * gv[0][c];
#pragma unroll
                for (int i = 1; i < 4; ++i) b[c] = fmaf(k.h[i], gv[i][c], b[c]);
            }
            if (d.limit) {
                const uint32_t keep = map.keep(s, d, key);
                drop(y, keep, d.scale);
                drop(b, keep, d.scale);
            }
            cols.store(dy + r * C, b);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int c = 0; c < K; ++c) acc[16 + i] = fmaf(gv[i][c], y[c], acc[16 + i]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int c = 0; c < K; ++c) {
                    b[c] = k.t[j] * gv[0][c];
#pragma unroll
                    for (int i = 1; i < 4; ++i) b[c] = fmaf(k.t[4 * i + j], gv[i][c], b[c]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[4 * i + j] = fmaf(gv[i][c], v[j][c], acc[4 * i + j]);
                }
                cols.store(dxr + static_cast<int64_t>(j) * C, b);
            }
        }
        sum = warp_sum20(acc);
    }
    if (warps > 1) {
        // one token in the block: its warps' sums in warp order
        if (lane < 20) part[threadIdx.x >> 5][lane] = sum;
        __syncthreads();
        if (threadIdx.x >= 32) return;
        sum = 0.0f;
        if (lane < 20)
            for (int w = 0; w < warps; ++w) sum += part[w][lane];
    }
    if (r >= N) return;
    if (lane < 16)
        store_any(dT, 16 * r + lane, in.T_dtype, sum);
    else if (lane < 20)
        store_any(dh, 4 * r + lane - 16, in.h_dtype, sum);
}

static bool aligned_streams(const void* p, int64_t stride, int64_t stream_stride, int elem)
{
    return aligned16(p, stride, elem) && ((stream_stride * elem) & 15) == 0;
}

template <class Elem>
static bool mix_in_pieces(const MixIn<Elem>& in, int64_t C)
{
    constexpr int e = sizeof(Elem);
    return ((C * e) & 15) == 0 && aligned_streams(in.x, in.stride, in.stream_stride, e) && aligned16(in.y, in.y_stride, e);
}

// Threads for a token of `pieces` pieces (a power of two from `least`): all
// of them at once if a block holds them.
static int mix_threads(int64_t pieces, int least)
{
    int t = least;
    while (t < kMixBlock && t < pieces) t *= 2;
    return t;
}

static unsigned mix_grid(int64_t N, int tokens) { return static_cast<unsigned>(ceil_div(N, tokens)); }

template <class Elem>
static int mix_forward(const MixIn<Elem>& in, void* out, const Dropout& d, int64_t N, int64_t C, cudaStream_t stream)
{
    Elem* o = static_cast<Elem*>(out);
    if (mix_in_pieces(in, C) && aligned16(out)) {
        int t = mix_threads(C / MixVecCols<Elem>::K, 8);
        if (N >= 148 * 16) t = std::min(t, MHC_MIXF_T);
        mix_fwd_kernel<Elem, MixVec<Elem>>
            <<<mix_grid(N, kMixBlock / t), dim3(t, kMixBlock / t), 0, stream>>>(in, o, d, N, static_cast<int>(C));
    } else {
        const int t = mix_threads(ceil_div(C, 8), 32);
        mix_fwd_kernel<Elem, MixLoose<Elem, 8>>
            <<<mix_grid(N, kMixBlock / t), dim3(t, kMixBlock / t), 0, stream>>>(in, o, d, N, static_cast<int>(C));
    }
    return static_cast<int>(cudaGetLastError());
}

template <class Elem>
static int mix_backward(const void* g, int64_t g_stride, int64_t g_stream_stride, const MixIn<Elem>& in, void* dx,
                        void* dT, void* dy, void* dh, const Dropout& d, int64_t N, int64_t C, cudaStream_t stream)
{
    const Elem* gp = static_cast<const Elem*>(g);
    Elem *dxp = static_cast<Elem*>(dx), *dyp = static_cast<Elem*>(dy);
    const bool pieces = mix_in_pieces(in, C) && aligned_streams(g, g_stride, g_stream_stride, sizeof(Elem)) &&
                        aligned16(dx) && aligned16(dy);
    // A warp per token once there are tokens for every warp the GPU holds,
    // else a block per token.
    const int64_t per_token = pieces ? C / MixVecCols<Elem>::K : ceil_div(C, 8);
    const int t = N >= 148 * 16 ? 32 : mix_threads(per_token, 32);
    const int tokens = t == 32 ? 4 : 1;
    if (pieces)
        mix_bwd_kernel<Elem, MixVec<Elem>><<<mix_grid(N, tokens), dim3(t, tokens), 0, stream>>>(
            gp, g_stride, g_stream_stride, in, dxp, dT, dyp, dh, d, N, static_cast<int>(C));
    else
        mix_bwd_kernel<Elem, MixLoose<Elem, 4>><<<mix_grid(N, tokens), dim3(t, tokens), 0, stream>>>(
            gp, g_stride, g_stream_stride, in, dxp, dT, dyp, dh, d, N, static_cast<int>(C));
    return static_cast<int>(cudaGetLastError());
}

static bool mix_args_ok(const void* X, int64_t token_stride, int64_t stream_stride, const void* y, int64_t y_stride,
                        int dtype, const void* T, int T_dtype, const void* h, int h_dtype, double p, int64_t N,
                        int64_t C)
{
    return N >= 0 && N < (int64_t{1} << 31) && C >= 1 && C <= kMaxWidth && token_stride >= 0 && stream_stride >= 0 && y_stride >= 0 && known_dtype(dtype) &&
           known_dtype(T_dtype) && known_dtype(h_dtype) && p >= 0.0 && p <= 1.0 && (N == 0 || (X && y && T && h));
}

}  // namespace mhcp

using namespace mhcp;

extern "C" int mhc_stream_mix_n4(const void* d_X, int64_t token_stride, int64_t stream_stride, const void* d_y,
                                 int64_t y_stride, int dtype, const void* d_T, int T_dtype, const void* d_h,
                                 int h_dtype, void* d_out, double p, int64_t seed, const int64_t* d_seed,
                                 int64_t offset, int64_t N, int64_t C, cudaStream_t stream)
{
    if (!mix_args_ok(d_X, token_stride, stream_stride, d_y, y_stride, dtype, d_T, T_dtype, d_h, h_dtype, p, N, C) ||
        (N > 0 && !d_out))
        return MHC_ERR_INVALID_VALUE;
    if (N == 0) return MHC_OK;
    const Dropout d = make_dropout(p, seed, d_seed, offset);
    auto run = [&](auto elem) {
        using Elem = decltype(elem);
        const MixIn<Elem> in{static_cast<const Elem*>(d_X), token_stride, stream_stride, static_cast<const Elem*>(d_y),
                             y_stride, d_T, d_h, T_dtype, h_dtype};
        return mix_forward(in, d_out, d, N, C, stream);
    };
    switch (dtype) {
        case MHC_DTYPE_BF16: return run(__nv_bfloat16{});
        case MHC_DTYPE_F16: return run(__half{});
        default: return run(float{});
    }
}

extern "C" int mhc_stream_mix_n4_backward(const void* d_G, int64_t g_token_stride, int64_t g_stream_stride,
                                          const void* d_X, int64_t token_stride, int64_t stream_stride,
                                          const void* d_y, int64_t y_stride, int dtype, const void* d_T, int T_dtype,
                                          const void* d_h, int h_dtype, void* d_dX, void* d_dT, void* d_dy, void* d_dh,
                                          double p, int64_t seed, const int64_t* d_seed, int64_t offset, int64_t N,
                                          int64_t C, cudaStream_t stream)
{
    if (!mix_args_ok(d_X, token_stride, stream_stride, d_y, y_stride, dtype, d_T, T_dtype, d_h, h_dtype, p, N, C) ||
        g_token_stride < 0 || g_stream_stride < 0 || (N > 0 && (!d_G || !d_dX || !d_dT || !d_dy || !d_dh)))
        return MHC_ERR_INVALID_VALUE;
    if (N == 0) return MHC_OK;
    const Dropout d = make_dropout(p, seed, d_seed, offset);
    auto run = [&](auto elem) {
        using Elem = decltype(elem);
        const MixIn<Elem> in{static_cast<const Elem*>(d_X), token_stride, stream_stride, static_cast<const Elem*>(d_y),
                             y_stride, d_T, d_h, T_dtype, h_dtype};
        return mix_backward(d_G, g_token_stride, g_stream_stride, in, d_dX, d_dT, d_dy, d_dh, d, N, C, stream);
    };
    switch (dtype) {
        case MHC_DTYPE_BF16: return run(__nv_bfloat16{});
        case MHC_DTYPE_F16: return run(__half{});
        default: return run(float{});
    }
}
