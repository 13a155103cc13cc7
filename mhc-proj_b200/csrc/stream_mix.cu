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

#include "mix_ring.cuh"
#include "mix_source.cuh"
#include "row_copy.cuh"

namespace mhcp {

constexpr int kMixBlock = 256;

// The kernels below read a token's columns directly, `threads` threads a
// token:
//   MixPieces   16-byte pieces, of rows of aligned, whole pieces
//   MixSingle   four columns a step, `threads` apart, of any rows
template <class Elem>
struct MixPieces {
    static constexpr int kPairs = 8 / sizeof(Elem);
    int64_t first;  // element index of the row's start in y
    int C, t, threads;

    __device__ __forceinline__ int steps() const { return (C / (2 * kPairs) + threads - 1) / threads; }
    __device__ __forceinline__ int col(int step) const { return (step * threads + t) * (2 * kPairs); }
    __device__ __forceinline__ void load(const Elem* __restrict__ row, int step, float2 (&v)[kPairs]) const
    {
        const int c = col(step);
        const uint4 q = c < C ? __ldg(reinterpret_cast<const uint4*>(row + c)) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int p = 0; p < kPairs; ++p) v[p] = pair_of<Elem>(q, p);
    }
    __device__ __forceinline__ void store(Elem* __restrict__ row, int step, const float2 (&v)[kPairs]) const
    {
        const uint4 q = piece_of<Elem>(v);
        if (col(step) < C) *reinterpret_cast<uint4*>(row + col(step)) = q;
    }
    // Bits 2 p and 2 p + 1: the columns of pair p are kept.
    __device__ __forceinline__ uint32_t keep(int step, const Dropout& d, uint2 key) const
    {
        const int64_t e = first + col(step);
        return keep_bits(e >> 3, d.offset, key, d.limit) >> (e & 7);
    }
};

template <class Elem>
struct MixSingle {
    static constexpr int kPairs = 2;
    int64_t first;
    int C, t, threads;

    __device__ __forceinline__ int steps() const { return (C + 2 * kPairs * threads - 1) / (2 * kPairs * threads); }
    __device__ __forceinline__ int col(int step, int j) const { return (step * 2 * kPairs + j) * threads + t; }
    __device__ __forceinline__ void load(const Elem* __restrict__ row, int step, float2 (&v)[kPairs]) const
    {
#pragma unroll
        for (int p = 0; p < kPairs; ++p) {
            v[p].x = col(step, 2 * p) < C ? to_f32(row[col(step, 2 * p)]) : 0.0f;
            v[p].y = col(step, 2 * p + 1) < C ? to_f32(row[col(step, 2 * p + 1)]) : 0.0f;
        }
    }
    __device__ __forceinline__ void store(Elem* __restrict__ row, int step, const float2 (&v)[kPairs]) const
    {
#pragma unroll
        for (int p = 0; p < kPairs; ++p) {
            if (col(step, 2 * p) < C) row[col(step, 2 * p)] = from_f32<Elem>(v[p].x);
            if (col(step, 2 * p + 1) < C) row[col(step, 2 * p + 1)] = from_f32<Elem>(v[p].y);
        }
    }
    // The lanes that share a token in a warp (8, 16 or 32 of them) have four runs of as
    // many columns; one call of the generator in each gives all the draws of
    // the (at most lanes / 8 + 1) groups of eight that each run touches.
    __device__ __forceinline__ uint32_t keep(int step, const Dropout& d, uint2 key) const
    {
        const int lanes = min(threads, 32), lane = t & (lanes - 1), groups = lanes / 8 + 1;
        const unsigned mask = lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1) << (threadIdx.x + threadIdx.y * threads & 31 & ~(lanes - 1));
        const int mine = min(lane / groups, 3);
        const int64_t run = first + col(step, mine) - lane;
        const uint32_t bits = keep_bits((run >> 3) + lane - mine * groups, d.offset, key, d.limit);
        uint32_t k = 0;
#pragma unroll
        for (int j = 0; j < 2 * kPairs; ++j) {
            const int64_t e = first + col(step, j);
            const int from = j * groups + static_cast<int>((e >> 3) - ((e - lane) >> 3));
            k |= (__shfl_sync(mask, bits, from, lanes) >> (e & 7) & 1u) << j;
        }
        return k;
    }
};

template <int kPairs>
__device__ __forceinline__ void drop(float2 (&y)[kPairs], uint32_t keep, float scale)
{
#pragma unroll
    for (int p = 0; p < kPairs; ++p) {
        y[p] = mul2(y[p], both(scale));
        if (!(keep >> (2 * p) & 1u)) y[p].x = 0.0f;
        if (!(keep >> (2 * p + 1) & 1u)) y[p].y = 0.0f;
    }
}

// Block: (threads of a token, tokens).
template <class Elem, class Map, bool kWide>
__global__ void __launch_bounds__(kMixBlock)
mix_fwd_direct(MixIn<Elem> in, Elem* __restrict__ out, Dropout d, int64_t N, int C)
{
    constexpr int kPairs = Map::kPairs;
    const int64_t r = blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y;
    if (r >= N) return;
    const uint2 key = dropout_key(d);
    const Elem* x = in.x + r * in.stride;
    const Map map{r * C, C, static_cast<int>(threadIdx.x), static_cast<int>(blockDim.x)};
    const MixCoef k = mix_coef<kWide>(in, r);
    const int steps = map.steps();
    for (int s = 0; s < steps; ++s) {
        float2 v[4][kPairs], y[kPairs];
#pragma unroll
        for (int j = 0; j < 4; ++j) map.load(x + j * in.stream_stride, s, v[j]);
        map.load(in.y + r * in.y_stride, s, y);
        if (d.limit) drop(y, map.keep(s, d, key), d.scale);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 a[kPairs];
#pragma unroll
            for (int p = 0; p < kPairs; ++p) {
                a[p] = mul2(both(k.h[i]), y[p]);
#pragma unroll
                for (int j = 0; j < 4; ++j) a[p] = fma2(both(k.t[4 * i + j]), v[j][p], a[p]);
            }
            map.store(out + (4 * r + i) * C, s, a);
        }
    }
}

template <class Elem, class Map, bool kWide>
__global__ void __launch_bounds__(kMixBlock)
mix_bwd_direct(const Elem* __restrict__ g, int64_t g_stride, int64_t g_stream_stride, MixIn<Elem> in,
               Elem* __restrict__ dx, void* __restrict__ dT, Elem* __restrict__ dy, void* __restrict__ dh, Dropout d,
               int64_t N, int C)
{
    constexpr int kPairs = Map::kPairs;
    __shared__ float part[kMixBlock / 32][20];
    const int64_t r = blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y;
    const bool live = r < N;
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    float2 acc[20];
    float sums[20];
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < 20; ++i) acc[i] = both(0.0f);
    if (live) {
        const uint2 key = dropout_key(d);
        const Elem *x = in.x + r * in.stride, *gr = g + r * g_stride;
        const Map map{r * C, C, static_cast<int>(threadIdx.x), static_cast<int>(blockDim.x)};
        const MixCoef k = mix_coef<kWide>(in, r);
        const int steps = map.steps();
        for (int s = 0; s < steps; ++s) {
            float2 gv[4][kPairs], v[4][kPairs], y[kPairs], b[kPairs];
#pragma unroll
            for (int i = 0; i < 4; ++i) map.load(gr + i * g_stream_stride, s, gv[i]);
            map.load(in.y + r * in.y_stride, s, y);
#pragma unroll
            for (int j = 0; j < 4; ++j) map.load(x + j * in.stream_stride, s, v[j]);
#pragma unroll
            for (int p = 0; p < kPairs; ++p) {
                b[p] = mul2(both(k.h[0]), gv[0][p]);
#pragma unroll
                for (int i = 1; i < 4; ++i) b[p] = fma2(both(k.h[i]), gv[i][p], b[p]);
            }
            if (d.limit) {
                const uint32_t keep = map.keep(s, d, key);
                drop(y, keep, d.scale);
                drop(b, keep, d.scale);
            }
            map.store(dy + r * C, s, b);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int p = 0; p < kPairs; ++p) acc[16 + i] = fma2(gv[i][p], y[p], acc[16 + i]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int p = 0; p < kPairs; ++p) {
                    b[p] = mul2(both(k.t[j]), gv[0][p]);
#pragma unroll
                    for (int i = 1; i < 4; ++i) b[p] = fma2(both(k.t[4 * i + j]), gv[i][p], b[p]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[4 * i + j] = fma2(gv[i][p], v[j][p], acc[4 * i + j]);
                }
                map.store(dx + (4 * r + j) * C, s, b);
            }
            constexpr int run = kMixRun / kPairs;  // steps: only a token of a whole block has more
            if (s % run != run - 1 || s + 1 == steps) continue;
#pragma unroll
            for (int i = 0; i < 20; ++i) {
                sums[i] = acc[i].x + acc[i].y;
                acc[i] = both(0.0f);
            }
            total += warp_sum20(sums);
        }
    }
#pragma unroll
    for (int i = 0; i < 20; ++i) sums[i] = acc[i].x + acc[i].y;
    if (warps <= 1) {
        put_token_sums(in, r, live, lane, blockDim.x, sums, dT, dh);
        return;
    }
    // one token in the block: its warps' sums in warp order
    total += warp_sum20(sums);
    if (lane < 20) part[threadIdx.x >> 5][lane] = static_cast<float>(total);
    __syncthreads();
    if (threadIdx.x >= 20) return;
    float all = 0.0f;
    for (int w = 0; w < warps; ++w) all += part[w][lane];
    put_token_sum(in, r, lane, all, dT, dh);
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

// A power of two from `least` to `most` that is at least `want`, if there is one.
static int mix_threads(int64_t want, int least, int most)
{
    int t = least;
    while (t < most && t < want) t *= 2;
    return t;
}

// Rows of single elements narrower than this take the direct kernels, where a
// token takes 8 to 32 lanes; the ring kernels give it a warp.  65536 tokens, bf16,
// forward / backward us: 25 wide 21 / 49 direct, 28 / 105 in the ring; 99 wide
// 76 / 251 direct, 55 / 111 in the ring.
constexpr int64_t kMixNarrow = 48;

template <class Elem, bool kVec, bool kWide>
static int mix_forward_ring(const MixIn<Elem>& in, Elem* out, const Dropout& d, int64_t N, int64_t C, cudaStream_t stream)
{
    using Chunk = MixChunk<Elem, kVec>;
    const int lanes = kVec ? mix_threads(C / Chunk::K, 1, 32) : 32;
    constexpr int warps = kMixRingBlock / 32, smem = warps * kMixFwdStages * 5 * Chunk::kPlace;
    const cudaError_t e = allow_smem<sizeof(MixMasks)>(mix_fwd_ring<Elem, kVec, kWide>, smem);
    if (e != cudaSuccess) return static_cast<int>(e);
    const int64_t items = ceil_div(N, 32 / lanes) * Chunk::count(static_cast<int>(C), lanes);
    const int64_t grid = std::min<int64_t>(ceil_div(items, warps), kMixFwdBlocks * sm_count());
    mix_fwd_ring<Elem, kVec, kWide><<<static_cast<unsigned>(grid), kMixRingBlock, smem, stream>>>(
        in, span_of(in.x, N, in.stride, 4, in.stream_stride, C), span_of(in.y, N, in.y_stride, 1, 0, C), out, d, N,
        static_cast<int>(C), lanes);
    return static_cast<int>(cudaGetLastError());
}

template <class Elem, bool kWide>
static int mix_forward(const MixIn<Elem>& in, void* out, const Dropout& d, int64_t N, int64_t C, cudaStream_t stream)
{
    Elem* o = static_cast<Elem*>(out);
    if (mix_in_pieces(in, C) && aligned16(out)) return mix_forward_ring<Elem, true, kWide>(in, o, d, N, C, stream);
    if (C >= kMixNarrow) return mix_forward_ring<Elem, false, kWide>(in, o, d, N, C, stream);
    const int t = mix_threads(ceil_div(C, 4), 8, 32), tokens = kMixBlock / t;
    mix_fwd_direct<Elem, MixSingle<Elem>, kWide><<<static_cast<unsigned>(ceil_div(N, tokens)), dim3(t, tokens), 0, stream>>>(
        in, o, d, N, static_cast<int>(C));
    return static_cast<int>(cudaGetLastError());
}

template <class Elem, bool kVec, bool kWide, bool kLong>
static int mix_backward_ring(const Elem* g, int64_t g_stride, int64_t g_stream_stride, const MixIn<Elem>& in, Elem* dx,
                             void* dT, Elem* dy, void* dh, const Dropout& d, int64_t N, int64_t C, cudaStream_t stream)
{
    using Chunk = MixChunk<Elem, kVec>;
    constexpr int warps = kMixRingBlock / 32, smem = warps * kMixBwdStages * 9 * Chunk::kPlace;
    const cudaError_t e = allow_smem<sizeof(MixMasks)>(mix_bwd_ring<Elem, kVec, kWide, kLong>, smem);
    if (e != cudaSuccess) return static_cast<int>(e);
    const int lanes = kVec ? mix_threads(C / Chunk::K, 1, 32) : 32;
    // Two blocks an SM (65536 tokens of 2048, bf16: 595 us, with three 675), or
    // three where a token is over before the next one's coefficients have come,
    // or single elements take more instructions.
    const int blocks = kVec && Chunk::count(static_cast<int>(C), lanes) > 2 ? 2 : 3;
    const int64_t grid = std::min<int64_t>(ceil_div(ceil_div(N, 32 / lanes), warps), blocks * sm_count());
    mix_bwd_ring<Elem, kVec, kWide, kLong><<<static_cast<unsigned>(grid), kMixRingBlock, smem, stream>>>(
        g, g_stride, g_stream_stride, span_of(g, N, g_stride, 4, g_stream_stride, C), in,
        span_of(in.x, N, in.stride, 4, in.stream_stride, C), span_of(in.y, N, in.y_stride, 1, 0, C), dx, dT, dy, dh, d, N,
        static_cast<int>(C), lanes);
    return static_cast<int>(cudaGetLastError());
}

template <class Elem, bool kWide>
static int mix_backward(const void* g, int64_t g_stride, int64_t g_stream_stride, const MixIn<Elem>& in, void* dx,
                        void* dT, void* dy, void* dh, const Dropout& d, int64_t N, int64_t C, cudaStream_t stream)
{
    const Elem* gp = static_cast<const Elem*>(g);
    Elem *dxp = static_cast<Elem*>(dx), *dyp = static_cast<Elem*>(dy);
    const bool pieces = mix_in_pieces(in, C) && aligned_streams(g, g_stride, g_stream_stride, sizeof(Elem)) &&
                        aligned16(dx) && aligned16(dy);
    const bool narrow = !pieces && C < kMixNarrow;
    // A warp per token once there are four tokens for every SM, else a block
    // (bf16, 4096 wide: 300 tokens 14.0 us a warp each, 11.3 a block each; 1000
    // tokens 23.6 and 30.4).
    if (N >= 4 * sm_count() && !narrow) {
        auto ring = [&](auto vec, auto is_long) {
            return mix_backward_ring<Elem, decltype(vec)::value, kWide, decltype(is_long)::value>(
                gp, g_stride, g_stream_stride, in, dxp, dT, dyp, dh, d, N, C, stream);
        };
        using std::false_type, std::true_type;
        // a run is 256 pairs of columns a lane
        if (C > 2 * 32 * kMixRun) return pieces ? ring(true_type{}, true_type{}) : ring(false_type{}, true_type{});
        return pieces ? ring(true_type{}, false_type{}) : ring(false_type{}, false_type{});
    }
    const int t = narrow ? mix_threads(ceil_div(C, 4), 8, 32)
                         : mix_threads(pieces ? C * static_cast<int64_t>(sizeof(Elem)) / 16 : ceil_div(C, 4), 32, kMixBlock);
    const int tokens = t <= 32 ? 128 / t : 1;
    const dim3 grid(static_cast<unsigned>(ceil_div(N, tokens))), block(t, tokens);
    if (pieces)
        mix_bwd_direct<Elem, MixPieces<Elem>, kWide><<<grid, block, 0, stream>>>(
            gp, g_stride, g_stream_stride, in, dxp, dT, dyp, dh, d, N, static_cast<int>(C));
    else
        mix_bwd_direct<Elem, MixSingle<Elem>, kWide><<<grid, block, 0, stream>>>(
            gp, g_stride, g_stream_stride, in, dxp, dT, dyp, dh, d, N, static_cast<int>(C));
    return static_cast<int>(cudaGetLastError());
}

static bool mix_args_ok(const void* X, int64_t token_stride, int64_t stream_stride, const void* y, int64_t y_stride,
                        int dtype, const void* T, int T_dtype, const void* h, int h_dtype, double p, int64_t N,
                        int64_t C, const int64_t* d_seed)
{
    return rows_ok(N, C) && token_stride >= 0 && stream_stride >= 0 && y_stride >= 0 && known_dtype(dtype) &&
           known_dtype(T_dtype) && known_dtype(h_dtype) && p >= 0.0 && p <= 1.0 &&
           (N == 0 || (X && y && T && h)) && at_elements(dtype, X, y) && at_elements(T_dtype, T) &&
           at_elements(h_dtype, h) && at_element(d_seed, 8);
}

// The coefficients in the form that is read 16 bytes at a time.
static bool wide_coefficients(const void* T, int T_dtype, const void* h, int h_dtype)
{
    return T_dtype == MHC_DTYPE_F32 && h_dtype == MHC_DTYPE_F32 && aligned16(T) && aligned16(h);
}

}  // namespace mhcp

using namespace mhcp;

extern "C" int mhc_stream_mix_n4(const void* d_X, int64_t token_stride, int64_t stream_stride, const void* d_y,
                                 int64_t y_stride, int dtype, const void* d_T, int T_dtype, const void* d_h,
                                 int h_dtype, void* d_out, double p, int64_t seed, const int64_t* d_seed,
                                 int64_t offset, int64_t N, int64_t C, cudaStream_t stream)
{
    if (!mix_args_ok(d_X, token_stride, stream_stride, d_y, y_stride, dtype, d_T, T_dtype, d_h, h_dtype, p, N, C, d_seed) ||
        (N > 0 && !d_out) || !at_elements(dtype, d_out))
        return MHC_ERR_INVALID_VALUE;
    if (N == 0) return MHC_OK;
    const Dropout d = make_dropout(p, seed, d_seed, offset);
    const bool wide = wide_coefficients(d_T, T_dtype, d_h, h_dtype);
    auto run = [&](auto elem) {
        using Elem = decltype(elem);
        const MixIn<Elem> in{static_cast<const Elem*>(d_X), token_stride, stream_stride, static_cast<const Elem*>(d_y),
                             y_stride, d_T, d_h, T_dtype, h_dtype};
        return wide ? mix_forward<Elem, true>(in, d_out, d, N, C, stream)
                    : mix_forward<Elem, false>(in, d_out, d, N, C, stream);
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
    if (!mix_args_ok(d_X, token_stride, stream_stride, d_y, y_stride, dtype, d_T, T_dtype, d_h, h_dtype, p, N, C, d_seed) ||
        g_token_stride < 0 || g_stream_stride < 0 || (N > 0 && (!d_G || !d_dX || !d_dT || !d_dy || !d_dh)) ||
        !at_elements(dtype, d_G, d_dX, d_dy) || !at_elements(T_dtype, d_dT) || !at_elements(h_dtype, d_dh))
        return MHC_ERR_INVALID_VALUE;
    if (N == 0) return MHC_OK;
    const Dropout d = make_dropout(p, seed, d_seed, offset);
    const bool wide = wide_coefficients(d_T, T_dtype, d_h, h_dtype);
    auto run = [&](auto elem) {
        using Elem = decltype(elem);
        const MixIn<Elem> in{static_cast<const Elem*>(d_X), token_stride, stream_stride, static_cast<const Elem*>(d_y),
                             y_stride, d_T, d_h, T_dtype, h_dtype};
        return wide ? mix_backward<Elem, true>(d_G, g_token_stride, g_stream_stride, in, d_dX, d_dT, d_dy, d_dh, d, N, C, stream)
                    : mix_backward<Elem, false>(d_G, g_token_stride, g_stream_stride, in, d_dX, d_dT, d_dy, d_dh, d, N, C, stream);
    };
    switch (dtype) {
        case MHC_DTYPE_BF16: return run(__nv_bfloat16{});
        case MHC_DTYPE_F16: return run(__half{});
        default: return run(float{});
    }
}
