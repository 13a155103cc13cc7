// Dropout whose mask is formed where it is needed: y = x * scale where the
// element's draw keeps it, 0 where not (philox.cuh), on contiguous elements.
// The gradient is the same function of the incoming gradient, so one kernel
// serves both directions and nothing is kept between them.
#include <algorithm>

#include "philox.cuh"
#include "row_ops.cuh"

namespace mhcp {

constexpr int kDropBlock = 256;
constexpr int kDropGroups = 4;  // groups a thread takes

// A group of eight elements, one counter's draws, from and to 16-byte aligned memory.
template <class Elem>
struct DropGroup {
    static constexpr int kPieces = 8 * sizeof(Elem) / 16;
    uint4 q[kPieces];

    __device__ __forceinline__ void load(const Elem* p)
    {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) q[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void store(Elem* p) const
    {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) reinterpret_cast<uint4*>(p)[i] = q[i];
    }
    __device__ __forceinline__ void drop(uint32_t keep, float scale)
    {
        Elem* e = reinterpret_cast<Elem*>(q);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_f32<Elem>((keep >> i & 1u) ? to_f32(e[i]) * scale : 0.0f);
    }
};

template <class Elem, bool kVec>
__global__ void __launch_bounds__(kDropBlock)
dropout_kernel(const Elem* x, Elem* y, int64_t count, Dropout d)
{
    const uint2 key = dropout_key(d);
    const int64_t q0 = blockIdx.x * static_cast<int64_t>(kDropBlock * kDropGroups) + threadIdx.x;
    const int64_t whole = count / 8;
    if (kVec && q0 + (kDropGroups - 1) * kDropBlock < whole) {
        DropGroup<Elem> g[kDropGroups];
#pragma unroll
        for (int k = 0; k < kDropGroups; ++k) g[k].load(x + 8 * (q0 + k * kDropBlock));
#pragma unroll
        for (int k = 0; k < kDropGroups; ++k) {
            const int64_t q = q0 + k * kDropBlock;
            g[k].drop(d.limit ? keep_bits(q, d.offset, key, d.limit) : 0xffu, d.scale);
            g[k].store(y + 8 * q);
        }
        return;
    }
    for (int k = 0; k < kDropGroups; ++k) {
        const int64_t q = q0 + k * kDropBlock, e = 8 * q;
        if (e >= count) return;
        const uint32_t keep = d.limit ? keep_bits(q, d.offset, key, d.limit) : 0xffu;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (e + i < count) y[e + i] = from_f32<Elem>((keep >> i & 1u) ? to_f32(x[e + i]) * d.scale : 0.0f);
    }
}

template <class Elem>
static int dropout_launch(const void* x, void* y, int64_t count, const Dropout& d, cudaStream_t stream)
{
    const int64_t blocks = ceil_div(count, 8 * kDropBlock * kDropGroups);
    if (blocks > 0x7fffffff) return MHC_ERR_INVALID_VALUE;
    const Elem* xe = static_cast<const Elem*>(x);
    Elem* ye = static_cast<Elem*>(y);
    if (aligned16(x) && aligned16(y))
        dropout_kernel<Elem, true><<<static_cast<unsigned>(blocks), kDropBlock, 0, stream>>>(xe, ye, count, d);
    else
        dropout_kernel<Elem, false><<<static_cast<unsigned>(blocks), kDropBlock, 0, stream>>>(xe, ye, count, d);
    return static_cast<int>(cudaGetLastError());
}

}  // namespace mhcp

using namespace mhcp;

extern "C" int mhc_dropout(const void* d_x, void* d_y, int dtype, int64_t count, double p, int64_t seed,
                           const int64_t* d_seed, int64_t offset, cudaStream_t stream)
{
    if (count < 0 || !(p >= 0.0 && p <= 1.0) || !known_dtype(dtype) || (count > 0 && (!d_x || !d_y)))
        return MHC_ERR_INVALID_VALUE;
    if (count == 0) return MHC_OK;
    const Dropout d = make_dropout(p, seed, d_seed, offset);
    switch (dtype) {
        case MHC_DTYPE_BF16: return dropout_launch<__nv_bfloat16>(d_x, d_y, count, d, stream);
        case MHC_DTYPE_F16: return dropout_launch<__half>(d_x, d_y, count, d, stream);
        default: return dropout_launch<float>(d_x, d_y, count, d, stream);
    }
}
