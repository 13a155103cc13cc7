// Dropout whose mask is formed where it is needed: y = x * scale where the
// element's draw keeps it, 0 where not (philox.cuh), on contiguous elements.
// The gradient is the same function of the incoming gradient, so one kernel
// serves both directions and nothing is kept between them.
#include <algorithm>

#include "philox.cuh"
#include "row_ops.cuh"

namespace mhcp {

constexpr int kDropBlock = 256;

// One thread takes a group of eight elements, one counter's draws.
template <class Elem, bool kVec>
__global__ void __launch_bounds__(kDropBlock)
dropout_kernel(const Elem* x, Elem* y, int64_t count, Dropout d)
{
    const uint2 key = dropout_key(d);
    const int64_t groups = ceil_div(count, 8);
    for (int64_t q = blockIdx.x * static_cast<int64_t>(kDropBlock) + threadIdx.x; q < groups;
         q += gridDim.x * static_cast<int64_t>(kDropBlock)) {
        const uint32_t keep = d.limit ? keep_bits(q, d.offset, key, d.limit) : 0xffu;
        const int64_t e = 8 * q;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (e + i < count) y[e + i] = from_f32<Elem>((keep >> i & 1u) ? to_f32(x[e + i]) * d.scale : 0.0f);
    }
}

template <class Elem>
static int dropout_launch(const void* x, void* y, int64_t count, const Dropout& d, cudaStream_t stream)
{
    const int64_t blocks = std::min(ceil_div(ceil_div(count, 8), kDropBlock), int64_t{1} << 30);
    dropout_kernel<Elem, false><<<static_cast<unsigned>(blocks), kDropBlock, 0, stream>>>(
        static_cast<const Elem*>(x), static_cast<Elem*>(y), count, d);
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
