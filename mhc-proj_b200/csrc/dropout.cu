// Dropout whose mask is formed where it is needed: y = x * scale where the
// element's draw keeps it, 0 where not (philox.cuh), on contiguous elements.
// The gradient is the same function of the incoming gradient, so one kernel
// serves both directions and nothing is kept between them.
#include <algorithm>

#include "philox.cuh"
#include "row_ops.cuh"

namespace mhcp {

constexpr int kDropBlock = 256;

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
    // The eight draws are the halves of w, low one first; an element is kept
    // when its draw, in the upper half of a word, is above `under`.
    __device__ __forceinline__ void drop(const uint4& draws, uint32_t under, float scale)
    {
        const uint32_t w[4] = {draws.x, draws.y, draws.z, draws.w};
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            float2 v[16 / sizeof(Elem) / 2];
#pragma unroll
            for (int j = 0; j < 16 / static_cast<int>(sizeof(Elem)) / 2; ++j) {
                const uint32_t d = w[i * (16 / sizeof(Elem) / 2) + j];
                v[j] = mul2(pair_of<Elem>(q[i], j), both(scale));
                if (d << 16 <= under) v[j].x = 0.0f;
                if (d <= under) v[j].y = 0.0f;
            }
            q[i] = piece_of<Elem>(v);
        }
    }
};

// kGroups: groups a thread takes.  65536 x 4096 bf16: 177 us, 6.1 TB/s (loads and
// stores of single elements 667); 195 us under a load of seconds, when the clock
// falls: the generator's multiplies and the selects fill the issue slots.
template <class Elem, bool kVec, int kGroups>
__global__ void __launch_bounds__(kDropBlock)
dropout_kernel(const Elem* x, Elem* y, int64_t count, Dropout d)
{
    const uint2 key = dropout_key(d);
    const int64_t q0 = blockIdx.x * static_cast<int64_t>(kDropBlock * kGroups) + threadIdx.x;
    const int64_t whole = count / 8;
    if (kVec && q0 + (kGroups - 1) * kDropBlock < whole) {
        DropGroup<Elem> g[kGroups];
#pragma unroll
        for (int k = 0; k < kGroups; ++k) g[k].load(x + 8 * (q0 + k * kDropBlock));
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            const int64_t q = q0 + k * kDropBlock;
            if (d.limit) g[k].drop(draws_of(q, d.offset, key), (d.limit << 16) - 1, d.scale);
            g[k].store(y + 8 * q);
        }
        return;
    }
    for (int k = 0; k < kGroups; ++k) {
        const int64_t q = q0 + k * kDropBlock, e = 8 * q;
        if (e >= count) return;
        const uint32_t keep = d.limit ? keep_bits(q, d.offset, key, d.limit) : 0xffu;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (e + i < count) y[e + i] = from_f32<Elem>((keep >> i & 1u) ? to_f32(x[e + i]) * d.scale : 0.0f);
    }
}

template <class Elem, bool kVec, int kGroups>
static int dropout_launch(const Elem* x, Elem* y, int64_t count, const Dropout& d, cudaStream_t stream)
{
    constexpr int64_t kPerBlock = 8 * kDropBlock * kGroups;
    const int64_t blocks = count / kPerBlock + (count % kPerBlock != 0);
    if (blocks > 0x7fffffff) return MHC_ERR_INVALID_VALUE;
    dropout_kernel<Elem, kVec, kGroups><<<static_cast<unsigned>(blocks), kDropBlock, 0, stream>>>(x, y, count, d);
    return static_cast<int>(cudaGetLastError());
}

// Four groups a thread where the batch fills the GPU several times over (bf16,
// 65536 x 4096: 177 us against 202 with one), one where it does not (fp32, 4099 x
// 1111: 6.3 us against 7.7) and for fp32, whose groups are two pieces.
template <class Elem>
static int dropout_typed(const void* x, void* y, int64_t count, const Dropout& d, cudaStream_t stream)
{
    const Elem* xe = static_cast<const Elem*>(x);
    Elem* ye = static_cast<Elem*>(y);
    if (!aligned16(x) || !aligned16(y)) return dropout_launch<Elem, false, 1>(xe, ye, count, d, stream);
    if (sizeof(Elem) == 4 || count < (int64_t{1} << 23)) return dropout_launch<Elem, true, 1>(xe, ye, count, d, stream);
    return dropout_launch<Elem, true, 4>(xe, ye, count, d, stream);
}

}  // namespace mhcp

using namespace mhcp;

extern "C" int mhc_dropout(const void* d_x, void* d_y, int dtype, int64_t count, double p, int64_t seed,
                           const int64_t* d_seed, int64_t offset, cudaStream_t stream)
{
    if (count < 0 || !(p >= 0.0 && p <= 1.0) || !known_dtype(dtype) || (count > 0 && (!d_x || !d_y)) ||
        !at_elements(dtype, d_x, d_y) || !at_element(d_seed, 8))
        return MHC_ERR_INVALID_VALUE;
    if (count == 0) return MHC_OK;
    const Dropout d = make_dropout(p, seed, d_seed, offset);
    switch (dtype) {
        case MHC_DTYPE_BF16: return dropout_typed<__nv_bfloat16>(d_x, d_y, count, d, stream);
        case MHC_DTYPE_F16: return dropout_typed<__half>(d_x, d_y, count, d, stream);
        default: return dropout_typed<float>(d_x, d_y, count, d, stream);
    }
}
