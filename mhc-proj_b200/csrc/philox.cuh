// Dropout's draws: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel Random
// Numbers: As Easy as 1, 2, 3", SC 2011), a bijection of a 128-bit counter
// under a 64-bit key.  Element e of a tensor (its row-major index) takes 16
// of the 128 bits that the counter (e / 8, offset) gives under the key seed:
// bits 16 (e % 8) and up.  So a mask is a function of (seed, offset, e) alone
// -- nothing of it is stored, and the backward pass, a captured graph's replay
// or a kernel with another thread layout forms the same one again.
//
// 16 bits a draw: an eighth of a Philox call per element, 20 wide multiplies
// over eight elements, so that at two bytes in and two out the integer pipe
// needs less time than the memory does.  An element is dropped when its draw is
// below limit = floor(65536 p + 1/2), and kept elements are scaled by
// 65536 / (65536 - limit), the inverse of the share of draws that keeps one:
// the expectation is exact although p is rounded to a multiple of 2^-16.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace mhcp {

// What a launch knows of its mask.  d_seed, if given, is the device memory
// that holds the seed (read by the kernel, so a captured graph can be
// replayed with another one); limit 0 drops nothing and draws nothing.
struct Dropout {
    int64_t seed, offset;
    const int64_t* d_seed;
    uint32_t limit;
    float scale;
};

// p in [0, 1], checked by the caller.
inline Dropout make_dropout(double p, int64_t seed, const int64_t* d_seed, int64_t offset)
{
    const uint32_t limit = static_cast<uint32_t>(p * 65536.0 + 0.5);
    const float scale = limit < 65536u ? static_cast<float>(65536.0 / (65536.0 - limit)) : 0.0f;
    return {seed, offset, d_seed, limit, scale};
}

__device__ __forceinline__ uint2 dropout_key(const Dropout& d)
{
    const uint64_t s = static_cast<uint64_t>(d.d_seed ? __ldg(reinterpret_cast<const long long*>(d.d_seed)) : d.seed);
    return make_uint2(static_cast<uint32_t>(s), static_cast<uint32_t>(s >> 32));
}

__device__ __forceinline__ uint4 philox4x32_10(uint4 c, uint2 k)
{
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = static_cast<uint64_t>(0xD2511F53u) * c.x;
        const uint64_t p1 = static_cast<uint64_t>(0xCD9E8D57u) * c.z;
        c = make_uint4(static_cast<uint32_t>(p1 >> 32) ^ c.y ^ k.x, static_cast<uint32_t>(p1),
                       static_cast<uint32_t>(p0 >> 32) ^ c.w ^ k.y, static_cast<uint32_t>(p0));
        k.x += 0x9E3779B9u;
        k.y += 0xBB67AE85u;
    }
    return c;
}

// The 128 bits that hold the draws of elements 8 * group ...
__device__ __forceinline__ uint4 draws_of(uint64_t group, uint64_t offset, uint2 key)
{
    return philox4x32_10(make_uint4(static_cast<uint32_t>(group), static_cast<uint32_t>(group >> 32),
                                    static_cast<uint32_t>(offset), static_cast<uint32_t>(offset >> 32)),
                         key);
}

// Bit i: element 8 * group + i is kept.  limit is not 0.
__device__ __forceinline__ uint32_t keep_bits(uint64_t group, uint64_t offset, uint2 key, uint32_t limit)
{
    const uint4 v = draws_of(group, offset, key);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    const uint32_t under = (limit << 16) - 1;  // a draw in a word's upper half is kept above it
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bits |= w[i] << 16 > under ? 1u << (2 * i) : 0u;
        bits |= w[i] > under ? 2u << (2 * i) : 0u;
    }
    return bits;
}

}  // namespace mhcp
