// Asynchronous copies of 16-byte pieces into shared memory: bytes on their way
// that hold no registers.
#pragma once

#include "ring_plan.h"
#include "row_ops.cuh"

namespace mhcp {

__device__ __forceinline__ void copy_piece_async(void* smem, const void* global)
{
    const unsigned s = static_cast<unsigned>(__cvta_generic_to_shared(smem));
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(global) : "memory");
}

__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// Waits until at most `stages` - 1 of this thread's batches of copies are under way.
__device__ __forceinline__ void copies_wait(int stages)
{
    if (stages >= 4)
        asm volatile("cp.async.wait_group 3;" ::: "memory");
    else if (stages == 3)
        asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (stages == 2)
        asm volatile("cp.async.wait_group 1;" ::: "memory");
    else
        asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// A tensor of rows: its bytes from the first to the last element, and whether
// its rows follow one another at 32 bytes or more, so that around every row
// but the first and the last token's there are 32 bytes of the tensor.
struct RowSpan {
    const char *lo, *hi;
    bool apart;

    __device__ __forceinline__ bool amid(int64_t r, int64_t N) const { return apart && r > 0 && r < N - 1; }
};

template <class Elem>
inline RowSpan span_of(const Elem* p, int64_t N, int64_t stride, int streams, int64_t stream_stride, int64_t C)
{
    return {reinterpret_cast<const char*>(p),
            reinterpret_cast<const char*>(p + (N - 1) * stride + (streams - 1) * stream_stride + C),
            stride * static_cast<int64_t>(sizeof(Elem)) >= 32};
}

// Where `from` comes to lie in shared memory, from the piece that holds it.
template <class Elem>
__device__ __forceinline__ int offset_in_piece(const Elem* from)
{
    return static_cast<int>(reinterpret_cast<uintptr_t>(from) & 15);
}

// The aligned piece at src to shared memory, as far as it has something of the
// row [begin, end): element by element where it reaches beyond the tensor.
template <class Elem>
__device__ __forceinline__ void copy_checked_piece(char* to, const char* src, const Elem* begin, const Elem* end,
                                                   const RowSpan& span)
{
    if (src + 16 <= reinterpret_cast<const char*>(begin) || src >= reinterpret_cast<const char*>(end)) return;
    if (src >= span.lo && src + 16 <= span.hi) {
        copy_piece_async(to, src);
        return;
    }
#pragma unroll
    for (int i = 0; i < 16 / static_cast<int>(sizeof(Elem)); ++i) {
        const Elem* e = reinterpret_cast<const Elem*>(src) + i;
        if (e >= begin && e < end) reinterpret_cast<Elem*>(to)[i] = *e;
    }
}

inline int sm_count()
{
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return 1;
    return sms;
}

// A launch may need more shared memory than a kernel has by default, which is
// for its static memory too (a four-stream norm backward's 20 KB).  The limit belongs to
// the kernel in the context and not to the launch, so every launch that has to
// ask sets the same one: two host threads with rows of two widths do not undo
// each other's.
template <int kStaticBytes, class Kernel>
inline cudaError_t allow_smem(Kernel kernel, int bytes)
{
    static_assert(kStaticBytes + kMostSmem <= kLargestSmem, "the static memory has to fit beside the rings");
    return asks_for_smem(kStaticBytes, bytes)
               ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem)
               : cudaSuccess;
}

}  // namespace mhcp
