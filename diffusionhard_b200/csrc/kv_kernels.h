// kv_kernels.h -- launches that dh_kv_attention puts together: the kernel for few rows
// (kv_few.cu) and the one that turns int8 keys into f16 (kv_widen.cu).
#pragma once

#include <cuda.h>

#include "kv_attention.cuh"

namespace dh {
namespace kv {

// Rows of an item of the few-row kernel at most (16 rows and tensor-core tiles instead:
// 128 sequences of 512 int8 keys 32.9 and 59.4 us, 16 of 8192 57.4 and 78.8, one of 1000
// 10.4 and 12.4; its work grows with every 8 rows, a tile's does not up to 128).
constexpr uint32_t kFewRows = 16;
constexpr uint32_t kFewKeys16 = 32;  // 16-bit keys of a tile

// smem_optin_once, with an SM's whole carve-out as shared memory: two kernels that
// run beside each other on an SM need the same one.
template <class Kernel>
inline cudaError_t all_shared_once(Kernel kernel, uint32_t bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64 && (done.load(std::memory_order_acquire) >> dev & 1u)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    return e == cudaSuccess ? smem_optin_once(kernel, bytes, done) : e;
}

// Class `cls` of a's items on clusters of `cluster` CTAs (0: a warp an item).  maps:
// prefix K, V, own K, V (16 bits, tiles of kFewKeys16 keys).  beside: may begin while
// the kernel before it in the stream runs, whose CTA on an SM has `taken` bytes of
// shared memory.
uint32_t launch_few(const CUtensorMap (&maps)[4], const Args& a, uint32_t cls, uint32_t cluster, bool int8, bool v_bf16,
                    bool beside, uint32_t taken, cudaStream_t st);

// f16 rows [lines][capacity][64] of K and V, `lo` elements behind them (0: none) what
// they lack, and [lines] their exponents.
struct WideKeys {
    __half* k = nullptr;
    __half* v = nullptr;
    size_t lo = 0;
    float2* exps = nullptr;
};

// The int8 keys of a's sequences and `prefixes` prefixes.
uint32_t launch_widen(const Args& a, const WideKeys& prefix, const WideKeys& own, uint32_t prefixes, cudaStream_t st);

}  // namespace kv
}  // namespace dh
