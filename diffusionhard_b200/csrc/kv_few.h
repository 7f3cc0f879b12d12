// kv_few.h -- the launch of the kernel for few rows (kv_few.cu).
#pragma once

#include <cuda.h>

#include "kv_attention.cuh"

namespace dh {
namespace kv {

constexpr uint32_t kFewRows = 32;     // rows of an item at most
constexpr uint32_t kMaxCluster = 8;   // CTAs that share an item's keys

// Class `cls` of a's items on clusters of `cluster` CTAs (0: a warp an item).  maps: prefix K, V, own K,
// V (16 bits).
uint32_t launch_few(const CUtensorMap (&maps)[4], const Args& a, uint32_t cls, uint32_t cluster, bool int8, bool v_bf16,
                    cudaStream_t st);

}  // namespace kv
}  // namespace dh
