// dense_tc.cuh - what the tcgen05 products of the dense feed-forward operators share: operand descriptors, launch helpers.
#pragma once

#include <atomic>

#include "dense.hpp"
#include "dense_launch.cuh"
#include "dense_math.cuh"
#include "sm100.cuh"

namespace vkernels::kernels::cuda {

CUtensorMap sm100_make_map_bf16(const void* ptr, uint64_t inner, uint64_t outer, uint64_t pitch_bytes, uint32_t box_outer);
int* sm100_status_address();

namespace {

// .aligned: the whole warp executes it as one. Its lanes part before it wherever rows behind the last are not stored, and nothing but
// the barrier brings them together for certain.
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t* v) {
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
// The same of two places at once.
__device__ __forceinline__ void tc_ld16_two(uint32_t taddr, uint32_t* v, uint32_t uaddr, uint32_t* u) {
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%32];\n"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%33];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(taddr), "r"(uaddr)
      : "memory");
}
// Descriptor of a staged operand. Contiguous along k: rows of 64 k, groups of 8 rows 1024 bytes apart. Contiguous along the
// other index: chunks of 64 indexes x 64 k, 8192 bytes apart, groups of 8 k 1024 bytes apart. 128-byte swizzle either way.
__device__ __forceinline__ uint64_t operand_desc(uint32_t smem_addr, int mn_major) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(mn_major ? 8192 >> 4 : 1) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// Instruction descriptor: fp32 accumulate, both operands of the one type, either order.
template <int TYPE>
__device__ __forceinline__ uint32_t operand_idesc(int m, int n, int a_mn, int b_mn) {
  return (1u << 4) | (TYPE == kDenseBf16 ? (1u << 7) | (1u << 10) : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

int* status_address() {
  static std::atomic<int*> known[64];
  int dev = 0;
  VK_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return sm100_status_address();
  int* p = known[dev].load();
  if (p == nullptr) known[dev].store(p = sm100_status_address());
  return p;
}

}  // namespace

}  // namespace vkernels::kernels::cuda
