// Bulk tensor copies (TMA) and the barriers that go with them.
//
// Every wait has a limit, after which it reports failure; what follows from
// that is the caller's, none of them may wait again without a limit.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

namespace semicrf {

constexpr unsigned kWaitLimit = 1u << 20;

__device__ __forceinline__ unsigned smem_addr(const void* p) {
  return (unsigned)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void barrier_init(uint64_t* b, unsigned n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void barrier_arrive_here(uint64_t* b) {
  asm volatile("{.reg .b64 t; mbarrier.arrive.shared::cta.b64 t, [%0];}" ::"r"(smem_addr(b))
               : "memory");
}
// False when the phase does not complete within the limit.
__device__ __forceinline__ bool barrier_wait(uint64_t* b, unsigned parity) {
  for (unsigned k = 0; k < kWaitLimit; ++k) {
    unsigned done;
    asm volatile(
        "{.reg .pred p;"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;"
        "selp.u32 %0, 1, 0, p;}"
        : "=r"(done)
        : "r"(smem_addr(b)), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}
__device__ __forceinline__ void expect_bytes(uint64_t* b, unsigned n) {
  asm volatile("{.reg .b64 t; mbarrier.arrive.expect_tx.shared::cta.b64 t, [%0], %1;}" ::"r"(
                   smem_addr(b)),
               "r"(n)
               : "memory");
}
__device__ __forceinline__ void fetch_tile(unsigned dst, const CUtensorMap* map, int x, int y,
                                           uint64_t* b) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(smem_addr(b))
      : "memory");
}
__device__ __forceinline__ void fetch_tile(unsigned dst, const CUtensorMap* map, int x, int y,
                                           int z, uint64_t* b) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(b))
      : "memory");
}

// cuTensorMapEncodeTiled, looked up once: the library does not link libcuda.
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) !=
            cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// A map of `rank` dimensions, fastest first; strides in bytes, from the second on.
inline bool make_tensor_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base,
                            const cuuint64_t* dims, const cuuint64_t* strides,
                            const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return false;
  const cuuint32_t ones[3] = {1, 1, 1};
  return encode(map, type, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, ones,
                CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace semicrf
