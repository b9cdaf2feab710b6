// What the tensor-core kernels of the paged cache share: tensor maps of the
// page pool, mbarriers, tensor-map loads.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "kvf_paged.cuh"

namespace kvf {

// A 16-bit page pool [pages * heads][page][dim] as boxes of 64 columns by
// `rows` slots of one (page, head), 128-byte swizzle; columns past dim arrive
// as zeros. false when the driver refuses.
inline bool paged_map(CUtensorMap* map, const PagedLayer& c, const void* pool, int rows) {
  auto enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tensor_map_encode_fn());
  if (!enc) return false;
  const cuuint64_t page = (cuuint64_t)1 << c.page_shift;
  const cuuint64_t gdim[3] = {(cuuint64_t)c.dim, page, (cuuint64_t)c.pages * c.heads};
  const cuuint64_t gstride[2] = {(cuuint64_t)c.dim * 2, page * c.dim * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)rows, 1};
  const cuuint32_t estride[3] = {1, 1, 1};
  const CUtensorMapDataType dt =
      c.dtype == KVF_IN_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return enc(map, dt, 3, const_cast<void*>(pool), gdim, gstride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// head dims that the tensor-core kernels take: 16-byte rows, at most 128
inline bool paged_tc_fits(int dtype, size_t dim) {
  return (dtype == KVF_IN_F16 || dtype == KVF_IN_BF16) && dim % 8 == 0 && dim <= 128;
}

#ifdef __CUDACC__
namespace ptx {
__device__ __forceinline__ uint32_t smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// one box: columns x.., slots y.. of (page, head) z
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
}  // namespace ptx

// 16-byte words of 16-bit elements: whether any is infinite or NaN (exponent
// bits all ones), and the word with those replaced by zero
template <typename T>
__device__ __forceinline__ bool drop_nonfinite(uint4& w) {
  constexpr uint32_t kExp = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  bool any = false;
  uint32_t* x = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((x[i] & kExp) == kExp) {
      x[i] &= 0xFFFF0000u;
      any = true;
    }
    if (((x[i] >> 16) & kExp) == kExp) {
      x[i] &= 0x0000FFFFu;
      any = true;
    }
  }
  return any;
}
#endif

}  // namespace kvf
