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
// mbar_wait_bounded behind a first few polls that read neither the clock nor the
// flag: a poll takes about 110 cycles here even when the phase is complete, and
// the rest of the loop should add little to it
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const volatile int* abort_flag) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .u32 n;\n mov.u32 n, 128;\n"
      "WAIT:\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n @p bra DONE;\n"
      " sub.u32 n, n, 1;\n setp.ne.u32 q, n, 0;\n @q bra WAIT;\n"
      "DONE:\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done || mbar_wait_bounded(bar, parity, kWaitNs, abort_flag);
}
// one box: columns x.., slots y.. of (page, head) z
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
// ---- tcgen05 ---------------------------------------------------------------------
constexpr int kTile = 128;          // rows of an operand tile: MMA M, TMEM lanes
constexpr int kHalf = kTile * 128;  // bytes of 128 rows by 64 columns of 16 bits
constexpr uint32_t kTmemCols = 512;
// byte offset of 16-byte chunk `chunk` (8 columns) of row `row` of a tile
__device__ __forceinline__ uint32_t tile_off(int row, int chunk) {
  return (uint32_t)((chunk >> 3) * kHalf + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}
// Shared-memory matrix descriptors, 128-byte swizzle: 8-row groups 1024 bytes
// apart. K-major (Q, K): 64 columns per 128-byte row. MN-major (V as the second
// product's B, whose N runs along the row): 64-column halves kHalf apart. Only
// the low word depends on the address; steps along an operand are added to it.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return (addr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr) { return (addr >> 4) | ((uint32_t)(kHalf >> 4) << 16); }
// instruction descriptor: f32 accumulators, A and B of type T, M = 128
template <typename T>
constexpr uint32_t idesc(int n, bool b_mn) {
  const uint32_t t = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (t << 7) | (t << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kTile >> 4) << 24);
}
// The MMA warp runs its loop with all lanes, so that addresses and descriptors
// stay in uniform registers (one lane alone in a branch took several hundred
// cycles per tile to move them there); `lead` holds on the one lane that issues.
__device__ __forceinline__ void mma_ss(bool lead, uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, e;\n .reg .b64 da, db;\n setp.ne.b32 e, %0, 0;\n setp.ne.b32 p, %5, 0;\n"
      " mov.b64 da, {%2, %6};\n mov.b64 db, {%3, %6};\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%1], da, db, %4, p;\n}\n" ::"r"((uint32_t)lead),
      "r"(d), "r"(a), "r"(b), "r"(id), "r"(acc), "n"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_ts(bool lead, uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, e;\n .reg .b64 db;\n setp.ne.b32 e, %0, 0;\n setp.ne.b32 p, %5, 0;\n"
      " mov.b64 db, {%3, %6};\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], db, %4, p;\n}\n" ::"r"((uint32_t)lead),
      "r"(d), "r"(a), "r"(b), "r"(id), "r"(acc), "n"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void commit(bool lead, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.b32 e, %0, 0;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n}\n" ::"r"((uint32_t)lead),
      "r"(bar)
      : "memory");
}
// the same value on every lane, known as such to the compiler
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]),
        "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]),
        "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]),
        "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float* v) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]),
      "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]),
      "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// the largest of three (one instruction on sm_100), NaN if any is
__device__ __forceinline__ float max3(float x, float y, float z) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(x), "f"(y), "f"(z));
  return d;
}
// two additions in one instruction, each rounded as usual
__device__ __forceinline__ float2 fadd2(float2 x, float2 y) {
  unsigned long long a, b, d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(x.x), "f"(x.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(b) : "f"(y.x), "f"(y.y));
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(d));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
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
