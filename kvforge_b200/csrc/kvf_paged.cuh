// Paged cache: what its kernels (kvf_paged*.cu) and the C-ABI layer share.
#pragma once

#include <cuda_bf16.h>

#include <atomic>
#include <vector>

#include "kvf_internal.cuh"

namespace kvf {

// one layer of the page pool
struct PagedLayer {
  int dtype = 0;
  int page_shift = 0;  // page size = 1 << page_shift
  int pages = 0, heads = 0, dim = 0;
  void* keys = nullptr;  // [pages, heads, page, dim]
  void* values = nullptr;
  float* weights = nullptr;  // [pages, heads, page] or nullptr
};

// the sequences of a plan, on the device
struct PagedSeqs {
  const int* table = nullptr;  // [n, stride] pages
  size_t stride = 0;
  const int* kv_len = nullptr;   // [n]
  const int* q_start = nullptr;  // [n + 1] first token of each sequence
};

// Attention work. A KV head's query rows of one sequence are numbered
// token * group + (query head within the group); a tile is `row_tile` of them,
// and an iteration is one tile of `key_tile` slots. One CTA walks the segments
// [first[cta], first[cta + 1]), each a range of iterations of one row tile. A
// tile cut into several segments leaves partial results (part >= 0: their
// slot) that are joined afterwards; part = -1 writes the output itself.
struct PagedSeg {
  int seq, head, row0, it0, it1, part;
};
struct PagedJoin {
  int seq, head, row0, part0, parts;
  int rows, token0;  // rows of the tile, first token of the sequence
};
// what covers one tile of slots of one sequence (weights): (sequence, first slot)
struct PagedSlots {
  int seq, slot0;
};
enum PagedKernel { kPagedGeneric = 0, kPagedDecode = 1, kPagedChunk = 2 };
struct PagedWork {
  int kernel = kPagedGeneric;
  int row_tile = 0, key_tile = 0;
  int ctas = 0, joins_n = 0, parts = 0;
  const PagedSeg* segs = nullptr;  // device
  const int* first = nullptr;
  const PagedJoin* joins = nullptr;
};

// Key tiles that a row tile visits: the first `nsink` tiles (sinks in front of
// the window), then the tiles from `first` on; iteration t is tile
// t < nsink ? t : first + t - nsink, `count` in all.
struct PagedSpan {
  int nsink, first, count;
};
__host__ __device__ inline PagedSpan paged_span(int row0, int row_tile, int group, int kv_len, int q_len, int window,
                                                int sinks, int key_tile) {
  const int ta = row0 / group;
  int last = row0 + row_tile - 1;  // row tiles stay far below 2^31 rows (checked when a plan is made)
  if (last > q_len * group - 1) last = q_len * group - 1;
  const int tb = last / group;
  const int pa = kv_len - q_len + ta, pb = kv_len - q_len + tb;  // slots of the first and last token
  PagedSpan s{0, 0, 0};
  if (pb < 0) return s;
  const int end = pb / key_tile + 1;
  if (window) {
    const int lo = pa - window + 1;
    s.first = lo > 0 ? lo / key_tile : 0;
    // without the rounding term the sum stays in range for any sinks
    const int st = sinks / key_tile + (sinks % key_tile ? 1 : 0);
    s.nsink = st < s.first ? st : s.first;
  }
  s.count = s.nsink + end - s.first;
  return s;
}

// whether the query at slot `pos` sees slot j
__host__ __device__ inline bool paged_sees(int pos, int j, int window, int sinks) {
  return j <= pos && (window == 0 || j > pos - window || j < sinks);
}

struct PagedAttn {
  PagedSeqs s;
  PagedLayer c;
  int group = 1, window = 0, sinks = 0;
  const void* q = nullptr;
  size_t q_token = 0, q_head = 0;  // strides in elements
  float scale2 = 0.f;              // scale * log2(e): scores are held in base 2
  void* out = nullptr;             // [tokens, heads * group, dim]
  float* lse = nullptr;            // [tokens, heads * group] or nullptr
  float* part_o = nullptr;         // [parts, row_tile, dim] sums before the division
  float* part_ml = nullptr;        // [parts, row_tile, 2] maximum (base 2) and sum
  unsigned* status = nullptr;
};

// host side of a work list
struct PagedWorkHost {
  int kernel = kPagedGeneric;
  int row_tile = 0, key_tile = 0, parts = 0;
  std::vector<PagedSeg> segs;
  std::vector<int> first;
  std::vector<PagedJoin> joins;
};
// Splits the row tiles of the sequences with lo <= rows <= hi (rows = new
// tokens * group) over at most `slots` CTAs of equal cost (iterations, at least
// one, plus `fixed` for every segment); no segment but a tile's last is shorter
// than `least` iterations. A tile without iterations is one segment.
void paged_split(const int* q_lens, const int* kv_lens, size_t n, int heads, int group, int window, int sinks,
                 long long lo, long long hi, int row_tile, int key_tile, int slots, int least, int fixed,
                 PagedWorkHost* out);

// Iterations of those row tiles.
long long paged_tiles(const int* q_lens, const int* kv_lens, size_t n, int heads, int group, int window, int sinks,
                      long long lo, long long hi, int row_tile, int key_tile);

// ---- launchers ---------------------------------------------------------------
// place [tokens]: page * 128 + row of every token, -1 for none
cudaError_t launch_paged_append(const long long* place, const PagedLayer& c, size_t tokens, const void* k, size_t kt,
                                size_t kh, const void* v, size_t vt, size_t vh, cudaStream_t st);
// host arrays of pages up to this many words travel as kernel parameters
constexpr int kPageListMax = 960;
// pages: the sequence's, on the host
cudaError_t launch_paged_gather(const int* pages, const PagedLayer& c, size_t len, void* k, void* v, cudaStream_t st);
// tables (host): lengths [n], pages [n, stride], new pages [n, new_stride], one
// behind the other, and the same on the device, or nullptr when they are at most
// kPageListMax words; longest: the largest length; layers stacked `pages` apart;
// kept [layers, n, heads, budget]
cudaError_t launch_paged_evict(const int* tables, const int* tables_dev, size_t n, size_t stride, size_t new_stride,
                               size_t longest, const PagedLayer& c, size_t layers, size_t budget, size_t recent,
                               size_t sinks, int* kept, cudaStream_t st);

// CUDA-core attention: every type and head_dim up to kGenDimMost
constexpr int kGenDimMost = 256;
constexpr int kGenRows = 64, kGenRowsShort = 16, kGenKeys = 64;
// tiles for more than kGenRows rows, head_dim up to kGenDimLong
constexpr int kGenRowsLong = 128, kGenKeysLong = 128, kGenDimLong = 128;
cudaError_t launch_paged_attn_generic(const PagedAttn& a, const PagedWork& w, cudaStream_t st);
// joins the partial results of its cut tiles
cudaError_t launch_paged_join(const PagedAttn& a, const PagedWork& w, cudaStream_t st);
// weight = decay * weight + column sums of the softmax, from a.lse (natural
// logarithm): CUDA cores, every type; slots: tiles of kGenKeys slots
cudaError_t launch_paged_weights_generic(const PagedAttn& a, const PagedSlots* tiles, size_t ntiles, bool few_rows,
                                         float decay, cudaStream_t st);

// 16-bit pools with head dims of whole 16-byte rows up to 128, sequences of at
// most kDecodeRows rows per KV head; scores (or nullptr): see the kernel
constexpr int kDecodeRows = 16, kDecodeKeys = 64;
constexpr int kDecodeWeightSlots = 256;  // slots of a tile of launch_paged_decode_weights
cudaError_t launch_paged_decode(const PagedAttn& a, const PagedWork& w, float* scores, const long long* score_at,
                                cudaStream_t st);
cudaError_t launch_paged_decode_weights(const PagedAttn& a, const PagedSlots* tiles, size_t ntiles,
                                        const float* scores, const long long* score_at, float decay, cudaStream_t st);

// the same pools, sequences of more rows
constexpr int kChunkRows = 256, kChunkKeys = 128;
cudaError_t launch_paged_chunk(const PagedAttn& a, const PagedWork& w, cudaStream_t st);

// their attention weights, from a.lse: up to 128 query heads per KV head;
// part_w: 2 * w.parts * kWeightSlots floats. cudaErrorNotSupported (before any
// launch) where the queries' strides or alignment do not suit tensor maps.
// The work: tiles of kWeightSlots slots by row tiles of 128 / group tokens.
constexpr int kWeightSlots = 256;
void paged_split_slots(const int* q_lens, const int* kv_lens, size_t n, int heads, int group, int window, int sinks,
                       long long more_than, int slots, PagedWorkHost* out);
cudaError_t launch_paged_chunk_weights(const PagedAttn& a, const PagedWork& w, size_t tokens, float* part_w,
                                       float decay, cudaStream_t st);

#ifdef __CUDACC__
// Opts a kernel in to `bytes` of dynamic shared memory, the most that any of its
// launches asks for, once per device (each call site passes flags of its own). A
// limit set for each launch could be lowered by another thread in front of it.
struct OptInOnce {
  static constexpr int kDevices = 64;
  std::atomic<size_t> bytes[kDevices];
};
template <typename K>
cudaError_t opt_in_once(OptInOnce& done, K kern, size_t bytes) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev < 0 || dev >= OptInOnce::kDevices) return e != cudaSuccess ? e : cudaErrorInvalidDevice;
  if (done.bytes[dev].load(std::memory_order_acquire) >= bytes) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done.bytes[dev].store(bytes, std::memory_order_release);
  return e;
}

// Launches a kernel that may begin while the one before it in the stream ends:
// what it does before wait_for_previous() must not depend on that one.
template <typename... P, typename... A>
cudaError_t launch_behind(void (*kern)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
}
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// first element of slot j of a sequence (its row of the page table) in head h
__device__ __forceinline__ size_t paged_row(const int* __restrict__ table, const PagedLayer& c, int h, int j) {
  const int page = __ldg(table + (j >> c.page_shift));
  return ((((size_t)page * c.heads + h) << c.page_shift) + (j & ((1 << c.page_shift) - 1))) * c.dim;
}
#endif

}  // namespace kvf
