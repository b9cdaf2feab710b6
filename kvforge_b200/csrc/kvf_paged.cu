// Paged cache: page transfer (append, gather), eviction by accumulated
// attention weight, and the host-side division of attention work. The
// reference has no paged cache; the formulas are in include/kvforge.h.
#include <algorithm>

#include "kvf_paged.cuh"

namespace kvf {

// ---- division of the attention work -------------------------------------------
void paged_split(const int* q_lens, const int* kv_lens, size_t n, int heads, int group, int window, int sinks,
                 long long lo, long long hi, int row_tile, int key_tile, int slots, int least, int fixed,
                 PagedWorkHost* out) {
  out->row_tile = row_tile;
  out->key_tile = key_tile;
  auto chosen = [&](size_t i) {
    const long long rows = (long long)q_lens[i] * group;
    return rows > 0 && rows >= lo && rows <= hi;
  };
  auto span = [&](size_t i, int row0) {
    return paged_span(row0, row_tile, group, kv_lens[i], q_lens[i], window, sinks, key_tile).count;
  };
  // a tile that sees no slot is a segment all the same: its rows are written
  auto price = [&](int iterations) { return std::max(iterations, 1) + fixed; };
  long long cost = 0;
  for (size_t i = 0; i < n; ++i)
    if (chosen(i))
      for (int r = 0; r < q_lens[i] * group; r += row_tile) cost += (long long)heads * price(span(i, r));
  if (!cost) return;
  long long quota = std::max<long long>((cost + slots - 1) / slots, least + fixed);
  // a CTA that closes early (what is left of its quota is too short to cut a
  // tile for) can push the count past `slots`: then with a larger quota
  for (int attempt = 0;; ++attempt) {
    out->segs.clear();
    out->first.assign(1, 0);
    out->joins.clear();
    out->parts = 0;
    long long left = quota;
    auto close = [&] {
      out->first.push_back((int)out->segs.size());
      left = quota;
    };
    int tokens = 0;  // in front of sequence i
    for (size_t i = 0; i < n; tokens += q_lens[i++]) {
      if (!chosen(i)) continue;
      for (int h = 0; h < heads; ++h)
        for (int r = 0; r < q_lens[i] * group; r += row_tile) {
          const int count = span(i, r);
          const size_t seg0 = out->segs.size();
          int it = 0;
          do {
            const bool fresh = (int)out->segs.size() == out->first.back();
            if (!fresh && left - fixed < std::min(least, count - it)) close();
            int take = (int)std::min<long long>(count - it, std::max<long long>(left - fixed, 1));
            if (count - it - take < least) take = count - it;  // no sliver behind the cut
            out->segs.push_back({(int)i, h, r, it, it + take, -1});
            it += take;
            left -= price(take);
            if (left <= fixed) close();
          } while (it < count);
          const int parts = (int)(out->segs.size() - seg0);
          if (parts > 1) {
            out->joins.push_back({(int)i, h, r, out->parts, parts, std::min(row_tile, q_lens[i] * group - r), tokens});
            for (size_t k = seg0; k < out->segs.size(); ++k) out->segs[k].part = out->parts++;
          }
        }
    }
    if ((int)out->segs.size() > out->first.back()) out->first.push_back((int)out->segs.size());
    // a quota of a whole number of tiles may need a few CTAs more; they only
    // cost a wave when the extra ones do not fit beside the others
    if ((int)out->first.size() - 1 <= slots || attempt == 16) return;
    quota += std::max<long long>(1, quota / 32);
  }
}

long long paged_tiles(const int* q_lens, const int* kv_lens, size_t n, int heads, int group, int window, int sinks,
                      long long lo, long long hi, int row_tile, int key_tile) {
  long long tiles = 0;
  for (size_t i = 0; i < n; ++i) {
    const long long rows = (long long)q_lens[i] * group;
    if (rows < lo || rows > hi) continue;
    for (int r = 0; r < rows; r += row_tile)
      tiles += (long long)heads * paged_span(r, row_tile, group, kv_lens[i], q_lens[i], window, sinks, key_tile).count;
  }
  return tiles;
}

namespace {

constexpr int kCopyThreads = 256;
constexpr int kRowsPerWarp = 8;

// New rows into pages. A warp takes kRowsPerWarp (token, head) pairs, whose
// places lanes 0-7 look up, and has all their loads in flight before the first
// store; a unit is one V (16 bytes, or one element where rows are not 16-byte
// aligned). `place` holds every token's page and row (page * 128 + row, -1
// where a query lies in front of slot 0). Bound by HBM: each byte is read once
// and written once (16384 tokens of 8 heads of 128 in 16 bits, 134 MB: 23 us,
// 5.8 TB/s; a warp per row with one load in flight took 30).
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) k_paged_append(const long long* __restrict__ place, PagedLayer c,
                                                               unsigned units, const V* __restrict__ k, size_t kt,
                                                               size_t kh, const V* __restrict__ v, size_t vt,
                                                               size_t vh, unsigned pairs) {
  const int lane = threadIdx.x & 31;
  const unsigned p0 = (blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5)) * kRowsPerWarp;
  unsigned long long row = ~0ull, from_k = 0, from_v = 0;
  if (lane < kRowsPerWarp && p0 + lane < pairs) {
    const unsigned t = (p0 + lane) / c.heads, h = (p0 + lane) - t * c.heads;
    const long long at = __ldg(place + t);
    if (at >= 0) {
      row = ((((unsigned long long)(at >> 7)) * c.heads + h) << c.page_shift) + (unsigned)(at & 127);
      if (c.weights) c.weights[row] = 0.0f;
    }
    from_k = t * kt + h * kh;
    from_v = t * vt + h * vh;
  }
  for (unsigned e0 = 0; e0 < 2 * units; e0 += 32) {
    const unsigned e = e0 + lane;
    const bool val = e >= units;
    const unsigned col = val ? e - units : e;
    V x[kRowsPerWarp];
    unsigned long long dst[kRowsPerWarp];
#pragma unroll
    for (int u = 0; u < kRowsPerWarp; ++u) {
      dst[u] = __shfl_sync(0xffffffffu, row, u);
      const unsigned long long sk = __shfl_sync(0xffffffffu, from_k, u), sv = __shfl_sync(0xffffffffu, from_v, u);
      if (dst[u] != ~0ull && e < 2 * units) x[u] = val ? v[sv + col] : k[sk + col];
    }
    V* pool = static_cast<V*>(val ? c.values : c.keys);
#pragma unroll
    for (int u = 0; u < kRowsPerWarp; ++u)
      if (dst[u] != ~0ull && e < 2 * units) pool[dst[u] * units + col] = x[u];
  }
}

// pages of a sequence, as a kernel parameter
struct PageList {
  int v[kPageListMax];
};

// One (page, head) block of a sequence is contiguous on both sides: keys
// (blockIdx.z = 0) or values, whole blocks of the page's used rows. Bound by HBM
// (32768 tokens of 8 heads of 128 in 16 bits, 268 MB: 42.5 us, 6.3 TB/s).
constexpr int kGatherUnroll = 4;
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) k_paged_gather(const __grid_constant__ PageList pages, PagedLayer c,
                                                               int first, int len, unsigned row_units,
                                                               V* __restrict__ k, V* __restrict__ v) {
  const int j0 = (first + (int)blockIdx.x) << c.page_shift, h = blockIdx.y;
  const int rows = min(1 << c.page_shift, len - j0);
  const int page = pages.v[blockIdx.x];
  const V* src = static_cast<const V*>(blockIdx.z ? c.values : c.keys) +
                 (((size_t)page * c.heads + h) << c.page_shift) * row_units;
  V* dst = (blockIdx.z ? v : k) + ((size_t)h * len + j0) * row_units;
  const unsigned n = rows * row_units;
  for (unsigned i0 = threadIdx.x; i0 < n; i0 += kCopyThreads * kGatherUnroll) {
    V x[kGatherUnroll];
#pragma unroll
    for (int u = 0; u < kGatherUnroll; ++u)
      if (i0 + u * kCopyThreads < n) x[u] = __ldg(src + i0 + u * kCopyThreads);
#pragma unroll
    for (int u = 0; u < kGatherUnroll; ++u)
      if (i0 + u * kCopyThreads < n) dst[i0 + u * kCopyThreads] = x[u];
  }
}

// order-preserving image of a weight: NaN lowest, -0 equal to +0
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w + 0.0f);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}

constexpr int kSelThreads = 1024;
constexpr int kSelBits = 11, kSelBins = 1 << kSelBits;  // 32 key bits in passes of 11, 11 and 10

// exclusive prefix sum over the block's threads; total in *sum
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* sum) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[w] = x;
  __syncthreads();
  if (w == 0) {
    int y = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    warp_sums[lane] = y;
  }
  __syncthreads();
  *sum = warp_sums[31];
  return x - v + (w ? warp_sums[w - 1] : 0);
}

// what an eviction reads of its sequences: lengths [n], pages [n, stride], new
// pages [n, new_stride], one behind the other; in the parameter where they fit
struct EvictTables {
  const int* p;  // device, or nullptr: v
  int n, stride, new_stride;
  int v[kPageListMax];
  __device__ __forceinline__ const int* lens() const { return p ? p : v; }
  __device__ __forceinline__ const int* pages(int b) const { return lens() + n + (size_t)b * stride; }
  __device__ __forceinline__ const int* new_pages(int b) const {
    return lens() + n + (size_t)n * stride + (size_t)b * new_stride;
  }
};

// Which slots stay, one CTA per (head, sequence, layer). The threshold among
// the slots that compete (all but the sinks and the recent ones) is the
// need-th largest key, found by a radix selection over three histograms of
// the key's bits; then every thread takes a run of slots and, after prefix sums
// over the runs' counts, writes those of its run that stay, in order: those
// above the threshold, and the first `need` of those equal to it. The keys are
// kept in shared memory (one word of padding after 32, so that runs start in
// different banks) where they fit, and read again from L2 otherwise. Integer
// counts only, so the result does not depend on the order of the atomics.
// Bound by latencies: four passes of a CTA over its keys (44 us for 128 CTAs of
// 32768 slots; 62 with every pass from L2).
__global__ void __launch_bounds__(kSelThreads) k_paged_select(const __grid_constant__ EvictTables tab, PagedLayer c,
                                                              int budget, int recent, int sinks, int cached,
                                                              int* __restrict__ kept) {
  extern __shared__ uint32_t keys[];  // [cached + cached / 32 + 1]
  const int h = blockIdx.x, b = blockIdx.y;
  const size_t layer = blockIdx.z;
  const int n = tab.lens()[b];
  int* out = kept + ((layer * tab.n + b) * c.heads + h) * (size_t)budget;
  const int tid = threadIdx.x;
  if (n <= budget) {
    for (int i = tid; i < budget; i += kSelThreads) out[i] = i < n ? i : -1;
    return;
  }
  __shared__ int hist[kSelBins];
  __shared__ int warp_sums[32];
  __shared__ uint32_t sh_prefix;
  __shared__ int sh_need;
  const int* table = tab.pages(b);
  const int mask = (1 << c.page_shift) - 1;
  const float* w = c.weights + (((layer * c.pages) * c.heads) << c.page_shift);
  auto load_key = [&](int j) {
    return weight_key(w[(((size_t)table[j >> c.page_shift] * c.heads + h) << c.page_shift) + (j & mask)]);
  };
  const bool have = n <= cached;
  if (have) {
#pragma unroll 8
    for (int j = tid; j < n; j += kSelThreads) keys[j + (j >> 5)] = load_key(j);
    __syncthreads();
  }
  auto key_at = [&](int j) { return have ? keys[j + (j >> 5)] : load_key(j); };
  const int j0 = sinks, j1 = n - recent;  // sinks + recent <= budget < n
  int need = budget - sinks - recent;
  const bool any = need > 0;
  uint32_t prefix = 0, known = 0;  // the threshold's leading bits, and which they are
  if (any) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass == 2 ? 32 - 2 * kSelBits : kSelBits;
      const int shift = pass == 0 ? 32 - kSelBits : pass == 1 ? 32 - 2 * kSelBits : 0;
      for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
#pragma unroll 4
      for (int j = j0 + tid; j < j1; j += kSelThreads) {
        const uint32_t u = key_at(j);
        if ((u & known) == prefix) atomicAdd(&hist[(u >> shift) & ((1u << bits) - 1)], 1);
      }
      __syncthreads();
      // the bin, counted from the largest, in which the need-th key lies:
      // thread t owns the bins 2047 - 2t and 2046 - 2t
      const int hi = kSelBins - 1 - 2 * tid;
      const int a = hist[hi], d = hist[hi - 1];
      int total;
      const int before = block_scan(a + d, warp_sums, &total);
      if (before < need && before + a + d >= need) {
        const bool second = before + a < need;
        sh_prefix = prefix | ((uint32_t)(second ? hi - 1 : hi) << shift);
        sh_need = need - before - (second ? a : 0);
      }
      __syncthreads();
      prefix = sh_prefix;
      need = sh_need;
      known |= ((1u << bits) - 1) << shift;
    }
  }
  // need: how many of the slots equal to the threshold stay, the lowest first
  const int run = (n + kSelThreads - 1) / kSelThreads;
  const int i0 = min(n, tid * run), i1 = min(n, i0 + run);
  int keep = 0, ties = 0;
  for (int j = i0; j < i1; ++j) {
    if (j < j0 || j >= j1) {
      ++keep;
    } else if (any) {
      const uint32_t u = key_at(j);
      keep += u > prefix;
      ties += u == prefix;
    }
  }
  int total;
  const int keep0 = block_scan(keep, warp_sums, &total), ties0 = block_scan(ties, warp_sums, &total);
  int pos = keep0 + (any ? min(ties0, need) : 0), left = any ? max(0, need - ties0) : 0;
  for (int j = i0; j < i1; ++j) {
    bool stays = j < j0 || j >= j1;
    if (!stays && any) {
      const uint32_t u = key_at(j);
      stays = u > prefix || (u == prefix && left-- > 0);
    }
    if (stays) out[pos++] = j;
  }
}

// Kept rows into their new pages, kRowsPerWarp slots per warp; bound by HBM (16
// layers, 8192 of 32768 slots, 8 heads of 128 in 16 bits, 1.04 GB: 172 us,
// 6.1 TB/s; a row per warp at a time took 243).
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) k_paged_move(const __grid_constant__ EvictTables tab, PagedLayer c,
                                                             int budget, const int* __restrict__ kept,
                                                             unsigned units) {
  const int bh = blockIdx.y, h = bh % c.heads, b = bh / c.heads;
  const size_t layer = blockIdx.z;
  const int m = min(tab.lens()[b], budget), lane = threadIdx.x & 31;
  const int r0 = (blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5)) * kRowsPerWarp;
  if (r0 >= m) return;
  const int mask = (1 << c.page_shift) - 1;
  const unsigned long long rows = layer * (((unsigned long long)c.pages * c.heads) << c.page_shift);
  unsigned long long from = ~0ull, to = 0;
  if (lane < kRowsPerWarp && r0 + lane < m) {
    const int r = r0 + lane;
    const int j = __ldg(kept + ((layer * tab.n + b) * c.heads + h) * (size_t)budget + r);
    from = rows + (((unsigned long long)tab.pages(b)[j >> c.page_shift] * c.heads + h) << c.page_shift) + (j & mask);
    to = rows + (((unsigned long long)tab.new_pages(b)[r >> c.page_shift] * c.heads + h) << c.page_shift) + (r & mask);
    c.weights[to] = c.weights[from];
  }
  for (unsigned e0 = 0; e0 < 2 * units; e0 += 32) {
    const unsigned e = e0 + lane;
    const bool val = e >= units;
    const unsigned col = val ? e - units : e;
    V* pool = static_cast<V*>(val ? c.values : c.keys);
    V x[kRowsPerWarp];
#pragma unroll
    for (int u = 0; u < kRowsPerWarp; ++u) {
      const unsigned long long src = __shfl_sync(0xffffffffu, from, u);
      if (src != ~0ull && e < 2 * units) x[u] = __ldcs(pool + src * units + col);
    }
#pragma unroll
    for (int u = 0; u < kRowsPerWarp; ++u) {
      const unsigned long long src = __shfl_sync(0xffffffffu, from, u), dst = __shfl_sync(0xffffffffu, to, u);
      if (src != ~0ull && e < 2 * units) pool[dst * units + col] = x[u];
    }
  }
}

size_t elem_size(int dtype) { return dtype == KVF_IN_F32 ? 4 : 2; }

template <typename V>
cudaError_t append_typed(const long long* place, const PagedLayer& c, size_t tokens, const void* k, size_t kt,
                         size_t kh, const void* v, size_t vt, size_t vh, cudaStream_t st) {
  const size_t e = elem_size(c.dtype), per = sizeof(V) / e;
  const size_t pairs = tokens * c.heads, per_block = kCopyThreads / 32 * kRowsPerWarp;
  if (pairs > 0x7fffffffu) return cudaErrorInvalidValue;
  k_paged_append<V><<<(unsigned)((pairs + per_block - 1) / per_block), kCopyThreads, 0, st>>>(
      place, c, (unsigned)(c.dim / per), static_cast<const V*>(k), kt / per, kh / per, static_cast<const V*>(v),
      vt / per, vh / per, (unsigned)pairs);
  note_launches(1);
  return cudaGetLastError();
}

template <typename V>
cudaError_t gather_typed(const int* pages, const PagedLayer& c, size_t len, void* k, void* v, cudaStream_t st) {
  const unsigned row_units = (unsigned)(c.dim * elem_size(c.dtype) / sizeof(V));
  const size_t page = (size_t)1 << c.page_shift, n = (len + page - 1) / page;
  for (size_t first = 0; first < n; first += kPageListMax) {
    const size_t m = std::min<size_t>(kPageListMax, n - first);
    PageList list;
    std::copy(pages + first, pages + first + m, list.v);
    k_paged_gather<V><<<dim3((unsigned)m, (unsigned)c.heads, 2), kCopyThreads, 0, st>>>(
        list, c, (int)first, (int)len, row_units, static_cast<V*>(k), static_cast<V*>(v));
    note_launches(1);
  }
  return cudaGetLastError();
}

template <typename V>
cudaError_t move_typed(const EvictTables& tab, const PagedLayer& c, size_t layers, size_t budget, const int* kept,
                       cudaStream_t st) {
  const unsigned units = (unsigned)(c.dim * elem_size(c.dtype) / sizeof(V));
  const size_t per = kCopyThreads / 32 * kRowsPerWarp;
  const dim3 grid((unsigned)((budget + per - 1) / per), (unsigned)(tab.n * c.heads), (unsigned)layers);
  k_paged_move<V><<<grid, kCopyThreads, 0, st>>>(tab, c, (int)budget, kept, units);
  note_launches(1);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_append(const long long* place, const PagedLayer& c, size_t tokens, const void* k, size_t kt,
                                size_t kh, const void* v, size_t vt, size_t vh, cudaStream_t st) {
  const size_t e = elem_size(c.dtype);
  const bool wide = c.dim * e % 16 == 0 && (kt | kh | vt | vh) * e % 16 == 0 && aligned(k, 16) && aligned(v, 16);
  if (wide) return append_typed<uint4>(place, c, tokens, k, kt, kh, v, vt, vh, st);
  if (e == 4) return append_typed<uint32_t>(place, c, tokens, k, kt, kh, v, vt, vh, st);
  return append_typed<uint16_t>(place, c, tokens, k, kt, kh, v, vt, vh, st);
}

cudaError_t launch_paged_gather(const int* pages, const PagedLayer& c, size_t len, void* k, void* v,
                                cudaStream_t st) {
  const size_t e = elem_size(c.dtype);
  if (c.dim * e % 16 == 0 && aligned(k, 16) && aligned(v, 16)) return gather_typed<uint4>(pages, c, len, k, v, st);
  if (e == 4) return gather_typed<uint32_t>(pages, c, len, k, v, st);
  return gather_typed<uint16_t>(pages, c, len, k, v, st);
}

cudaError_t launch_paged_evict(const int* tables, const int* tables_dev, size_t n, size_t stride, size_t new_stride,
                               size_t longest, const PagedLayer& c, size_t layers, size_t budget, size_t recent,
                               size_t sinks, int* kept, cudaStream_t st) {
  EvictTables tab;
  tab.p = tables_dev;
  tab.n = (int)n;
  tab.stride = (int)stride;
  tab.new_stride = (int)new_stride;
  if (!tables_dev) std::copy(tables, tables + n + n * stride + n * new_stride, tab.v);
  // as many keys as shared memory holds
  constexpr size_t kKeyMost = 50 * 1024;
  auto key_bytes = [](size_t keys) { return (keys + keys / 32 + 1) * 4; };
  const size_t cached = std::min(longest, kKeyMost), smem = key_bytes(cached);
  static OptInOnce done;
  cudaError_t e = opt_in_once(done, k_paged_select, key_bytes(kKeyMost));
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)c.heads, (unsigned)n, (unsigned)layers);
  k_paged_select<<<grid, kSelThreads, smem, st>>>(tab, c, (int)budget, (int)recent, (int)sinks, (int)cached, kept);
  note_launches(1);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const size_t es = elem_size(c.dtype);
  if (c.dim * es % 16 == 0) return move_typed<uint4>(tab, c, layers, budget, kept, st);
  if (es == 4) return move_typed<uint32_t>(tab, c, layers, budget, kept, st);
  return move_typed<uint16_t>(tab, c, layers, budget, kept, st);
}

}  // namespace kvf
