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
  long long cost = 0;
  for (size_t i = 0; i < n; ++i)
    if (chosen(i))
      for (int r = 0; r < q_lens[i] * group; r += row_tile) cost += (long long)heads * (span(i, r) + fixed);
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
    for (size_t i = 0; i < n; ++i) {
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
            left -= take + fixed;
            if (left <= fixed) close();
          } while (it < count);
          const int parts = (int)(out->segs.size() - seg0);
          if (parts > 1) {
            out->joins.push_back({(int)i, h, r, out->parts, parts});
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

namespace {

constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;

// sequence of token t: the last i with q_start[i] <= t
__device__ __forceinline__ int seq_of(const PagedSeqs& s, int t) {
  int lo = 0, hi = s.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(s.q_start + mid) <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// New rows into pages. A unit is one V (16 bytes, or one element where rows
// are not 16-byte aligned) of the key or value of one (token, head); every
// thread has kCopyUnroll units in flight. Bound by HBM (each byte read once
// and written once).
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) k_paged_append(PagedSeqs s, PagedLayer c, unsigned units,
                                                               unsigned row_units, const V* __restrict__ k, size_t kt,
                                                               size_t kh, const V* __restrict__ v, size_t vt,
                                                               size_t vh, size_t tokens) {
  const unsigned per_token = units;  // heads * 2 * row_units
  const size_t total = tokens * per_token;
  const size_t base = (size_t)blockIdx.x * (kCopyThreads * kCopyUnroll) + threadIdx.x;
  V x[kCopyUnroll];
  V* dst[kCopyUnroll];
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u) {
    const size_t i = base + (size_t)u * kCopyThreads;
    dst[u] = nullptr;
    if (i >= total) continue;
    const size_t t = i / per_token;
    unsigned r = (unsigned)(i - t * per_token);
    const unsigned which = r / (units >> 1);
    r -= which * (units >> 1);
    const unsigned h = r / row_units, e = r - h * row_units;
    const int b = seq_of(s, (int)t);
    const int q1 = __ldg(s.q_start + b + 1);
    const int j = __ldg(s.kv_len + b) - (q1 - (int)t);
    if (j < 0) continue;  // a query in front of slot 0 has no slot
    const int page = __ldg(s.table + (size_t)b * s.stride + (j >> c.page_shift));
    const size_t row = (((size_t)page * c.heads + h) << c.page_shift) + (j & ((1 << c.page_shift) - 1));
    x[u] = which ? v[t * vt + h * vh + e] : k[t * kt + h * kh + e];
    dst[u] = static_cast<V*>(which ? c.values : c.keys) + row * row_units + e;
    if (!which && e == 0 && c.weights) c.weights[row] = 0.0f;
  }
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (dst[u]) *dst[u] = x[u];
}

// One (page, head) block of a sequence is contiguous on both sides: keys
// (blockIdx.z = 0) or values, whole blocks of the page's used rows.
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) k_paged_gather(const int* __restrict__ table, PagedLayer c, int len,
                                                               unsigned row_units, V* __restrict__ k,
                                                               V* __restrict__ v) {
  const int j0 = (int)blockIdx.x << c.page_shift, h = blockIdx.y;
  const int rows = min(1 << c.page_shift, len - j0);
  const int page = __ldg(table + blockIdx.x);
  const V* src = static_cast<const V*>(blockIdx.z ? c.values : c.keys) +
                 (((size_t)page * c.heads + h) << c.page_shift) * row_units;
  V* dst = (blockIdx.z ? v : k) + ((size_t)h * len + j0) * row_units;
  const unsigned n = rows * row_units;
  for (unsigned i0 = threadIdx.x; i0 < n; i0 += kCopyThreads * kCopyUnroll) {
    V x[kCopyUnroll];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
      if (i0 + u * kCopyThreads < n) x[u] = __ldg(src + i0 + u * kCopyThreads);
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
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

// Which slots stay, one CTA per (head, sequence, layer). The threshold among
// the slots that compete (all but the sinks and the recent ones) is the
// need-th largest key, found by a radix selection over three histograms of
// the key's bits; then one pass in slot order writes the kept slots: those
// above the threshold, and the first `ties` of those equal to it. Integer
// counts only, so the result does not depend on the order of the atomics.
__global__ void __launch_bounds__(kSelThreads) k_paged_select(PagedSeqs s, PagedLayer c, int budget, int recent,
                                                              int sinks, int* __restrict__ kept) {
  const int h = blockIdx.x, b = blockIdx.y;
  const size_t layer = blockIdx.z;
  const int n = __ldg(s.kv_len + b);
  int* out = kept + ((layer * s.n + b) * c.heads + h) * (size_t)budget;
  const int tid = threadIdx.x;
  if (n <= budget) {
    for (int i = tid; i < budget; i += kSelThreads) out[i] = i < n ? i : -1;
    return;
  }
  __shared__ int hist[kSelBins];
  __shared__ int warp_sums[32];
  __shared__ uint32_t sh_prefix;
  __shared__ int sh_need;
  const int* table = s.table + (size_t)b * s.stride;
  const int mask = (1 << c.page_shift) - 1;
  const float* w = c.weights + (((layer * c.pages) * c.heads) << c.page_shift);
  auto key_at = [&](int j) {
    const int page = __ldg(table + (j >> c.page_shift));
    return weight_key(__ldg(w + (((size_t)page * c.heads + h) << c.page_shift) + (j & mask)));
  };
  const int j0 = sinks, j1 = n - recent;  // sinks + recent <= budget < n
  int need = budget - sinks - recent;
  uint32_t prefix = 0, known = 0;  // the threshold's leading bits, and which they are
  if (need > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass == 2 ? 32 - 2 * kSelBits : kSelBits;
      const int shift = pass == 0 ? 32 - kSelBits : pass == 1 ? 32 - 2 * kSelBits : 0;
      for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
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
  const bool any = budget - sinks - recent > 0;
  int at = 0, ties = 0;
  for (int base = 0; base < n; base += kSelThreads) {
    const int j = base + tid;
    bool keep = false, tie = false;
    if (j < n) {
      if (j < j0 || j >= j1) keep = true;
      else if (any) {
        const uint32_t u = key_at(j);
        keep = u > prefix;
        tie = u == prefix;
      }
    }
    int sum;
    // both counts in one scan: at most 1024 of each
    const int pre = block_scan((keep ? 1 : 0) | (tie ? 1 << 16 : 0), warp_sums, &sum);
    const int tie_pre = ties + (pre >> 16);
    if (tie && tie_pre < need) keep = true;
    // of the ties in front of this slot, the first `need` of all are kept
    const int pos = at + (pre & 0xffff) + min(max(need - ties, 0), pre >> 16);
    if (keep) out[pos] = j;
    at += (sum & 0xffff) + min(max(need - ties, 0), sum >> 16);
    ties += sum >> 16;
  }
}

// Kept rows into their new pages. A unit is one V of the key or value of one
// kept slot; bound by HBM.
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) k_paged_move(PagedSeqs s, PagedLayer c, int budget,
                                                             const int* __restrict__ new_table, size_t new_stride,
                                                             const int* __restrict__ kept, unsigned row_units) {
  const int bh = blockIdx.y, h = bh % c.heads, b = bh / c.heads;
  const size_t layer = blockIdx.z;
  const int m = min(__ldg(s.kv_len + b), budget);
  const int* from = kept + ((layer * s.n + b) * c.heads + h) * (size_t)budget;
  const int* table = s.table + (size_t)b * s.stride;
  const int* to = new_table + (size_t)b * new_stride;
  const size_t layer_rows = ((size_t)c.pages * c.heads) << c.page_shift;
  const int mask = (1 << c.page_shift) - 1;
  const size_t total = (size_t)m * 2 * row_units;
  const size_t base = (size_t)blockIdx.x * (kCopyThreads * kCopyUnroll) + threadIdx.x;
  V x[kCopyUnroll];
  V* dst[kCopyUnroll];
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u) {
    const size_t i = base + (size_t)u * kCopyThreads;
    dst[u] = nullptr;
    if (i >= total) continue;
    const unsigned r = (unsigned)(i / (2 * row_units)), f = (unsigned)(i - (size_t)r * (2 * row_units));
    const bool val = f >= row_units;
    const unsigned e = val ? f - row_units : f;
    const int j = __ldg(from + r);
    const size_t src = layer * layer_rows +
                       (((size_t)__ldg(table + (j >> c.page_shift)) * c.heads + h) << c.page_shift) + (j & mask);
    const size_t row =
        layer * layer_rows + (((size_t)__ldg(to + (r >> c.page_shift)) * c.heads + h) << c.page_shift) + (r & mask);
    V* pool = static_cast<V*>(val ? c.values : c.keys);
    x[u] = pool[src * row_units + e];
    dst[u] = pool + row * row_units + e;
    if (f == 0) c.weights[row] = c.weights[src];
  }
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (dst[u]) *dst[u] = x[u];
}

size_t elem_size(int dtype) { return dtype == KVF_IN_F32 ? 4 : 2; }

template <typename V>
cudaError_t append_typed(const PagedSeqs& s, const PagedLayer& c, size_t tokens, const void* k, size_t kt, size_t kh,
                         const void* v, size_t vt, size_t vh, cudaStream_t st) {
  const size_t e = elem_size(c.dtype), per = sizeof(V) / e;
  const unsigned row_units = (unsigned)(c.dim / per), units = (unsigned)(2 * row_units * c.heads);
  const size_t blocks = (tokens * units + kCopyThreads * kCopyUnroll - 1) / (kCopyThreads * kCopyUnroll);
  if (blocks > 0x7fffffffu) return cudaErrorInvalidValue;
  k_paged_append<V><<<(unsigned)blocks, kCopyThreads, 0, st>>>(s, c, units, row_units, static_cast<const V*>(k),
                                                               kt / per, kh / per, static_cast<const V*>(v), vt / per,
                                                               vh / per, tokens);
  note_launches(1);
  return cudaGetLastError();
}

template <typename V>
cudaError_t gather_typed(const PagedSeqs& s, const PagedLayer& c, size_t seq, size_t len, void* k, void* v,
                         cudaStream_t st) {
  const unsigned row_units = (unsigned)(c.dim * elem_size(c.dtype) / sizeof(V));
  const size_t page = (size_t)1 << c.page_shift;
  const dim3 grid((unsigned)((len + page - 1) / page), (unsigned)c.heads, 2);
  k_paged_gather<V><<<grid, kCopyThreads, 0, st>>>(s.table + seq * s.stride, c, (int)len, row_units,
                                                   static_cast<V*>(k), static_cast<V*>(v));
  note_launches(1);
  return cudaGetLastError();
}

template <typename V>
cudaError_t move_typed(const PagedSeqs& s, const PagedLayer& c, size_t layers, size_t budget, const int* new_table,
                       size_t new_stride, const int* kept, cudaStream_t st) {
  const unsigned row_units = (unsigned)(c.dim * elem_size(c.dtype) / sizeof(V));
  const size_t per = kCopyThreads * kCopyUnroll;
  const size_t blocks = (budget * 2 * row_units + per - 1) / per;
  if (blocks > 0x7fffffffu) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)blocks, (unsigned)(s.n * c.heads), (unsigned)layers);
  k_paged_move<V><<<grid, kCopyThreads, 0, st>>>(s, c, (int)budget, new_table, new_stride, kept, row_units);
  note_launches(1);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_append(const PagedSeqs& s, const PagedLayer& c, size_t tokens, const void* k, size_t kt,
                                size_t kh, const void* v, size_t vt, size_t vh, cudaStream_t st) {
  const size_t e = elem_size(c.dtype);
  const bool wide = c.dim * e % 16 == 0 && (kt | kh | vt | vh) * e % 16 == 0 && aligned(k, 16) && aligned(v, 16);
  if (wide) return append_typed<uint4>(s, c, tokens, k, kt, kh, v, vt, vh, st);
  if (e == 4) return append_typed<uint32_t>(s, c, tokens, k, kt, kh, v, vt, vh, st);
  return append_typed<uint16_t>(s, c, tokens, k, kt, kh, v, vt, vh, st);
}

cudaError_t launch_paged_gather(const PagedSeqs& s, const PagedLayer& c, size_t seq, size_t len, void* k, void* v,
                                cudaStream_t st) {
  const size_t e = elem_size(c.dtype);
  if (c.dim * e % 16 == 0 && aligned(k, 16) && aligned(v, 16)) return gather_typed<uint4>(s, c, seq, len, k, v, st);
  if (e == 4) return gather_typed<uint32_t>(s, c, seq, len, k, v, st);
  return gather_typed<uint16_t>(s, c, seq, len, k, v, st);
}

cudaError_t launch_paged_evict(const PagedSeqs& s, const PagedLayer& c, size_t layers, size_t budget, size_t recent,
                               size_t sinks, const int* new_table, size_t new_stride, int* kept, cudaStream_t st) {
  const dim3 grid((unsigned)c.heads, (unsigned)s.n, (unsigned)layers);
  k_paged_select<<<grid, kSelThreads, 0, st>>>(s, c, (int)budget, (int)recent, (int)sinks, kept);
  note_launches(1);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const size_t es = elem_size(c.dtype);
  if (c.dim * es % 16 == 0) return move_typed<uint4>(s, c, layers, budget, new_table, new_stride, kept, st);
  if (es == 4) return move_typed<uint32_t>(s, c, layers, budget, new_table, new_stride, kept, st);
  return move_typed<uint16_t>(s, c, layers, budget, new_table, new_stride, kept, st);
}

}  // namespace kvf
