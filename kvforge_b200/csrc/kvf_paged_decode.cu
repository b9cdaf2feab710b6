// Attention of few rows (single tokens, short drafts) over a paged 16-bit
// cache: at most 16 query rows per KV head and sequence.
//
// The formulas are those of kvf_paged_attn.cu. Every key and value is read
// once for up to 16 rows, so the kernel is bound by HBM; its products run on
// mma.sync m16n8k16 with the rows as M (tcgen05's M of 128 would be mostly
// padding, and the tensor cores are not what limits here). One producer warp
// keeps tensor-map loads of 64-slot tiles in flight, a box per page, and puts
// the rows of the next segment beside them; two CTAs per SM keep about 190 KB of
// loads in flight, four times what the latency-bandwidth product asks for.
// Four consumer warps take 16 slots each for the scores, tell each other their
// maxima, and put the numerators in shared memory; then each takes a quarter of
// the columns of V over all 64 slots. So a segment ends without joining sums
// across warps, and short sequences cost little more than their loads (with a
// running maximum and sums of its own for each warp, joined at the end of every
// segment, a batch of 64 sequences of 0 to 16383 slots took 256 us). That batch,
// 8 KV heads of 128 in bf16, 632 MB: 104 us, 6.1 TB/s; one sequence of 2048
// slots, a tile per CTA: 6.2 us, all latency.
//
// Slots that no row sees are masked by selection, and their values are
// replaced by zeros in shared memory, whatever the pages hold. A non-finite
// value that only some of the rows see is replaced as well and added, to the
// rows that see it, at the end: its product with any positive weight is the
// value itself.
#include <algorithm>
#include <cmath>

#include "kvf_paged_tc.cuh"

namespace kvf {
namespace {

constexpr int kRows = kDecodeRows, kKeys = kDecodeKeys;
constexpr int kWarps = 4;
constexpr int kThreads = 32 * (kWarps + 1);
template <int DP>
constexpr int stages() { return DP == 128 ? 3 : 6; }
template <int DP>
constexpr int tile_bytes() { return kKeys * DP * 2; }
// a segment as the producer hands it to the consumers
struct Head {
  int seq, head, row0, it0, it1, part, n, nq, q0;
};
constexpr int kPStride = kKeys + 8;  // numerators of a row, 16-bit: eight rows apart lie in different banks
template <int DP>
struct Shared {
  uint16_t q[2][kRows * DP];  // rows of two segments, 16-byte chunks permuted by the row
  uint16_t p[kRows * kPStride];
  float m[kWarps][kRows];
  float l[kWarps][kRows];
  Head head[2];
  uint64_t bars[2 * stages<DP>() + 4];
  // whether a segment's tiles held non-finite values (by the segment's parity:
  // the other one is cleared meanwhile); whether a consumer gave up waiting for
  // the segment's rows or for a tile: each is read between the barrier behind
  // its wait and the next one, so all four stop together
  int bad[2], stop_rows, stop, abort;
};
template <int DP>
constexpr size_t smem_bytes() {
  return 1024 + (size_t)stages<DP>() * 2 * tile_bytes<DP>() + sizeof(Shared<DP>);
}

__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
using ptx::ex2;
using ptx::pack2;

// byte offset of 16-byte chunk `chunk` (8 columns) of slot `row` in a tile:
// halves of 64 columns, 128 bytes a row, chunks permuted by the row
__device__ __forceinline__ uint32_t tile_off(int row, int chunk) {
  return (uint32_t)((chunk >> 3) * (kKeys * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// the sum of the non-finite values of one column that the query at slot pos
// sees in 16-slot groups that not every row of the segment sees whole (v: the
// column in the pool's first row)
template <typename T>
__device__ __noinline__ float nonfinite_sum(const T* v, const int* table, int shift, int heads, int head, int dim,
                                            int it0, int it1, PagedSpan span, int pa, int pb, int pos, int window,
                                            int sinks) {
  float sum = 0.0f;
  for (int it = it0; it < it1; ++it) {
    const int t0 = (it < span.nsink ? it : span.first + it - span.nsink) * kKeys;
    for (int j = t0; j < t0 + kKeys && j <= pos; ++j) {
      const int b0 = j & ~15;
      if ((b0 + 15 <= pa && (!window || b0 > pb - window || b0 + 16 <= sinks)) || !paged_sees(pos, j, window, sinks))
        continue;
      const size_t row = (((size_t)__ldg(table + (j >> shift)) * heads + head) << shift) + (j & ((1 << shift) - 1));
      const float y = to_float<T>(v[row * dim]);
      if (!isfinite(y)) sum += y;
    }
  }
  return sum;
}

// scores != nullptr: every score (base 2, -inf where unseen) is also written,
// for the attention weights: sequence i's at scores + score_at[i], [head][row][slot],
// rows of a multiple of four slots
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 2)
    k_paged_decode(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, PagedAttn a,
                   const PagedSeg* __restrict__ segs, const int* __restrict__ first, float* __restrict__ scores,
                   const long long* __restrict__ score_at, bool wide_q) {
  constexpr int kStages = stages<DP>(), kTile = tile_bytes<DP>(), kSteps = DP / 16;
  constexpr int kCols = DP / (8 * kWarps);  // 8-wide column tiles of a warp
  extern __shared__ uint8_t sm_raw[];
  // the 128-byte swizzle takes its pattern from address bits 7-9
  uint8_t* sm = sm_raw + ((1024u - (ptx::smem(sm_raw) & 1023u)) & 1023u);
  Shared<DP>& sh = *reinterpret_cast<Shared<DP>*>(sm + (size_t)kStages * 2 * kTile);
  volatile int* abort_flag = &sh.abort;
  const int tid = threadIdx.x, w = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t full = ptx::smem(sh.bars), empty = full + 8 * kStages, q_full = empty + 8 * kStages,
                 q_empty = q_full + 16;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(full + 8 * i, 1);
      ptx::mbar_init(empty + 8 * i, kWarps);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(q_full + 8 * i, 1);
      ptx::mbar_init(q_empty + 8 * i, kWarps);
    }
    sh.abort = sh.stop_rows = sh.stop = sh.bad[0] = sh.bad[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  const int seg0 = __ldg(first + blockIdx.x), seg1 = __ldg(first + blockIdx.x + 1);
  bool gave_up = false;

  if (w == kWarps) {
    // ---------------- producer: one lane per box of a tile ----------------
    const int box = min(kKeys, 1 << a.c.page_shift);  // slots of one load
    int n_tile = 0;
    auto describe = [&](int si) {
      Head d{};
      if (si < seg1) {
        const PagedSeg g = segs[si];
        const int q0 = __ldg(a.s.q_start + g.seq);
        d = {g.seq, g.head, g.row0, g.it0, g.it1, g.part, __ldg(a.s.kv_len + g.seq),
             __ldg(a.s.q_start + g.seq + 1) - q0, q0};
      }
      return d;
    };
    Head next = describe(seg0);
    for (int si = seg0; si < seg1 && !gave_up; ++si) {
      const Head g = next;
      next = describe(si + 1);  // in flight while this segment is loaded
      const int nth = si - seg0, qb = nth & 1;
      if (nth >= 2 && !ptx::mbar_wait(q_empty + 8 * qb, ((nth >> 1) - 1) & 1, abort_flag)) gave_up = true;
      if (__any_sync(0xffffffffu, gave_up)) {
        gave_up = true;
        break;
      }
      const int* table = a.s.table + (size_t)g.seq * a.s.stride;
      const PagedSpan span = paged_span(g.row0, kRows, a.group, g.n, g.nq, a.window, a.sinks, kKeys);
      auto load = [&](int it) {
        const int j0 = (it < span.nsink ? it : span.first + it - span.nsink) * kKeys;
        const int j = j0 + lane * box;
        const bool mine = lane * box < kKeys && j < g.n;
        const int page = mine ? __ldg(table + (j >> a.c.page_shift)) : 0;
        const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
        const int s = n_tile % kStages, round = n_tile / kStages;
        if (round > 0 && !ptx::mbar_wait(empty + 8 * s, (round - 1) & 1, abort_flag)) gave_up = true;
        if (__any_sync(0xffffffffu, gave_up)) {
          gave_up = true;
          return;
        }
        if (lane == 0) ptx::mbar_expect(full + 8 * s, (uint32_t)(boxes * 2 * box * DP * 2));
        __syncwarp();
        if (mine) {
          const uint32_t dst = ptx::smem(sm) + (uint32_t)(s * 2 * kTile + lane * box * 128);
          const int y = j & ((1 << a.c.page_shift) - 1), z = page * a.c.heads + g.head;
#pragma unroll
          for (int half = 0; half < DP / 64; ++half) {
            ptx::load_box(dst + half * (kKeys * 128), &kmap, 64 * half, y, z, full + 8 * s);
            ptx::load_box(dst + kTile + half * (kKeys * 128), &vmap, 64 * half, y, z, full + 8 * s);
          }
        }
        ++n_tile;
      };
      if (g.it0 < g.it1) load(g.it0);  // ahead of the rows: it takes longer
      // the segment's rows, rows and columns that are not there as zeros
      const int rows = min(kRows, g.nq * a.group - g.row0);
#pragma unroll 4
      for (int i = lane; i < kRows * (DP / 8); i += 32) {
        const int r = i / (DP / 8), ch = i - r * (DP / 8);
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < rows && 8 * ch < a.c.dim) {
          const int t = (g.row0 + r) / a.group, hq = g.head * a.group + (g.row0 + r) % a.group;
          const uint16_t* p =
              static_cast<const uint16_t*>(a.q) + (size_t)(g.q0 + t) * a.q_token + (size_t)hq * a.q_head + 8 * ch;
          if (wide_q) x = __ldg(reinterpret_cast<const uint4*>(p));
          else
            x = make_uint4(__ldg(p) | ((uint32_t)__ldg(p + 1) << 16), __ldg(p + 2) | ((uint32_t)__ldg(p + 3) << 16),
                           __ldg(p + 4) | ((uint32_t)__ldg(p + 5) << 16), __ldg(p + 6) | ((uint32_t)__ldg(p + 7) << 16));
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(sh.q[qb]) + r * (DP * 2) + ((ch ^ (r & 7)) << 4)) = x;
      }
      if (lane == 0) sh.head[qb] = g;
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(q_full + 8 * qb);
      for (int it = g.it0 + 1; it < g.it1 && !gave_up; ++it) load(it);
    }
    // after a timeout the loads in flight still land in this CTA's memory
    if (gave_up) {
      *abort_flag = 1;
      for (int t = max(0, n_tile - kStages); t < n_tile; ++t)
        mbar_wait_bounded(full + 8 * (t % kStages), (t / kStages) & 1, kWaitNs);
    }
  } else {
    // ---------------- consumers ----------------
    const int r0 = lane >> 2, c0 = (lane & 3) * 2;  // rows r0, r0 + 8; columns c0, c0 + 1 of an 8-wide tile
    const int Hq = a.c.heads * a.group, D = a.c.dim;
    int s = 0;
    uint32_t s_phase = 0;
    for (int si = seg0; si < seg1; ++si) {
      const int nth = si - seg0, qb = nth & 1;
      if (!ptx::mbar_wait(q_full + 8 * qb, (nth >> 1) & 1, abort_flag)) gave_up = true;
      if (__any_sync(0xffffffffu, gave_up)) {
        gave_up = true;
        *abort_flag = 1;
        sh.stop_rows = 1;
      }
      const Head g = sh.head[qb];
      uint32_t qf[kSteps][4];
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        // matrices: rows 0-7 and 8-15 of columns 0-7, then of columns 8-15
        const int r = lane & 15, ch = 2 * k + (lane >> 4);
        ldsm4(ptx::smem(sh.q[qb]) + r * (DP * 2) + ((ch ^ (r & 7)) << 4), qf[k]);
      }
      consumer_sync();  // also: the last segment's maxima and sums are read
      if (sh.stop_rows) break;
      if (tid == 0) sh.bad[(si + 1) & 1] = 0;
      if (lane == 0) ptx::mbar_arrive(q_empty + 8 * qb);
      const int rows = min(kRows, g.nq * a.group - g.row0);
      const PagedSpan span = paged_span(g.row0, kRows, a.group, g.n, g.nq, a.window, a.sinks, kKeys);
      int pos[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) pos[i] = g.n - g.nq + (g.row0 + r0 + 8 * i) / a.group;
      const int pa = g.n - g.nq + g.row0 / a.group, pb = g.n - g.nq + (g.row0 + rows - 1) / a.group;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[kCols][4];
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[c][e] = 0.0f;
      const size_t sc_row = (size_t)((g.n + 3) & ~3);
      float* sc = scores ? scores + score_at[g.seq] + ((size_t)g.head * g.nq * a.group + g.row0) * sc_row : nullptr;
      bool stop = false;

      for (int it = g.it0; it < g.it1; ++it) {
        const int j0 = (it < span.nsink ? it : span.first + it - span.nsink) * kKeys + 16 * w;  // this warp's slots
        const uint32_t kt = ptx::smem(sm) + (uint32_t)(s * 2 * kTile), vt = kt + kTile;
        if (!ptx::mbar_wait(full + 8 * s, s_phase, abort_flag)) gave_up = true;
        if (__any_sync(0xffffffffu, gave_up)) {  // all four stop at the next barrier
          gave_up = true;
          *abort_flag = 1;
          sh.stop = 1;
        }
        float x[2][4] = {};
        {
          const int row = 16 * w + ((lane >> 4) << 3) + (lane & 7), odd = (lane >> 3) & 1;
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            uint32_t b[4];
            ldsm4(kt + tile_off(row, 2 * k + odd), b);
            mma16816<T>(x[0], qf[k], b[0], b[1]);
            mma16816<T>(x[1], qf[k], b[2], b[3]);
          }
        }
        // slots that every row sees need no masks
        const bool whole = j0 + 15 <= pa && (!a.window || j0 > pb - a.window || j0 + 16 <= a.sinks);
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[t][e] *= a.scale2;
            if (!whole && !paged_sees(pos[e >> 1], j0 + 8 * t + c0 + (e & 1), a.window, a.sinks)) x[t][e] = -INFINITY;
            mx[e >> 1] = fmaxf(mx[e >> 1], x[t][e]);
          }
        if (sc) {  // pairs of slots: a row's padding takes the one past its end
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int r = r0 + 8 * i, j = j0 + 8 * t + c0;
              if (r < rows && j < g.n)
                *reinterpret_cast<float2*>(sc + r * sc_row + j) = make_float2(x[t][2 * i], x[t][2 * i + 1]);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
          mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
          if ((lane & 3) == 0) sh.m[w][r0 + 8 * i] = mx[i];
        }
        if (!whole) {  // this warp's 16 rows of V, two lanes a row
          const int row = lane >> 1, j = j0 + row;
          const bool any = j <= pb && (!a.window || j > pa - a.window || j < a.sinks);
          bool bad = false;
#pragma unroll 1
          for (int c = lane & 1; c < DP / 8; c += 2) {
            uint4* q = reinterpret_cast<uint4*>(sm + (size_t)s * 2 * kTile + kTile + tile_off(16 * w + row, c));
            if (!any) *q = make_uint4(0, 0, 0, 0);
            else {
              uint4 v = *q;
              if (drop_nonfinite<T>(v)) {
                *q = v;
                bad = true;
              }
            }
          }
          if (bad) sh.bad[si & 1] = 1;
          // the stage's next tile is written by tensor-map loads: behind these stores
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        consumer_sync();  // the maxima are there
        if (sh.stop) {
          stop = true;
          break;
        }
        float f[2], mu[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float M = m[i];
#pragma unroll
          for (int k = 0; k < kWarps; ++k) M = fmaxf(M, sh.m[k][r0 + 8 * i]);
          mu[i] = M == -INFINITY ? 0.0f : M;
          f[i] = ex2(m[i] - mu[i]);
          l[i] *= f[i];
          m[i] = M;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[t][e] = ex2(x[t][e] - mu[e >> 1]);
            l[e >> 1] += x[t][e];
          }
          // the numerators are rounded to the cache's type for the product with
          // the values; the sum keeps them in f32
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *reinterpret_cast<uint32_t*>(&sh.p[(r0 + 8 * i) * kPStride + 16 * w + 8 * t + c0]) =
                pack2<T>(x[t][2 * i], x[t][2 * i + 1]);
        }
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          o[c][0] *= f[0];
          o[c][1] *= f[0];
          o[c][2] *= f[1];
          o[c][3] *= f[1];
        }
        consumer_sync();  // the numerators (and V, put right) are there
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k) {
          uint32_t pf[4];
          ldsm4(ptx::smem(sh.p) + ((lane & 15) * kPStride + 16 * k + 8 * (lane >> 4)) * 2, pf);
#pragma unroll
          for (int c = 0; c < kCols; c += 2) {
            uint32_t b[4];
            ldsm4t(vt + tile_off(16 * k + (lane & 15), kCols * w + c + (lane >> 4)), b);
            mma16816<T>(o[c], pf, b[0], b[1]);
            mma16816<T>(o[c + 1], pf, b[2], b[3]);
          }
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(empty + 8 * s);
        if (++s == kStages) {
          s = 0;
          s_phase ^= 1u;
        }
      }
      if (stop) break;
      // every warp knows the rows' maxima; their sums are added up
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if ((lane & 3) == 0) sh.l[w][r0 + 8 * i] = l[i];
      }
      consumer_sync();
      const bool bad = sh.bad[si & 1] != 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = r0 + 8 * i;
        if (r >= rows) continue;
        float L = sh.l[0][r];
#pragma unroll
        for (int k = 1; k < kWarps; ++k) L += sh.l[k][r];
        const int t = (g.row0 + r) / a.group, hq = g.head * a.group + (g.row0 + r) % a.group;
        const size_t at = (size_t)(g.q0 + t) * Hq + hq;
        const bool none = L == 0.0f;
        const float inv = none ? 0.0f : 1.0f / L;
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int col = 8 * (kCols * w + c) + c0 + e;
            if (col >= D) continue;
            float v = o[c][2 * i + e];
            if (bad)
              v += nonfinite_sum<T>(static_cast<const T*>(a.c.values) + col, a.s.table + (size_t)g.seq * a.s.stride,
                                    a.c.page_shift, a.c.heads, g.head, D, g.it0, g.it1, span, pa, pb, g.n - g.nq + t,
                                    a.window, a.sinks);
            if (g.part >= 0) a.part_o[((size_t)g.part * kRows + r) * D + col] = v;
            else static_cast<T*>(a.out)[at * D + col] = from_float<T>(none ? 0.0f : v * inv);
          }
        if (w == 0 && (lane & 3) == 0) {
          if (g.part >= 0)
            *reinterpret_cast<float2*>(a.part_ml + ((size_t)g.part * kRows + r) * 2) = make_float2(m[i], L);
          else if (a.lse)
            a.lse[at] = none ? -INFINITY : (m[i] + log2f(L)) * (float)M_LN2;
        }
      }
    }
  }
  if (gave_up && a.status) atomicOr(a.status, kDevErrTimeout);
}

// Attention weights from the scores that k_paged_decode wrote: a thread adds
// four slots' rows in order, 64 threads a (tile, head), the loads of eight rows
// in flight. Bound by reading the scores, mostly from L2 (10.6 us for 16
// sequences of 3000 to 16000 slots with 64 query heads; 22 with a slot per thread).
// The scores may still be written while this kernel starts: ordinary loads behind
// the wait, never the read-only path.
constexpr int kWeightThreads = 256;
constexpr int kWeightHeads = kWeightThreads * 4 / kDecodeWeightSlots;
__global__ void __launch_bounds__(kWeightThreads) k_paged_decode_weights(PagedAttn a, const PagedSlots* __restrict__ tiles,
                                                                         const float* scores,
                                                                         const long long* __restrict__ score_at,
                                                                         float decay) {
  __shared__ float lse2[kWeightHeads][kRows];
  const PagedSlots g = tiles[blockIdx.x];
  const int n = __ldg(a.s.kv_len + g.seq), q0 = __ldg(a.s.q_start + g.seq);
  const int nq = __ldg(a.s.q_start + g.seq + 1) - q0, rows = nq * a.group;
  const int hs = threadIdx.x / (kDecodeWeightSlots / 4), h = blockIdx.y * kWeightHeads + hs;
  const int j = g.slot0 + 4 * (threadIdx.x % (kDecodeWeightSlots / 4));
  // tiles that no row visits were not written
  const PagedSpan span = paged_span(0, kRows, a.group, n, nq, a.window, a.sinks, kKeys);
  const int tile = j / kKeys;
  const bool there = tile < span.nsink || (tile >= span.first && tile < span.first + span.count - span.nsink);
  const size_t sc_row = (size_t)((n + 3) & ~3);
  const float* sc = scores + score_at[g.seq] + (size_t)h * rows * sc_row + j;
  wait_for_previous();
  if ((int)threadIdx.x < kWeightHeads * kRows) {
    const int r = threadIdx.x % kRows, hl = blockIdx.y * kWeightHeads + threadIdx.x / kRows;
    float z = INFINITY;  // a row that is not there, or sees nothing, adds 0
    if (r < rows && hl < a.c.heads) {
      z = a.lse[(size_t)(q0 + r / a.group) * (a.c.heads * a.group) + hl * a.group + r % a.group] * (float)M_LOG2E;
      if (z == -INFINITY) z = INFINITY;
    }
    lse2[threadIdx.x / kRows][r] = z;
  }
  __syncthreads();
  if (h >= a.c.heads || j >= n) return;
  float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (there) {
#pragma unroll
    for (int r0 = 0; r0 < kRows; r0 += 8) {
      if (r0 >= rows) break;
      float4 x[8];
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r0 + r < rows) x[r] = *reinterpret_cast<const float4*>(sc + (r0 + r) * sc_row);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (r0 + r >= rows) continue;
        const float z = lse2[hs][r0 + r];
        if (z != z) {  // a NaN row: NaN for the slots that it sees, nothing for the others
          const int pos = n - nq + (r0 + r) / a.group;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (paged_sees(pos, j + e, a.window, a.sinks)) t[e] = z;
          continue;
        }
        t[0] += exp2f(x[r].x - z);
        t[1] += exp2f(x[r].y - z);
        t[2] += exp2f(x[r].z - z);
        t[3] += exp2f(x[r].w - z);
      }
    }
  }
  // four slots lie in one page
  const int page = __ldg(a.s.table + (size_t)g.seq * a.s.stride + (j >> a.c.page_shift));
  float* p = a.c.weights + (((size_t)page * a.c.heads + h) << a.c.page_shift) + (j & ((1 << a.c.page_shift) - 1));
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (j + e < n) p[e] = decay == 0.0f ? t[e] : fmaf(decay, p[e], t[e]);
}

template <typename T, int DP>
cudaError_t launch_typed(const CUtensorMap& km, const CUtensorMap& vm, const PagedAttn& a, const PagedWork& w,
                         float* scores, const long long* score_at, cudaStream_t st) {
  auto kern = k_paged_decode<T, DP>;
  constexpr size_t smem = smem_bytes<DP>();
  static OptInOnce done;
  cudaError_t e = opt_in_once(done, kern, smem);
  if (e != cudaSuccess) return e;
  const bool wide_q = (a.q_token | a.q_head) % 8 == 0 && aligned(a.q, 16);
  kern<<<w.ctas, kThreads, smem, st>>>(km, vm, a, w.segs, w.first, scores, score_at, wide_q);
  note_launches(1);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_decode(const PagedAttn& a, const PagedWork& w, float* scores, const long long* score_at,
                                cudaStream_t st) {
  if (w.ctas == 0) return cudaSuccess;
  CUtensorMap km, vm;
  const int rows = std::min(kKeys, 1 << a.c.page_shift);
  if (!paged_map(&km, a.c, a.c.keys, rows) || !paged_map(&vm, a.c, a.c.values, rows)) return cudaErrorInvalidValue;
  if (a.c.dtype == KVF_IN_F16)
    return a.c.dim <= 64 ? launch_typed<__half, 64>(km, vm, a, w, scores, score_at, st)
                         : launch_typed<__half, 128>(km, vm, a, w, scores, score_at, st);
  return a.c.dim <= 64 ? launch_typed<__nv_bfloat16, 64>(km, vm, a, w, scores, score_at, st)
                       : launch_typed<__nv_bfloat16, 128>(km, vm, a, w, scores, score_at, st);
}

cudaError_t launch_paged_decode_weights(const PagedAttn& a, const PagedSlots* tiles, size_t ntiles,
                                        const float* scores, const long long* score_at, float decay, cudaStream_t st) {
  if (ntiles == 0) return cudaSuccess;
  note_launches(1);
  return launch_behind(k_paged_decode_weights, dim3((unsigned)ntiles, (unsigned)((a.c.heads + kWeightHeads - 1) / kWeightHeads)), kWeightThreads, 0, st, a,
                       tiles, scores, score_at, decay);
}

}  // namespace kvf
