// Attention weights of cached slots for chunks of new tokens, on tcgen05:
//   w_j = sum over the rows i that see j of 2^(scale2 q_i.k_j - lse2_i),
// the column sums of the softmax, whose row sums are known from the attention.
//
// A segment owns 256 slots of one (sequence, KV head) and walks tiles of the
// rows that may see them. The scores are made transposed, S = K Q^T, so that a
// slot is a TMEM lane and a thread adds the terms of one slot in a fixed
// order: no atomics and no reduction across threads. K stays in shared memory
// for the segment; per row tile and SM the products take 1024 cycles and the
// 32768 exponentials 2048, which bound the kernel. The row tiles are divided
// over the SMs in equal shares; the parts of a slot are added, in order, and
// joined with the old weight by a second small kernel.
//   warps 0-7, 8-15: the sums of the first and the second 128 slots, four warps
//     for one half of a tile's rows and four for the other (two warps per
//     scheduler left the exponential unit half idle: 238 instead of 165 us for two
//     1000-token chunks on 7000 slots)
//   warp 16: tensor-map loads of K (a box per page; the next segment's while
//     this one runs) and of the rows (group heads by 128 / group tokens)
//   warp 17: the MMAs, issued by one thread; two TMEM buffers per 128 slots
//   warps 18, 19: lse of the tile's rows, +inf for rows that see nothing and
//     for padding, whose terms so become 0
// Every wait is bounded; one that runs out ends all roles and sets kDevErrTimeout.
#include <algorithm>
#include <cmath>

#include "kvf_paged_tc.cuh"

namespace kvf {

void paged_split_slots(const int* q_lens, const int* kv_lens, size_t n, int heads, int group, int window, int sinks,
                       long long more_than, int slots, PagedWorkHost* out) {
  const int TQ = 128 / group;
  out->row_tile = kWeightSlots;
  out->key_tile = TQ;
  out->first.assign(1, 0);
  // row tiles that may see slots j0..j1-1
  auto range = [&](size_t i, int j0, int* t0, int* t1) {
    const int nq = q_lens[i], old = kv_lens[i] - nq;
    const int j1 = std::min(j0 + kWeightSlots, kv_lens[i]);
    const long long ta = std::max(0, j0 - old);
    long long tb = nq;
    if (window && j0 >= sinks) tb = std::min<long long>(nq, (long long)j1 - 1 + window - old);
    *t0 = (int)(ta / TQ);
    *t1 = tb > ta ? (int)((tb + TQ - 1) / TQ) : *t0;
  };
  auto chosen = [&](size_t i) { return (long long)q_lens[i] * group > more_than; };
  constexpr int kFixed = 2;  // what a segment's start and end cost, in row tiles
  long long cost = 0;
  for (size_t i = 0; i < n; ++i)
    if (chosen(i))
      for (int j = 0; j < kv_lens[i]; j += kWeightSlots) {
        int t0, t1;
        range(i, j, &t0, &t1);
        if (t1 > t0) cost += (long long)heads * (t1 - t0 + kFixed);
      }
  long long quota = std::max<long long>((cost + slots - 1) / slots, 4 + kFixed);
  // CTAs that close early may push their count past `slots`, and one CTA more
  // than the SMs hold costs a whole wave: then with a larger quota
  for (int attempt = 0;; ++attempt) {
    out->segs.clear();
    out->joins.clear();
    out->first.assign(1, 0);
    out->parts = 0;
    long long left = quota;
    auto close = [&] {
      if ((int)out->segs.size() > out->first.back()) out->first.push_back((int)out->segs.size());
      left = quota;
    };
    for (size_t i = 0; i < n; ++i) {
      if (!chosen(i)) continue;
      for (int h = 0; h < heads; ++h)
        for (int j = 0; j < kv_lens[i]; j += kWeightSlots) {
          int t0, t1;
          range(i, j, &t0, &t1);
          const int part0 = out->parts;
          while (t0 < t1) {
            if (left - kFixed < std::min(4, t1 - t0) && left < quota) close();
            int take = (int)std::min<long long>(t1 - t0, std::max<long long>(left - kFixed, 1));
            if (t1 - t0 - take < 4) take = t1 - t0;
            out->segs.push_back({(int)i, h, j, t0, t0 + take, out->parts++});
            t0 += take;
            left -= take + kFixed;
            if (left <= kFixed) close();
          }
          out->joins.push_back({(int)i, h, j, part0, out->parts - part0, 0, 0});
        }
    }
    close();
    if ((int)out->first.size() - 1 <= slots || attempt == 16) return;
    quota += std::max<long long>(1, quota / 32);
  }
}

namespace {

using namespace ptx;

constexpr int kSumWarps = 16;
constexpr int kThreads = 32 * (kSumWarps + 4);
template <int DP>
constexpr int tile_bytes() { return kTile * DP * 2; }
template <int DP>
constexpr int stages() { return DP == 128 ? 3 : 6; }
template <int DP>
constexpr size_t smem_bytes() { return 1024 + (size_t)(4 + stages<DP>()) * tile_bytes<DP>(); }
static_assert(2 * (smem_bytes<64>() + 1024) > 228 * 1024, "one CTA per SM keeps the TMEM allocation non-blocking");

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    k_paged_chunk_weights(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap qmap,
                          PagedAttn a, const PagedSeg* __restrict__ segs, const int* __restrict__ first,
                          float* __restrict__ part_w) {
  constexpr int kStages = stages<DP>(), kBytes = tile_bytes<DP>();
  extern __shared__ uint8_t sm_raw[];
  uint8_t* sm = sm_raw + ((1024u - (smem(sm_raw) & 1023u)) & 1023u);
  uint8_t* ks = sm;                // [2 segments][2 tiles]
  uint8_t* qs = sm + 4 * kBytes;   // [kStages]
  __shared__ __align__(16) float lse2[kStages][kTile];
  __shared__ uint64_t bars[2 * kStages + 4 + 8 + 1];
  __shared__ uint32_t sh_tmem;
  __shared__ int sh_abort;
  volatile int* abort_flag = &sh_abort;
  const uint32_t q_full = smem(bars), q_empty = q_full + 8 * kStages, k_full = q_empty + 8 * kStages,
                 k_empty = k_full + 16, s_full = k_empty + 16, s_empty = s_full + 32, drained = s_empty + 32;
  const int tid = threadIdx.x, w = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int TQ = kTile / a.group, cols = TQ * a.group;  // tokens and rows of a row tile

  if (w == kSumWarps + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem(&sh_tmem)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(q_full + 8 * i, 3);               // the load and warps 18 and 19
      mbar_init(q_empty + 8 * i, 1 + kSumWarps);  // the MMAs' completion and the summing warps
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + 8 * i, 1);
      mbar_init(k_empty + 8 * i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(s_empty + 8 * i, kSumWarps / 2);
    }
    mbar_init(drained, 1);
    sh_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (cols < kTile) {  // rows that no load writes: their products must be finite
    for (int i = tid; i < kStages * kBytes / 16; i += kThreads) reinterpret_cast<uint4*>(qs)[i] = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  constexpr uint32_t tmem = 0;  // all columns are this CTA's, so they start at 0
  const int seg0 = __ldg(first + blockIdx.x), seg1 = __ldg(first + blockIdx.x + 1);
  bool gave_up = false;
  wait_for_previous();  // lse

  if (w == kSumWarps) {
    // ---------------- loads ----------------
    const int page = 1 << a.c.page_shift, box = min(kTile, page);
    int n = 0;
    for (int si = seg0; si < seg1 && !gave_up; ++si) {
      const PagedSeg g = segs[si];
      const int kv = __ldg(a.s.kv_len + g.seq), q0 = __ldg(a.s.q_start + g.seq);
      const int* table = a.s.table + (size_t)g.seq * a.s.stride;
      const int nth = si - seg0, kb = nth & 1;
      if (nth >= 2 && !mbar_wait(k_empty + 8 * kb, ((nth >> 1) - 1) & 1, abort_flag)) gave_up = true;
      if (__any_sync(0xffffffffu, gave_up)) {
        gave_up = true;
        break;
      }
      const int j = g.row0 + lane * box;  // a box per lane: at most 16
      const bool mine = lane * box < kWeightSlots && j < kv;
      const int p = mine ? __ldg(table + (j >> a.c.page_shift)) : 0;
      const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
      if (lane == 0) mbar_expect(k_full + 8 * kb, (uint32_t)(boxes * box * DP * 2));
      __syncwarp();
      if (mine) {
        const int at = lane * box;  // slot in the segment
        const uint32_t dst = smem(ks) + (uint32_t)((2 * kb + at / kTile) * kBytes + (at % kTile) * 128);
#pragma unroll
        for (int half = 0; half < DP / 64; ++half)
          load_box(dst + half * kHalf, &kmap, 64 * half, j & (page - 1), p * a.c.heads + g.head, k_full + 8 * kb);
      }
      for (int it = g.it0; it < g.it1; ++it, ++n) {
        const int st = n % kStages, round = n / kStages;
        if (round > 0 && !mbar_wait(q_empty + 8 * st, (round - 1) & 1, abort_flag)) gave_up = true;
        if (__any_sync(0xffffffffu, gave_up)) {
          gave_up = true;
          break;
        }
        if (lane == 0) {
          mbar_expect(q_full + 8 * st, (uint32_t)(cols * DP * 2));
#pragma unroll
          for (int half = 0; half < DP / 64; ++half)
            load_box(smem(qs) + (uint32_t)(st * kBytes + half * kHalf), &qmap, 64 * half, g.head * a.group,
                     q0 + it * TQ, q_full + 8 * st);
        }
        __syncwarp();
      }
    }
    if (gave_up) *abort_flag = 1;
  } else if (w == kSumWarps + 1) {
    // ---------------- MMAs ----------------
    const bool lead = lane == 0;
    const uint32_t kd = desc_k(smem(ks)), qd = desc_k(smem(qs));
    int n = 0, st = 0;
    uint32_t st_phase = 0;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (!mbar_wait(bar, parity, abort_flag)) gave_up = true;
      if (__any_sync(0xffffffffu, gave_up)) gave_up = true;
      return !gave_up;
    };
    for (int si = uniform(seg0); si < uniform(seg1) && !gave_up; ++si) {
      const int count = uniform(segs[si].it1 - segs[si].it0);
      const int nth = si - uniform(seg0), kb = nth & 1;
      if (!wait(k_full + 8 * kb, (nth >> 1) & 1)) break;
      for (int it = 0; it < count; ++it, ++n) {
        const int buf = n & 1;
        if (!wait(q_full + 8 * st, st_phase)) break;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          const int b = 2 * kt + buf;
          if (n >= 2 && !gave_up) wait(s_empty + 8 * b, ((n >> 1) - 1) & 1);
          if (gave_up) continue;
          fence_after();
          const uint32_t k = kd + (2 * kb + kt) * (kBytes >> 4), q = qd + st * (kBytes >> 4);
#pragma unroll
          for (int d = 0; d < DP / 16; ++d) {
            const uint32_t off = ((d >> 2) * kHalf + (d & 3) * 32) >> 4;
            mma_ss(lead, tmem + b * 128, k + off, q + off, idesc<T>(kTile, false), d > 0);
          }
          commit(lead, s_full + 8 * b);
        }
        if (gave_up) break;
        commit(lead, q_empty + 8 * st);
        if (++st == kStages) {
          st = 0;
          st_phase ^= 1u;
        }
      }
      if (!gave_up) commit(lead, k_empty + 8 * kb);
    }
    if (gave_up) {  // the MMAs in flight still use this CTA's memory
      *abort_flag = 1;
      commit(lead, drained);
      mbar_wait_bounded(drained, 0, kWaitNs);
    }
  } else if (w > kSumWarps + 1) {
    // ---------------- lse of the rows ----------------
    const int c0 = (w - kSumWarps - 2) * 32 + lane;  // columns c0 and c0 + 64
    const int Hq = a.c.heads * a.group;
    int n = 0;
    for (int si = seg0; si < seg1 && !gave_up; ++si) {
      const PagedSeg g = segs[si];
      const int q0 = __ldg(a.s.q_start + g.seq), nq = __ldg(a.s.q_start + g.seq + 1) - q0;
      for (int it = g.it0; it < g.it1; ++it, ++n) {
        const int st = n % kStages, round = n / kStages;
        float z[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int c = c0 + 64 * u, t = it * TQ + c / a.group;
          z[u] = -INFINITY;
          if (c < cols && t < nq)
            z[u] = a.lse[(size_t)(q0 + t) * Hq + g.head * a.group + c % a.group] * (float)M_LOG2E;
          if (z[u] == -INFINITY) z[u] = INFINITY;
        }
        if (round > 0 && !mbar_wait(q_empty + 8 * st, (round - 1) & 1, abort_flag)) gave_up = true;
        if (__any_sync(0xffffffffu, gave_up)) {
          gave_up = true;
          break;
        }
        lse2[st][c0] = z[0];
        lse2[st][c0 + 64] = z[1];
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full + 8 * st);
      }
    }
    if (gave_up) *abort_flag = 1;
  } else {
    // ---------------- sums ----------------
    const int kt = w >> 3, half = (w >> 2) & 1, t = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (w & 3)) << 16;
    int n = 0, st = 0;
    for (int si = seg0; si < seg1 && !gave_up; ++si) {
      const PagedSeg g = segs[si];
      const int kv = __ldg(a.s.kv_len + g.seq);
      const int nq = __ldg(a.s.q_start + g.seq + 1) - __ldg(a.s.q_start + g.seq);
      const int jt = g.row0 + kt * kTile, j = jt + t;
      float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
      const float2 c2 = make_float2(a.scale2, a.scale2);
      for (int it = g.it0; it < g.it1; ++it, ++n) {
        const int b = 2 * kt + (n & 1);
        if (!mbar_wait(s_full + 8 * b, (n >> 1) & 1, abort_flag)) gave_up = true;
        if (__any_sync(0xffffffffu, gave_up)) {
          gave_up = true;
          break;
        }
        fence_after();
        // slots of the tile's first and last token; columns lo..hi-1 see slot j
        const int pos0 = kv - nq + it * TQ, pos1 = kv - nq + min(nq, (it + 1) * TQ) - 1;
        const bool whole = jt + kTile - 1 <= pos0 && (it + 1) * TQ <= nq &&
                           (!a.window || jt > pos1 - a.window || jt + kTile <= a.sinks);
        int lo = 0, hi = kTile;
        if (!whole) {
          lo = min(max(j - pos0, 0), kTile) * a.group;
          hi = (pos1 - pos0 + 1) * a.group;
          if (a.window && j >= a.sinks) hi = min(hi, max(0, min(j + a.window - pos0, kTile)) * a.group);
        }
#pragma unroll 1
        for (int q = 64 * half; q < 64 * half + 64; q += 32) {
          float x[32];
          tmem_ld32(tmem + lanes + b * 128 + q, x);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 z = *reinterpret_cast<const float4*>(&lse2[st][q + e]);
            const float2 y0 = ffma2(make_float2(x[e], x[e + 1]), c2, make_float2(-z.x, -z.y));
            const float2 y1 = ffma2(make_float2(x[e + 2], x[e + 3]), c2, make_float2(-z.z, -z.w));
            x[e] = y0.x;
            x[e + 1] = y0.y;
            x[e + 2] = y1.x;
            x[e + 3] = y1.y;
          }
          if (!whole) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (e < lo - q || e >= hi - q) x[e] = -INFINITY;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            sum0 = fadd2(sum0, make_float2(ex2(x[e]), ex2(x[e + 1])));
            sum1 = fadd2(sum1, make_float2(ex2(x[e + 2]), ex2(x[e + 3])));
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(s_empty + 8 * b);
          mbar_arrive(q_empty + 8 * st);
        }
        if (++st == kStages) st = 0;
      }
      if (!gave_up)
        part_w[((size_t)g.part * 2 + half) * kWeightSlots + kt * kTile + t] = (sum0.x + sum0.y) + (sum1.x + sum1.y);
    }
    if (gave_up) *abort_flag = 1;
  }
  if (gave_up && a.status) atomicOr(a.status, kDevErrTimeout);
  fence_before();
  __syncthreads();
  fence_after();
  if (w == kSumWarps && sh_abort && lane < kStages + 2) {
    // after a timeout, the loads in flight still land in this CTA's memory: give
    // them the time of one more bounded wait each (their barriers' phases are
    // not known here, so both are waited for)
    const uint32_t bar = lane < kStages ? q_full + 8 * lane : k_full + 8 * (lane - kStages);
    mbar_wait_bounded(bar, 0, 10000000ull);
    mbar_wait_bounded(bar, 1, 10000000ull);
  }
  if (w == kSumWarps + 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}

// weight = decay * weight + the parts of its slot (written by the kernel before,
// whose end this one overlaps: ordinary loads behind the wait)
__global__ void __launch_bounds__(kWeightSlots) k_paged_chunk_weights_join(PagedAttn a,
                                                                           const PagedJoin* __restrict__ joins,
                                                                           const float* part_w, float decay) {
  const PagedJoin g = joins[blockIdx.x];
  const int j = g.row0 + threadIdx.x;
  const bool there = j < __ldg(a.s.kv_len + g.seq);
  wait_for_previous();
  if (!there) return;
  float t = 0.0f;
#pragma unroll 4
  for (int p = 0; p < 2 * g.parts; ++p) t += part_w[((size_t)2 * g.part0 + p) * kWeightSlots + threadIdx.x];
  const int page = __ldg(a.s.table + (size_t)g.seq * a.s.stride + (j >> a.c.page_shift));
  float* p = a.c.weights + (((size_t)page * a.c.heads + g.head) << a.c.page_shift) + (j & ((1 << a.c.page_shift) - 1));
  *p = decay == 0.0f ? t : fmaf(decay, *p, t);
}

// queries [tokens][heads][dim] as boxes of 64 columns, one KV head's group, and
// as many tokens as make up to 128 rows
bool query_map(CUtensorMap* map, const PagedAttn& a, size_t tokens) {
  auto enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tensor_map_encode_fn());
  if (!enc || !aligned(a.q, 16) || (a.q_token | a.q_head) % 8) return false;
  const cuuint64_t gdim[3] = {(cuuint64_t)a.c.dim, (cuuint64_t)a.c.heads * a.group, (cuuint64_t)tokens};
  const cuuint64_t gstride[2] = {(cuuint64_t)a.q_head * 2, (cuuint64_t)a.q_token * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)(kTile / a.group)};
  const cuuint32_t estride[3] = {1, 1, 1};
  const CUtensorMapDataType dt =
      a.c.dtype == KVF_IN_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return enc(map, dt, 3, const_cast<void*>(a.q), gdim, gstride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP>
cudaError_t launch_typed(const CUtensorMap& km, const CUtensorMap& qm, const PagedAttn& a, const PagedWork& w,
                         float* part_w, cudaStream_t st) {
  auto kern = k_paged_chunk_weights<T, DP>;
  constexpr size_t bytes = smem_bytes<DP>();
  static OptInOnce done;
  cudaError_t e = opt_in_once(done, kern, bytes);
  if (e != cudaSuccess) return e;
  note_launches(1);
  return launch_behind(kern, dim3(w.ctas), kThreads, bytes, st, km, qm, a, w.segs, w.first, part_w);
}

}  // namespace

cudaError_t launch_paged_chunk_weights(const PagedAttn& a, const PagedWork& w, size_t tokens, float* part_w,
                                       float decay, cudaStream_t st) {
  CUtensorMap km, qm;
  if (!query_map(&qm, a, tokens) || !paged_map(&km, a.c, a.c.keys, std::min(kTile, 1 << a.c.page_shift)))
    return cudaErrorNotSupported;
  cudaError_t e = cudaSuccess;
  if (w.ctas) {
    if (a.c.dtype == KVF_IN_F16)
      e = a.c.dim <= 64 ? launch_typed<__half, 64>(km, qm, a, w, part_w, st)
                        : launch_typed<__half, 128>(km, qm, a, w, part_w, st);
    else
      e = a.c.dim <= 64 ? launch_typed<__nv_bfloat16, 64>(km, qm, a, w, part_w, st)
                        : launch_typed<__nv_bfloat16, 128>(km, qm, a, w, part_w, st);
  }
  if (e != cudaSuccess || w.joins_n == 0) return e;
  note_launches(1);
  return launch_behind(k_paged_chunk_weights_join, dim3(w.joins_n), kWeightSlots, 0, st, a, w.joins, part_w, decay);
}

}  // namespace kvf
