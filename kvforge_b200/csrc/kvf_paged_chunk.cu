// Attention of many rows (chunks of new tokens, long drafts) over a paged
// 16-bit cache, on tcgen05.
//
// The formulas are those of kvf_paged_attn.cu. With R rows per (sequence, KV
// head) the two products cost 4 R n D operations and the softmax R n
// exponentials; at D = 128 an SM's tensor core needs 1024 cycles for a tile of
// 128 rows by 128 slots, and its 16 exponentials per cycle need 1024 as well,
// so the kernel is bound by both and must keep them busy at the same time.
//
// One persistent CTA per SM walks segments of (sequence, KV head, 256 rows),
// two row tiles of 128 whose work alternates on the tensor core: while one
// tile's scores go through the softmax, the other tile's products run.
//   warps 0-3, 4-7: softmax of row tile 0 and 1, a row per thread. A tile of
//     scores is read from TMEM, the numerators go back over it in the cache's
//     16-bit type, as the A operand of the second product. The running maximum
//     is followed only when it grows by more than 2^8 (then the sums in TMEM
//     are rescaled): numerators stay below 2^8, which f16 holds, and the
//     rescaling all but vanishes after the first tiles.
//   warp 8: tensor-map loads of K and V tiles, a box per page.
//   warp 9: the MMAs, one thread. S = Q K^T of a tile is issued directly behind
//     the same row tile's O += P V: MMAs run in order, so S may overwrite P, and
//     the barrier that announces S also announces that O is free.
//   warps 10, 11: V tiles that not every row sees whole: slots that no row sees
//     become zeros (their pages may hold anything), non-finite values that only
//     some rows see become zeros and are added to the rows that see them at the
//     end (their product with any positive weight is the value itself).
// TMEM: 2 x 128 columns of scores (numerators over them), 2 x D of sums. Every
// wait is bounded; one that runs out ends all roles and sets kDevErrTimeout.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "kvf_paged_tc.cuh"

namespace kvf {
namespace {

using namespace ptx;

constexpr int kRows = kChunkRows, kKeys = kChunkKeys;
constexpr int kTiles = kRows / kTile;
constexpr int kThreads = 384;
// registers per thread: launched with 168 (65536 / 384), the softmax warps take
// what the others give up: 2 x 128 x 200 + 128 x 104 = 384 x 168
constexpr int kRegsSoftmax = 200, kRegsOther = 104;

template <int DP>
constexpr int tile_bytes() { return kTile * DP * 2; }
template <int DP>
constexpr int stages() { return DP == 128 ? 5 : 10; }
template <int DP>
constexpr size_t smem_bytes() { return 1024 + (size_t)(kTiles + stages<DP>()) * tile_bytes<DP>(); }
// more than half of an SM's shared memory: one CTA per SM, whose TMEM is free
static_assert(2 * (smem_bytes<64>() + 1024) > 228 * 1024 && smem_bytes<128>() + 2048 <= 227 * 1024 + 1024, "one CTA");

// a segment as its roles see it
struct Seg {
  PagedSeg g;
  PagedSpan span;
  int n, nq, q0, rows, pa, pb;
  __device__ __forceinline__ Seg(const PagedAttn& a, const PagedSeg& seg) : g(seg) {
    n = __ldg(a.s.kv_len + g.seq);
    q0 = __ldg(a.s.q_start + g.seq);
    nq = __ldg(a.s.q_start + g.seq + 1) - q0;
    rows = min(kRows, nq * a.group - g.row0);
    span = paged_span(g.row0, kRows, a.group, n, nq, a.window, a.sinks, kKeys);
    pa = n - nq + g.row0 / a.group;
    pb = n - nq + (g.row0 + rows - 1) / a.group;
  }
  __device__ __forceinline__ int slot0(int it) const {
    return (it < span.nsink ? it : span.first + it - span.nsink) * kKeys;
  }
  __device__ __forceinline__ int tiles() const { return rows > kTile ? 2 : 1; }
};
// whether queries at slots pa..pb see all of the tile at j0
__device__ __forceinline__ bool sees_whole(int j0, int pa, int pb, int window, int sinks) {
  return j0 + kKeys - 1 <= pa && (!window || j0 > pb - window || j0 + kKeys <= sinks);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    k_paged_chunk(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, PagedAttn a,
                  const PagedSeg* __restrict__ segs, const int* __restrict__ first, bool wide_q, bool wide_out) {
  constexpr int kStages = stages<DP>(), kBytes = tile_bytes<DP>();
  extern __shared__ uint8_t sm_raw[];
  uint8_t* sm = sm_raw + ((1024u - (smem(sm_raw) & 1023u)) & 1023u);
  uint8_t* ring = sm + kTiles * kBytes;
  __shared__ uint64_t bars[3 * kStages + 4 * kTiles + 1];
  __shared__ uint32_t sh_tmem;
  __shared__ int sh_abort;
  // segment that last had non-finite values in tiles not seen whole, by the
  // segment's index mod 8 (loads run less than three segments ahead)
  __shared__ int sh_bad[8];
  volatile int* abort_flag = &sh_abort;
  const uint32_t full = smem(bars), empty = full + 8 * kStages, fixed = empty + 8 * kStages;
  const uint32_t q_full = fixed + 8 * kStages, s_full = q_full + 8 * kTiles, p_ready = s_full + 8 * kTiles,
                 o_full = p_ready + 8 * kTiles, drained = o_full + 8 * kTiles;
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;

  if (w == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem(&sh_tmem)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 3);  // the MMAs' completion and warps 10 and 11
      mbar_init(fixed + 8 * i, 2);
    }
    for (int i = 0; i < kTiles; ++i) {
      mbar_init(q_full + 8 * i, kTile);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_ready + 8 * i, 4);
      mbar_init(o_full + 8 * i, 1);
    }
    mbar_init(drained, 1);
    sh_abort = 0;
    for (int i = 0; i < 8; ++i) sh_bad[i] = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh_tmem;
  const int seg0 = __ldg(first + blockIdx.x), seg1 = __ldg(first + blockIdx.x + 1);
  bool gave_up = false;

  if (w >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (w == 8) {
      // ---------------- loads: K of the first tile, then V and the next K ----------------
      const int page = 1 << a.c.page_shift, box = min(kKeys, page);
      int n_tile = 0;
      auto load = [&](const Seg& s, const int* table, const CUtensorMap* map, int it) {
        const int j = s.slot0(it) + lane * box;
        const bool mine = lane * box < kKeys && j < s.n;
        const int p = mine ? __ldg(table + (j >> a.c.page_shift)) : 0;
        const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
        const int st = n_tile % kStages, round = n_tile / kStages;
        if (round > 0 && !mbar_wait_bounded(empty + 8 * st, (round - 1) & 1, kWaitNs, abort_flag)) gave_up = true;
        if (__any_sync(0xffffffffu, gave_up)) {
          gave_up = true;
          return;
        }
        if (lane == 0) mbar_expect(full + 8 * st, (uint32_t)(boxes * box * DP * 2));
        __syncwarp();
        if (mine) {
          const uint32_t dst = smem(ring) + (uint32_t)(st * kBytes + lane * box * 128);
#pragma unroll
          for (int half = 0; half < DP / 64; ++half)
            load_box(dst + half * kHalf, map, 64 * half, j & (page - 1), p * a.c.heads + s.g.head, full + 8 * st);
        }
        ++n_tile;
      };
      for (int si = seg0; si < seg1 && !gave_up; ++si) {
        const Seg s(a, segs[si]);
        const int* table = a.s.table + (size_t)s.g.seq * a.s.stride;
        if (s.g.it0 >= s.g.it1) continue;
        load(s, table, &kmap, s.g.it0);
        for (int it = s.g.it0; it < s.g.it1 && !gave_up; ++it) {
          load(s, table, &vmap, it);
          if (it + 1 < s.g.it1 && !gave_up) load(s, table, &kmap, it + 1);
        }
      }
      if (gave_up) {  // the loads in flight still land in this CTA's memory
        *abort_flag = 1;
        for (int t = max(0, n_tile - kStages); t < n_tile; ++t)
          mbar_wait_bounded(full + 8 * (t % kStages), (t / kStages) & 1, kWaitNs);
      }
    } else if (w == 9) {
      // ---------------- MMAs ----------------
      if (lane == 0) {
        int n_tile = 0;
        uint32_t fix_phase = 0;  // per stage
        int cnt_p[kTiles] = {}, cnt_q[kTiles] = {};
        auto wait = [&](uint32_t bar, int phase) {
          if (!gave_up && !mbar_wait_bounded(bar, phase & 1, kWaitNs, abort_flag)) gave_up = true;
          return !gave_up;
        };
        auto scores = [&](int i, int st) {
          const uint32_t q = smem(sm) + i * kBytes, k = smem(ring) + st * kBytes;
#pragma unroll
          for (int ks = 0; ks < DP / 16; ++ks) {
            const uint32_t off = (ks >> 2) * kHalf + (ks & 3) * 32;
            mma_ss(tmem + i * 128, desc_k(q + off), desc_k(k + off), idesc<T>(kKeys, false), ks > 0);
          }
          commit(s_full + 8 * i);
        };
        for (int si = seg0; si < seg1 && !gave_up; ++si) {
          const Seg s(a, segs[si]);
          const int nt = s.tiles();
          if (s.g.it0 >= s.g.it1) continue;
          const int k0 = n_tile % kStages;
          if (!wait(full + 8 * k0, n_tile / kStages)) break;
          for (int i = 0; i < nt; ++i) {
            if (!wait(q_full + 8 * i, cnt_q[i]++)) break;
            fence_after();
            scores(i, k0);
          }
          if (gave_up) break;
          commit(empty + 8 * k0);
          ++n_tile;
          for (int it = s.g.it0; it < s.g.it1 && !gave_up; ++it) {
            const int sv = n_tile % kStages;
            if (!wait(full + 8 * sv, n_tile / kStages)) break;
            if (!sees_whole(s.slot0(it), s.pa, s.pb, a.window, a.sinks)) {
              if (!wait(fixed + 8 * sv, (fix_phase >> sv) & 1)) break;
              fix_phase ^= 1u << sv;
            }
            ++n_tile;
            const bool more = it + 1 < s.g.it1;
            const int sk = n_tile % kStages;
            for (int i = 0; i < nt; ++i) {
              if (!wait(p_ready + 8 * i, cnt_p[i]++)) break;
              fence_after();
              const uint32_t v = smem(ring) + sv * kBytes;
#pragma unroll
              for (int ks = 0; ks < kKeys / 16; ++ks)
                mma_ts(tmem + 256 + i * DP, tmem + i * 128 + ks * 8, desc_mn(v + ks * 2048), idesc<T>(DP, true),
                       it > s.g.it0 || ks > 0);
              if (more) {
                if (i == 0 && !wait(full + 8 * sk, n_tile / kStages)) break;
                scores(i, sk);
              } else {
                commit(o_full + 8 * i);
              }
            }
            if (gave_up) break;
            commit(empty + 8 * sv);
            if (more) {
              commit(empty + 8 * sk);
              ++n_tile;
            }
          }
        }
        if (gave_up) {  // the MMAs in flight still use this CTA's memory
          *abort_flag = 1;
          commit(drained);
          mbar_wait_bounded(drained, 0, kWaitNs);
        }
      }
      __syncwarp();
    } else {
      // ---------------- V tiles that not every row sees whole ----------------
      // These warps see every tile, in order, and a stage is not filled again
      // before they have: the parity that they wait for is never ambiguous.
      const int t = (w - 10) * 32 + lane;
      int n_tile = 0;
      for (int si = seg0; si < seg1 && !gave_up; ++si) {
        const Seg s(a, segs[si]);
        // K of the first tile, then V, K, V, ..., V
        for (int k = 0; k < 2 * (s.g.it1 - s.g.it0); ++k, ++n_tile) {
          const int st = n_tile % kStages;
          if (!mbar_wait_bounded(full + 8 * st, (n_tile / kStages) & 1, kWaitNs, abort_flag)) gave_up = true;
          if (__any_sync(0xffffffffu, gave_up)) {
            gave_up = true;
            break;
          }
          const int j0 = s.slot0(s.g.it0 + (k >> 1));
          if ((k & 1) && !sees_whole(j0, s.pa, s.pb, a.window, a.sinks)) {
            bool bad = false;
            for (int i = t; i < kKeys * (DP / 8); i += 64) {
              const int row = i / (DP / 8), c = i - row * (DP / 8), j = j0 + row;
              const bool any = j <= s.pb && (!a.window || j > s.pa - a.window || j < a.sinks);
              uint4* q = reinterpret_cast<uint4*>(ring + (size_t)st * kBytes + tile_off(row, c));
              if (!any) *q = make_uint4(0, 0, 0, 0);
              else {
                uint4 v = *q;
                if (drop_nonfinite<T>(v)) {
                  *q = v;
                  bad = true;
                }
              }
            }
            if (bad) sh_bad[si & 7] = si;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the tensor core reads what was written
            __syncwarp();
            if (lane == 0) mbar_arrive(fixed + 8 * st);
          }
          if (lane == 0) mbar_arrive(empty + 8 * st);
        }
      }
      if (gave_up) *abort_flag = 1;
    }
  } else {
    // ---------------- softmax and output ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int i = w >> 2, t = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (w & 3)) << 16;
    const uint32_t ts = tmem + lanes + i * 128, to = tmem + lanes + 256 + i * DP;
    const int D = a.c.dim, Hq = a.c.heads * a.group;
    // a negative scale turns the queries' sign, a zero one makes them zero
    const float c = a.scale2 == 0.0f ? 1.0f : fabsf(a.scale2), lag = 8.0f / c;
    const uint32_t q_xor = a.scale2 < 0.0f ? 0x80008000u : 0u, q_and = a.scale2 == 0.0f ? 0u : 0xFFFFFFFFu;
    int cnt_s = 0, cnt_o = 0;
    for (int si = seg0; si < seg1 && !gave_up; ++si) {
      const Seg s(a, segs[si]);
      if (i >= s.tiles()) continue;
      const int r = i * kTile + t;
      const bool valid = r < s.rows;
      const int tok = (s.g.row0 + r) / a.group, hq = s.g.head * a.group + (s.g.row0 + r) % a.group;
      const int pos = s.n - s.nq + tok;
      const int count = s.g.it1 - s.g.it0;
      float m = -INFINITY, l = 0.0f;
      if (count > 0) {
        const uint16_t* p =
            static_cast<const uint16_t*>(a.q) + (size_t)(s.q0 + tok) * a.q_token + (size_t)hq * a.q_head;
#pragma unroll
        for (int ch = 0; ch < DP / 8; ++ch) {
          uint4 x = make_uint4(0, 0, 0, 0);
          if (valid && 8 * ch < D) {
            if (wide_q) x = __ldg(reinterpret_cast<const uint4*>(p + 8 * ch));
            else {
              uint16_t e[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) e[k] = __ldg(p + 8 * ch + k);
              x = make_uint4(e[0] | ((uint32_t)e[1] << 16), e[2] | ((uint32_t)e[3] << 16),
                             e[4] | ((uint32_t)e[5] << 16), e[6] | ((uint32_t)e[7] << 16));
            }
          }
          x.x = (x.x & q_and) ^ q_xor;
          x.y = (x.y & q_and) ^ q_xor;
          x.z = (x.z & q_and) ^ q_xor;
          x.w = (x.w & q_and) ^ q_xor;
          *reinterpret_cast<uint4*>(sm + i * kBytes + tile_off(t, ch)) = x;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(q_full + 8 * i);
      }
      // the slots of this row tile's first and last query
      const int pa = s.n - s.nq + (s.g.row0 + i * kTile) / a.group;
      const int pb = s.n - s.nq + (s.g.row0 + min(s.rows, (i + 1) * kTile) - 1) / a.group;
      for (int it = s.g.it0; it < s.g.it1; ++it, ++cnt_s) {
        const int j0 = s.slot0(it);
        if (!mbar_wait_bounded(s_full + 8 * i, cnt_s & 1, kWaitNs, abort_flag)) gave_up = true;
        if (__any_sync(0xffffffffu, gave_up)) {
          gave_up = true;
          break;
        }
        fence_after();
        float x[kKeys];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(ts + 32 * q, x + 32 * q);
        tmem_wait_ld();
        if (!sees_whole(j0, pa, pb, a.window, a.sinks)) {
          const int hi = pos - j0, lo = a.window ? hi - a.window : -1, sk = a.sinks - j0;
#pragma unroll
          for (int e = 0; e < kKeys; ++e)
            if (e > hi || (e <= lo && e >= sk)) x[e] = -INFINITY;
        }
        float mx = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int e = 0; e < kKeys; e += 4) {
          mx = fmaxf(mx, fmaxf(x[e], x[e + 1]));
          mx1 = fmaxf(mx1, fmaxf(x[e + 2], x[e + 3]));
        }
        mx = fmaxf(mx, mx1);
        if (it == s.g.it0) {
          m = mx;
        } else {
          const bool up = mx > m + lag;
          if (__any_sync(0xffffffffu, up)) {
            // this tile's scores were announced behind the last O += P V
            const float f = up ? ex2((m - mx) * c) : 1.0f;
            if (up) m = mx;
            l *= f;
#pragma unroll 1
            for (int q = 0; q < DP / 32; ++q) {
              float o[32];
              tmem_ld32(to + 32 * q, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] *= f;
              tmem_st32(to + 32 * q, o);
            }
          }
        }
        const float mu = m == -INFINITY ? 0.0f : m * c;
        const float2 c2 = make_float2(c, c), mu2 = make_float2(-mu, -mu);
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float2 y = ffma2(make_float2(x[32 * q + 2 * e], x[32 * q + 2 * e + 1]), c2, mu2);
            y.x = ex2(y.x);
            y.y = ex2(y.y);
            sum.x += y.x;
            sum.y += y.y;
            // the numerators are rounded to the cache's type for the product
            // with the values; the sum keeps them in f32
            pk[e] = pack2<T>(y.x, y.y);
          }
          tmem_st16(ts + 16 * q, pk);
        }
        l += sum.x + sum.y;
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + 8 * i);
      }
      if (gave_up) break;
      if (count > 0) {
        if (!mbar_wait_bounded(o_full + 8 * i, cnt_o & 1, kWaitNs, abort_flag)) gave_up = true;
        if (__any_sync(0xffffffffu, gave_up)) {
          gave_up = true;
          break;
        }
        ++cnt_o;
        fence_after();
      }
      const bool bad = count > 0 && sh_bad[si & 7] == si;
      const bool none = l == 0.0f;
      const float inv = none ? 0.0f : 1.0f / l;
      const size_t at = (size_t)(s.q0 + tok) * Hq + hq;
#pragma unroll 1
      for (int q = 0; q < DP / 32; ++q) {
        float o[32];
        if (count > 0) {
          tmem_ld32(to + 32 * q, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.0f;
        }
        if (!valid) continue;
        if (bad) {
          const int* table = a.s.table + (size_t)s.g.seq * a.s.stride;
          for (int it = s.g.it0; it < s.g.it1; ++it) {
            const int j0 = s.slot0(it);
            if (sees_whole(j0, s.pa, s.pb, a.window, a.sinks)) continue;
            for (int j = j0; j < j0 + kKeys && j <= pos; ++j) {
              if (!paged_sees(pos, j, a.window, a.sinks)) continue;
              const T* v = static_cast<const T*>(a.c.values) + paged_row(table, a.c, s.g.head, j) + 32 * q;
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                if (32 * q + e >= D) continue;
                const float y = to_float<T>(v[e]);
                if (!isfinite(y)) o[e] += y;
              }
            }
          }
        }
        if (s.g.part >= 0) {
          float* dst = a.part_o + ((size_t)s.g.part * kRows + r) * D + 32 * q;
#pragma unroll
          for (int e = 0; e < 32; e += 4)  // D is a multiple of 8
            if (32 * q + e < D) *reinterpret_cast<float4*>(dst + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        } else {
          T* dst = static_cast<T*>(a.out) + at * D + 32 * q;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            if (32 * q + e >= D) continue;
            uint32_t y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              y[k] = none ? 0u : pack2<T>(o[e + 2 * k] * inv, o[e + 2 * k + 1] * inv);
            if (wide_out) *reinterpret_cast<uint4*>(dst + e) = make_uint4(y[0], y[1], y[2], y[3]);
            else
#pragma unroll
              for (int k = 0; k < 8; ++k)
                reinterpret_cast<uint16_t*>(dst)[e + k] = (uint16_t)(y[k >> 1] >> (16 * (k & 1)));
          }
        }
      }
      if (valid) {
        const float m2 = m == -INFINITY ? -INFINITY : m * c;
        if (s.g.part >= 0)
          *reinterpret_cast<float2*>(a.part_ml + ((size_t)s.g.part * kRows + r) * 2) = make_float2(m2, l);
        else if (a.lse)
          a.lse[at] = none ? -INFINITY : (m2 + log2f(l)) * (float)M_LN2;
      }
      // the next segment's products overwrite O: ordered by its numerators' barrier
      fence_before();
    }
    if (gave_up) *abort_flag = 1;
  }
  if (gave_up && a.status) atomicOr(a.status, kDevErrTimeout);
  fence_before();
  __syncthreads();
  fence_after();
  if (w == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}

template <typename T, int DP>
cudaError_t launch_typed(const CUtensorMap& km, const CUtensorMap& vm, const PagedAttn& a, const PagedWork& w,
                         cudaStream_t st) {
  auto kern = k_paged_chunk<T, DP>;
  constexpr size_t bytes = smem_bytes<DP>();
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) return e;
  const bool wide_q = (a.q_token | a.q_head) % 8 == 0 && aligned(a.q, 16);
  kern<<<w.ctas, kThreads, bytes, st>>>(km, vm, a, w.segs, w.first, wide_q, aligned(a.out, 16));
  note_launches(1);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_chunk(const PagedAttn& a, const PagedWork& w, cudaStream_t st) {
  if (w.ctas == 0) return cudaSuccess;
  CUtensorMap km, vm;
  const int rows = std::min(kKeys, 1 << a.c.page_shift);
  if (!paged_map(&km, a.c, a.c.keys, rows) || !paged_map(&vm, a.c, a.c.values, rows)) return cudaErrorInvalidValue;
  if (a.c.dtype == KVF_IN_F16)
    return a.c.dim <= 64 ? launch_typed<__half, 64>(km, vm, a, w, st) : launch_typed<__half, 128>(km, vm, a, w, st);
  return a.c.dim <= 64 ? launch_typed<__nv_bfloat16, 64>(km, vm, a, w, st)
                       : launch_typed<__nv_bfloat16, 128>(km, vm, a, w, st);
}

}  // namespace kvf
