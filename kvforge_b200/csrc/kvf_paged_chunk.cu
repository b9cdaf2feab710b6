// Attention of many rows (chunks of new tokens, long drafts) over a paged
// 16-bit cache, on tcgen05.
//
// The formulas are those of kvf_paged_attn.cu. With R rows per (sequence, KV
// head) the two products cost 4 R n D operations and the softmax R n
// exponentials; at D = 128 an SM's tensor core needs 1024 cycles for a tile of
// 128 rows by 128 slots, and its 16 exponentials per cycle need 1024 as well,
// so the kernel is bound by both and must keep them busy at the same time.
// 2048 tokens on 30720 cached, 32 query and 8 KV heads of 128 in f16: 957-967
// us at 1965 MHz (1100 TFLOP/s), 1110-1140 in steady calls, whose load brings
// the clock down. Neither unit is full (45 % each in ncu, 1184 tokens on 8192): a
// row tile's products wait for its softmax and the other way round.
//
// One persistent CTA per SM walks segments of (sequence, KV head, 256 rows),
// two row tiles of 128 whose work alternates on the tensor core: while one
// tile's scores go through the softmax, the other tile's products run.
//   warps 0-3, 4-7: softmax of row tile 0 and 1, a row per thread. A tile of
//     scores is read from TMEM, the numerators go back over it in the cache's
//     16-bit type, as the A operand of the second product. The running maximum
//     is followed only when it grows by more than 2^8 (then the sums in TMEM
//     are rescaled): numerators stay below 2^8, which f16 holds, and the
//     rescaling all but vanishes after the first tiles. The two row tiles take
//     turns: left to themselves they fall into step, both in the softmax and
//     then both on the tensor core (4400 instead of 3400 cycles per pair of
//     tiles). Eight more warps, two threads a row, are slower (993 against 960
//     us at full clock): the halves of a row have to meet for its maximum.
//   warp 8: tensor-map loads of K and V tiles, a box per page.
//   warps 9, 10: the MMAs of row tile 0 and 1, each issued by one thread, so
//     that one warp's waits (about 110 cycles even when there is nothing to
//     wait for) pass while the other's products run. S = Q K^T of a tile is
//     issued directly behind the same row tile's O += P V: MMAs of one thread
//     run in order, so S may overwrite P, and the barrier that announces S also
//     announces that O is free.
// A V tile that not every row sees whole is put right in shared memory by the
// first row tile's warps: slots that no row sees become zeros (their pages may
// hold anything), non-finite values that only some rows see become zeros and
// are added to the rows that see them at the end (their product with any
// positive weight is the value itself).
// TMEM: 2 x 128 columns of scores (numerators over them), 2 x D of sums. Every
// wait is bounded; one that runs out ends all roles and sets kDevErrTimeout.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "kvf_paged_tc.cuh"

namespace kvf {
namespace {

using namespace ptx;

constexpr int kRows = kChunkRows, kKeys = kChunkKeys;
constexpr int kTiles = kRows / kTile;
constexpr int kSoftmaxWarps = 8;
constexpr int kThreads = 32 * (kSoftmaxWarps + 4);
// registers per thread: launched with 168 (65536 / 384), the softmax warps take
// what the others give up: 256 x 200 + 128 x 104 = 384 x 168
constexpr int kRegsSoftmax = 200, kRegsOther = 104;

// quarter of a tile after which the other row tile may start its own
constexpr int kHandOver = 0;

template <int DP>
constexpr int tile_bytes() { return kTile * DP * 2; }
template <int DP>
constexpr int stages() { return DP == 128 ? 5 : 10; }
template <int DP>
struct Shared {
  uint64_t bars[3 * stages<DP>() + 6 * kTiles];
  // segment that last had non-finite values in tiles not seen whole: places 0 and
  // 1 in turn for segments of two row tiles, 2 and 3 for those of one. (The second
  // row tile may still look a segment up while the first is past any number of
  // single ones, but the first begins a third of two tiles only behind its turn.)
  int bad[4];
  uint32_t tmem;
  int abort;
};
template <int DP>
constexpr size_t smem_bytes() { return (size_t)(kTiles + stages<DP>()) * tile_bytes<DP>() + sizeof(Shared<DP>); }
// more than half of an SM's shared memory: one CTA per SM, whose TMEM is free
static_assert(2 * (smem_bytes<64>() + 1024) > 228 * 1024 && smem_bytes<128>() <= 227 * 1024, "one CTA");

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

// the sum of the non-finite values of one column that the query at slot pos
// sees in tiles that not every row of the segment sees whole (v: the column in
// the pool's first row)
template <typename T>
__device__ __noinline__ float nonfinite_sum(const T* v, const int* table, int shift, int heads, int head, int dim,
                                            int it0, int it1, PagedSpan span, int pa, int pb, int pos, int window,
                                            int sinks) {
  float sum = 0.0f;
  for (int it = it0; it < it1; ++it) {
    const int j0 = (it < span.nsink ? it : span.first + it - span.nsink) * kKeys;
    if (sees_whole(j0, pa, pb, window, sinks)) continue;
    for (int j = j0; j < j0 + kKeys && j <= pos; ++j) {
      if (!paged_sees(pos, j, window, sinks)) continue;
      const size_t row = (((size_t)__ldg(table + (j >> shift)) * heads + head) << shift) + (j & ((1 << shift) - 1));
      const float y = to_float<T>(v[row * dim]);
      if (!isfinite(y)) sum += y;
    }
  }
  return sum;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    k_paged_chunk(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, PagedAttn a,
                  const PagedSeg* __restrict__ segs, const int* __restrict__ first, bool wide_q, bool wide_out) {
  constexpr int kStages = stages<DP>(), kBytes = tile_bytes<DP>();
  // all shared memory is dynamic: the tiles first, on the 1024 bytes that the
  // swizzle's pattern wants (checked below), then what the roles share
  extern __shared__ __align__(1024) uint8_t sm[];
  uint8_t* ring = sm + kTiles * kBytes;
  Shared<DP>& sh = *reinterpret_cast<Shared<DP>*>(ring + kStages * kBytes);
  if (smem(sm) & 1023u) {
    if (threadIdx.x == 0 && a.status) atomicOr(a.status, kDevErrTimeout);
    return;
  }
  volatile int* abort_flag = &sh.abort;
  const uint32_t full = smem(sh.bars), empty = full + 8 * kStages, fixed = empty + 8 * kStages;
  const uint32_t q_full = fixed + 8 * kStages, s_full = q_full + 8 * kTiles, p_ready = s_full + 8 * kTiles,
                 o_full = p_ready + 8 * kTiles, drained = o_full + 8 * kTiles, turn = drained + 8 * kTiles;
  const int tid = threadIdx.x, w = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

  if (w == kSoftmaxWarps + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem(&sh.tmem)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, kTiles);
      mbar_init(fixed + 8 * i, 4);
    }
    for (int i = 0; i < kTiles; ++i) {
      mbar_init(q_full + 8 * i, 4);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_ready + 8 * i, 4);
      mbar_init(o_full + 8 * i, 1);
      mbar_init(drained + 8 * i, 1);
      mbar_init(turn + 8 * i, 4);
    }
    sh.abort = 0;
    for (int i = 0; i < 4; ++i) sh.bad[i] = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  constexpr uint32_t tmem = 0;  // all columns are this CTA's, so they start at 0
  const int seg0 = __ldg(first + blockIdx.x), seg1 = __ldg(first + blockIdx.x + 1);
  bool gave_up = false;

  if (w >= kSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (w == kSoftmaxWarps) {
      // ---------------- loads: K of the first tile, then V and the next K ----------------
      const int page = 1 << a.c.page_shift, box = min(kKeys, page);
      int n_tile = 0;
      auto load = [&](const Seg& s, const int* table, const CUtensorMap* map, int it) {
        const int j = s.slot0(it) + lane * box;
        const bool mine = lane * box < kKeys && j < s.n;
        const int p = mine ? __ldg(table + (j >> a.c.page_shift)) : 0;
        const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
        const int st = n_tile % kStages, round = n_tile / kStages;
        if (round > 0 && !mbar_wait(empty + 8 * st, (round - 1) & 1, abort_flag)) gave_up = true;
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
    } else if (w < kSoftmaxWarps + 1 + kTiles) {
      // ---------------- MMAs of row tile i ----------------
      // One copy of this code for both warps, with short inner loops: the roles'
      // loops together have to stay within the instruction caches (a copy per
      // warp made all warps of the SM wait for instructions, 25 % in all).
      const int i = w - kSoftmaxWarps - 1;
      const bool lead = lane == 0;
      const uint32_t qd = desc_k(smem(sm)) + i * (kBytes >> 4), kd = desc_k(smem(ring)), vd = desc_mn(smem(ring));
      const uint32_t ts = tmem + i * 128, to = tmem + 256 + i * DP;
      int st = 0;                                                      // the stage of the ring's next tile
      uint32_t st_phase = 0, fix_phase = 0, p_phase = 0, q_phase = 0;  // parities: the ring's, one per stage, the others
      auto wait = [&](uint32_t bar, uint32_t parity) {
        if (!mbar_wait(bar, parity, abort_flag)) gave_up = true;
        if (__any_sync(0xffffffffu, gave_up)) gave_up = true;
        return !gave_up;
      };
      auto next = [&] {
        if (++st == kStages) {
          st = 0;
          st_phase ^= 1u;
        }
      };
      auto scores = [&](int stage) {
        const uint32_t k = kd + stage * (kBytes >> 4);
#pragma unroll 1
        for (int half = 0; half < DP / 64; ++half)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const uint32_t off = (half * kHalf + ks * 32) >> 4;
            mma_ss(lead, ts, qd + off, k + off, idesc<T>(kKeys, false), half + ks > 0);
          }
        commit(lead, s_full + 8 * i);
      };
      for (int si = uniform(seg0); si < uniform(seg1) && !gave_up; ++si) {
        const Seg s(a, segs[si]);
        const int it0 = uniform(s.g.it0), it1 = uniform(s.g.it1);
        if (it0 >= it1) continue;
        if (i >= uniform(s.tiles())) {  // no rows here: the tiles pass by
          for (int k = 0; k < 2 * (it1 - it0); ++k) {
            if (!wait(full + 8 * st, st_phase)) break;
            if (lead) mbar_arrive(empty + 8 * st);
            const int j0 = s.slot0(it0 + (k >> 1));
            if ((k & 1) && !uniform(sees_whole(j0, s.pa, s.pb, a.window, a.sinks))) fix_phase ^= 1u << st;
            next();
          }
          continue;
        }
        if (!wait(q_full + 8 * i, q_phase) || !wait(full + 8 * st, st_phase)) break;
        q_phase ^= 1u;
        fence_after();
        scores(st);
        commit(lead, empty + 8 * st);
        next();
        for (int it = it0; it < it1; ++it) {
          const int sv = st;
          if (!wait(full + 8 * sv, st_phase)) break;
          // the first row tile's numerators come behind its own work on V
          if (i == 1 && !uniform(sees_whole(s.slot0(it), s.pa, s.pb, a.window, a.sinks))) {
            if (!wait(fixed + 8 * sv, (fix_phase >> sv) & 1)) break;
            fix_phase ^= 1u << sv;
          }
          next();
          const bool more = it + 1 < it1;
          // the next K is looked for first: the numerators come last
          if (more && !wait(full + 8 * st, st_phase)) break;
          if (!wait(p_ready + 8 * i, p_phase)) break;
          p_phase ^= 1u;
          fence_after();
          const uint32_t v = vd + sv * (kBytes >> 4);
#pragma unroll 1
          for (int k4 = 0; k4 < kKeys / 16; k4 += 4)
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              mma_ts(lead, to, ts + (k4 + ks) * 8, v + (k4 + ks) * (2048 >> 4), idesc<T>(DP, true),
                     k4 + ks > 0 || it > it0);
          if (more) {
            scores(st);
            commit(lead, empty + 8 * sv);
            commit(lead, empty + 8 * st);
            next();
          } else {
            commit(lead, o_full + 8 * i);
            commit(lead, empty + 8 * sv);
          }
        }
      }
      if (gave_up) {  // the MMAs in flight still use this CTA's memory
        *abort_flag = 1;
        commit(lead, drained + 8 * i);
        mbar_wait_bounded(drained + 8 * i, 0, kWaitNs);
      }
    }
  } else {
    // ---------------- softmax and output ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int i = w >> 2, t = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (w & 3)) << 16;
    const uint32_t ts = tmem + lanes + i * 128, to = tmem + lanes + 256 + i * DP;
    const int D = a.c.dim;
    // a negative scale turns the queries' sign; the smallest number stands for zero
    // (every finite score becomes 0 to within 5e-7, and NaN stays NaN)
    const float c = a.scale2 == 0.0f ? 1.4e-45f : fabsf(a.scale2);
    const float lag = fminf(8.0f / c, FLT_MAX);  // finite: nothing seen yet (-inf) stays -inf with it added
    int cnt_s = 0, cnt_o = 0;
    uint32_t turns = 0;
    int ring0 = 0;  // tiles of K and V before this segment
    uint32_t bad_at = 0;  // bit 0: the place of the next segment of two row tiles, bit 1: of one
    for (int si = seg0; si < seg1; ++si) {
      const Seg s(a, segs[si]);
      const int count = s.g.it1 - s.g.it0;
      if (i >= s.tiles()) continue;
      const int r = i * kTile + t;
      const bool valid = r < s.rows;
      const int tok = (s.g.row0 + r) / a.group, hq = s.g.head * a.group + (s.g.row0 + r) % a.group;
      const int pos = s.n - s.nq + tok;
      const bool two = s.tiles() == kTiles;
      float m = -INFINITY, l = 0.0f;
      if (count > 0) {
        const uint32_t q_xor = a.scale2 < 0.0f ? 0x80008000u : 0u;
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
              for (int u = 0; u < 8; ++u) e[u] = __ldg(p + 8 * ch + u);
              x = make_uint4(e[0] | ((uint32_t)e[1] << 16), e[2] | ((uint32_t)e[3] << 16),
                             e[4] | ((uint32_t)e[5] << 16), e[6] | ((uint32_t)e[7] << 16));
            }
          }
          x.x ^= q_xor;
          x.y ^= q_xor;
          x.z ^= q_xor;
          x.w ^= q_xor;
          *reinterpret_cast<uint4*>(sm + i * kBytes + tile_off(t, ch)) = x;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full + 8 * i);
      }
      // the slots of this row tile's first and last query
      const int pa = s.n - s.nq + (s.g.row0 + i * kTile) / a.group;
      const int pb = s.n - s.nq + (s.g.row0 + min(s.rows, (i + 1) * kTile) - 1) / a.group;
      for (int it = s.g.it0; it < s.g.it1; ++it, ++cnt_s) {
        const int j0 = s.slot0(it);
        // row tile 0 first, then in turns, where there are two
        if (two) {
          if ((i != 0 || turns != 0) && !mbar_wait(turn + 8 * i, (turns - (i == 0)) & 1u, abort_flag)) gave_up = true;
          ++turns;
        }
        if (!mbar_wait(s_full + 8 * i, cnt_s & 1, abort_flag)) gave_up = true;
        if (__any_sync(0xffffffffu, gave_up)) {
          gave_up = true;
          break;
        }
        fence_after();
        if (!sees_whole(j0, pa, pb, a.window, a.sinks)) {
          // a pass of its own over the scores in TMEM, so that the softmax has no
          // code for it: slots past the row's own, or in front of its window
          const int hi = pos - j0, lo = a.window ? hi - a.window : -1, sk = a.sinks - j0;
#pragma unroll 1
          for (int q = 0; q < kKeys; q += 32) {
            if (j0 + q + 31 <= pa && (!a.window || j0 + q > pb - a.window || j0 + q + 32 <= a.sinks)) continue;
            float x[32];
            tmem_ld32(ts + q, x);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (e > hi - q || (e <= lo - q && e >= sk - q)) x[e] = -INFINITY;
            tmem_st32(ts + q, x);
          }
          tmem_wait_st();
        }
        if (i == 0 && !sees_whole(j0, s.pa, s.pb, a.window, a.sinks)) {
          // the V tile of these slots: tile 2 (it - it0) + 1 of the segment. Its
          // stage's earlier tiles are all used up, so the parity is not ambiguous
          const int tile = ring0 + 2 * (it - s.g.it0) + 1, st = tile % kStages;
          if (!mbar_wait(full + 8 * st, (tile / kStages) & 1, abort_flag)) gave_up = true;
          if (__any_sync(0xffffffffu, gave_up)) {
            gave_up = true;
            break;
          }
          bool bad = false;
#pragma unroll 4
          for (int k = t; k < kKeys * (DP / 8); k += kTile) {
            const int row = k / (DP / 8), ch = k - row * (DP / 8), j = j0 + row;
            // a slot that all rows see stays as it is
            if (j <= s.pa && (!a.window || j > s.pb - a.window || j < a.sinks)) continue;
            uint4* q = reinterpret_cast<uint4*>(ring + (size_t)st * kBytes + tile_off(row, ch));
            if (j > s.pb || (a.window && j <= s.pa - a.window && j >= a.sinks)) {
              *q = make_uint4(0, 0, 0, 0);
            } else {
              uint4 v = *q;
              if (drop_nonfinite<T>(v)) {
                *q = v;
                bad = true;
              }
            }
          }
          if (bad) sh.bad[two ? bad_at & 1 : 2 + (bad_at >> 1)] = si;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the tensor core reads what was written
          __syncwarp();
          if (lane == 0) mbar_arrive(fixed + 8 * st);
        }
        float x[kKeys];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(ts + 32 * q, x + 32 * q);
        tmem_wait_ld();
        float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int e = 4; e < kKeys - 4; e += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], x[e + k], x[e + 4 + k]);
        mx[0] = max3(mx[0], mx[1], x[kKeys - 4]);
        mx[2] = max3(mx[2], mx[3], x[kKeys - 3]);
        float own = max3(mx[0], x[kKeys - 2], x[kKeys - 1]);
        own = max3(own, mx[2], mx[2]);
        // a NaN or +inf score makes all of its row NaN: through the maximum, so
        // that each single exponential need not look for it
        if (own == INFINITY) own = NAN;
        if (it == s.g.it0) {
          m = own;
        } else {
          const bool up = !(own <= m + lag);  // NaN too
          if (__any_sync(0xffffffffu, up)) {
            // this tile's scores were announced behind the last O += P V
            const float f = up ? ex2((m - own) * c) : 1.0f;
            if (up) m = own;
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
        float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float2 y0 = ffma2(make_float2(x[32 * q + 2 * e], x[32 * q + 2 * e + 1]), c2, mu2);
            float2 y1 = ffma2(make_float2(x[32 * q + 2 * e + 2], x[32 * q + 2 * e + 3]), c2, mu2);
            y0.x = ex2(y0.x);
            y0.y = ex2(y0.y);
            y1.x = ex2(y1.x);
            y1.y = ex2(y1.y);
            sum0 = fadd2(sum0, y0);
            sum1 = fadd2(sum1, y1);
            // the numerators are rounded to the cache's type for the product
            // with the values; the sum keeps them in f32
            pk[e] = pack2<T>(y0.x, y0.y);
            pk[e + 1] = pack2<T>(y1.x, y1.y);
          }
          tmem_st16(ts + 16 * q, pk);
          if (q == kHandOver && two) {  // the other tile's wake-up and loads pass meanwhile
            __syncwarp();
            if (lane == 0) mbar_arrive(turn + 8 * (i ^ 1));
          }
        }
        l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + 8 * i);
      }
      if (count > 0 && !gave_up) {
        if (!mbar_wait(o_full + 8 * i, cnt_o & 1, abort_flag)) gave_up = true;
        if (__any_sync(0xffffffffu, gave_up)) gave_up = true;
        ++cnt_o;
        fence_after();
      }
      if (gave_up) break;
      bool bad = false;
      if (count > 0) {
        bad = sh.bad[two ? bad_at & 1 : 2 + (bad_at >> 1)] == si;
        bad_at ^= two ? 1u : 2u;
      }
      const bool none = l == 0.0f;
      const float inv = none ? 0.0f : 1.0f / l;
      const size_t at = (size_t)(s.q0 + tok) * (a.c.heads * a.group) + hq;
#pragma unroll 1
      for (int q = 0; q < DP / 32; ++q) {
        const int col = 32 * q;
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
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (col + e < D)
              o[e] += nonfinite_sum<T>(static_cast<const T*>(a.c.values) + col + e,
                                       a.s.table + (size_t)s.g.seq * a.s.stride, a.c.page_shift, a.c.heads, s.g.head,
                                       D, s.g.it0, s.g.it1, s.span, s.pa, s.pb, pos, a.window, a.sinks);
        }
        if (s.g.part >= 0) {
          float* dst = a.part_o + ((size_t)s.g.part * kRows + r) * D + col;
#pragma unroll
          for (int e = 0; e < 32; e += 4)  // D is a multiple of 8
            if (col + e < D) *reinterpret_cast<float4*>(dst + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        } else {
          T* dst = static_cast<T*>(a.out) + at * D + col;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            if (col + e >= D) continue;
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
      ring0 += 2 * count;  // (only the first row tile, which every segment has, uses it)
      // the next segment's products overwrite O: ordered by its numerators' barrier
      fence_before();
    }
    if (gave_up) *abort_flag = 1;
  }
  if (gave_up && a.status) atomicOr(a.status, kDevErrTimeout);
  fence_before();
  __syncthreads();
  fence_after();
  if (w == kSoftmaxWarps + 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}

template <typename T, int DP>
cudaError_t launch_typed(const CUtensorMap& km, const CUtensorMap& vm, const PagedAttn& a, const PagedWork& w,
                         cudaStream_t st) {
  auto kern = k_paged_chunk<T, DP>;
  constexpr size_t bytes = smem_bytes<DP>();
  static OptInOnce done;
  cudaError_t e = opt_in_once(done, kern, bytes);
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
