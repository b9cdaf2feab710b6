// Attention over a paged cache on CUDA cores (every type, head_dim up to 256),
// the joining of cut tiles, and the attention weights of cached slots.
//
// One pass over the slots with the running maximum m and sum l of the softmax
// (base 2: s2 = scale * log2(e) * q.k):
//   m' = max(m, max s2);  f = 2^(m - m');  l' = f l + sum 2^(s2 - m');
//   O' = f O + sum 2^(s2 - m') v
// and out = O / l, lse = (m + log2 l) ln 2. A segment of the slots leaves
// (m, l, O); k_paged_join adds segments up with the weights 2^(m_i - max m).
// These kernels serve f32 pools and head dims that the tensor-core kernels do
// not take: products of all 24 bits on the multiply-add units. (Operands split
// into parts would give f32 products on the tensor cores too; not built.)
// Whole calls, against the bytes' time in brackets: f32 single tokens of 16
// sequences of 3000 to 16000 slots, 8 KV and 64 query heads of 128, 799 us (178);
// the same in bf16 with 32 query heads of 256, 2464 (178).
#include <cfloat>
#include <cmath>

#include "kvf_paged.cuh"

namespace kvf {
namespace {

constexpr int kGenThreads = 256;
constexpr int kPStride = kGenKeys + 4;  // rows of P, 16-byte aligned, four banks apart

constexpr int kPStrideLong = kGenKeysLong + 16;  // half a set of banks apart: two rows are written at once
constexpr int kSlabs = 4, kSlabFloats = 32 * 128;

// element (r, c) of a tile of f32 rows in shared memory, rows of DP floats (a
// multiple of 32): 16-byte groups are permuted by the row so that eight rows
// at one column lie in different banks
__device__ __forceinline__ int tile_at(int r, int c4, int DP) { return r * DP + ((c4 ^ (r & 7)) << 2); }

__device__ float4 g_zero;
__device__ __forceinline__ const void* sm_zero() { return &g_zero; }

// four (f32) or eight (16-bit) elements of a row as floats
template <typename T>
__device__ __forceinline__ void load16(const T* p, float (&x)[16 / sizeof(T)]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
  for (int i = 0; i < (int)(16 / sizeof(T)); ++i) x[i] = to_float(e[i]);
}

// Fills `rows` rows of DP floats; row(r) points at row r's first element, or
// is nullptr for a row of zeros. Rows of f32 in 16-byte pieces are copied
// asynchronously: one group, committed here; everything else is there at once.
template <typename T, typename Row>
__device__ __forceinline__ void fill_tile(float* sm, int rows, int DP, int D, bool wide, Row row) {
  if (wide) {
    constexpr int E = 16 / sizeof(T);
    // piece i = (r, c): i grows by the block's threads, without a division
    const int per = DP / E, dr = kGenThreads / per, dc = kGenThreads - dr * per;
    int r = threadIdx.x / per, c = threadIdx.x - r * per;
#pragma unroll 4
    while (r < rows) {
      const T* p = row(r);
      const bool there = p && c * E < D;
      if constexpr (sizeof(T) == 4) {
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(sm + tile_at(r, c, DP));
        // (a piece of zero bytes is filled with zeros; its address is any valid one)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst),
                     "l"(there ? (const void*)(p + c * E) : (const void*)sm_zero()), "r"(there ? 16 : 0)
                     : "memory");
      } else {
        float x[E];
        if (there) load16(p + c * E, x);
        else
#pragma unroll
          for (int e = 0; e < E; ++e) x[e] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e += 4)
          *reinterpret_cast<float4*>(sm + tile_at(r, (c * E + e) >> 2, DP)) =
              make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
      }
      r += dr;
      c += dc;
      if (c >= per) {
        c -= per;
        ++r;
      }
    }
  } else {
    for (int i = threadIdx.x; i < rows * DP; i += kGenThreads) {
      const int r = i / DP, c = i - r * DP;
      const T* p = row(r);
      sm[tile_at(r, c >> 2, DP) + (c & 3)] = (p && c < D) ? to_float(p[c]) : 0.0f;
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}
// waits until at most N of this thread's groups are still on their way
template <int N>
__device__ __forceinline__ void filled() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// scores of RT rows (ty * RT + i) and four slots (tx + 16 u) of this thread
template <int RT>
__device__ __forceinline__ void scores(const float* Q, const float* K, int DP, int ty, int tx, float (&s)[RT][4]) {
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int u = 0; u < 4; ++u) s[i][u] = 0.0f;
#pragma unroll 2
  for (int c = 0; c < DP / 4; ++c) {
    float4 q[RT], k[4];
#pragma unroll
    for (int i = 0; i < RT; ++i) q[i] = *reinterpret_cast<const float4*>(Q + tile_at(ty * RT + i, c, DP));
#pragma unroll
    for (int u = 0; u < 4; ++u) k[u] = *reinterpret_cast<const float4*>(K + tile_at(tx + 16 * u, c, DP));
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        s[i][u] = fmaf(q[i].x, k[u].x, s[i][u]);
        s[i][u] = fmaf(q[i].y, k[u].y, s[i][u]);
        s[i][u] = fmaf(q[i].z, k[u].z, s[i][u]);
        s[i][u] = fmaf(q[i].w, k[u].w, s[i][u]);
      }
  }
}

// 16 lanes share a row
__device__ __forceinline__ float half_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float half_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A 16 x 16 arrangement of threads: thread (ty, tx) holds the scores of RT
// rows and four slots, then those rows' sums of NU groups of four columns.
// Tiles of 64 slots; 64 rows (RT = 4), or 16 (RT = 1) for single tokens. Bound
// by shared-memory loads and the CUDA cores' multiply-adds at 64 rows and by
// loads at 16; two CTAs (64 rows, head_dim 128: 113 KB each) or three share an SM.
template <typename T, int RT, int NU>
__global__ void __launch_bounds__(kGenThreads, NU <= 2 ? 2 : 1) k_paged_attn(PagedAttn a, const PagedSeg* __restrict__ segs,
                                                            const int* __restrict__ first, int DP, bool wide,
                                                            bool wide_q) {
  constexpr int BR = 16 * RT;
  extern __shared__ float4 sm4[];
  float* Q = reinterpret_cast<float*>(sm4);  // [BR][DP]
  float* V = Q + BR * DP;                    // [64][DP]
  float* K = V + kGenKeys * DP;              // [64][DP]
  float* P = K + kGenKeys * DP;              // [BR][kPStride]
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int D = a.c.dim, Hq = a.c.heads * a.group;
  const int s1 = __ldg(first + blockIdx.x + 1);
  for (int si = __ldg(first + blockIdx.x); si < s1; ++si) {
    const PagedSeg g = segs[si];
    const int n = __ldg(a.s.kv_len + g.seq), q0 = __ldg(a.s.q_start + g.seq);
    const int nq = __ldg(a.s.q_start + g.seq + 1) - q0, rows = min(BR, nq * a.group - g.row0);
    const int* table = a.s.table + (size_t)g.seq * a.s.stride;
    const PagedSpan span = paged_span(g.row0, BR, a.group, n, nq, a.window, a.sinks, kGenKeys);
    __syncthreads();  // the previous segment's tiles are read
    fill_tile<T>(Q, BR, DP, D, wide_q, [&](int r) -> const T* {
      if (r >= rows) return nullptr;
      const int t = (g.row0 + r) / a.group, hq = g.head * a.group + (g.row0 + r) % a.group;
      return static_cast<const T*>(a.q) + (size_t)(q0 + t) * a.q_token + (size_t)hq * a.q_head;
    });
    int pos[RT];
    float m[RT], l[RT];
    float2 o[RT][NU][2];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      pos[i] = n - nq + (g.row0 + ty * RT + i) / a.group;
      m[i] = -INFINITY;
      l[i] = 0.0f;
#pragma unroll
      for (int u = 0; u < NU; ++u) o[i][u][0] = o[i][u][1] = make_float2(0.0f, 0.0f);
    }
    const int pa = n - nq + g.row0 / a.group, pb = n - nq + (g.row0 + rows - 1) / a.group;
    auto slot0 = [&](int it) { return (it < span.nsink ? it : span.first + it - span.nsink) * kGenKeys; };
    // slots that no row of the tile sees (past the last one, between the sinks
    // and the window) are zeros here, whatever their pages hold
    auto fill = [&](float* to, const void* pool, int it) {
      const int j0 = slot0(it);
      fill_tile<T>(to, kGenKeys, DP, D, wide, [&](int r) -> const T* {
        const int j = j0 + r;
        if (j > pb || (a.window && j <= pa - a.window && j >= a.sinks)) return nullptr;
        return static_cast<const T*>(pool) + paged_row(table, a.c, g.head, j);
      });
    };
    // K of the next tile is on its way while the values are summed, V of the
    // next one while its scores are computed
    if (g.it0 < g.it1) {
      fill(K, a.c.keys, g.it0);
      fill(V, a.c.values, g.it0);
    }
    for (int it = g.it0; it < g.it1; ++it) {
      const int j0 = slot0(it);
      filled<1>();
      __syncthreads();
      float s[RT][4];
      scores<RT>(Q, K, DP, ty, tx, s);
      __syncthreads();  // K is read
      if (it + 1 < g.it1) fill(K, a.c.keys, it + 1);
      // a tile that every row sees whole needs no masks
      const bool whole = j0 + kGenKeys - 1 <= pa &&
                         (!a.window || j0 > pb - a.window || j0 + kGenKeys <= a.sinks);
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        float mx = m[i];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          s[i][u] *= a.scale2;
          if (!whole && !paged_sees(pos[i], j0 + tx + 16 * u, a.window, a.sinks)) s[i][u] = -INFINITY;
          mx = fmaxf(mx, s[i][u]);
        }
        mx = half_max(mx);
        const float mu = mx == -INFINITY ? 0.0f : mx;  // nothing seen yet: all terms are 0
        const float f = exp2f(m[i] - mu);
        m[i] = mx;
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float p = exp2f(s[i][u] - mu);
          sum += p;
          // a slot that the row does not see is marked, so that its value
          // (infinite, or NaN) is skipped instead of multiplied by 0
          const bool see = whole || paged_sees(pos[i], j0 + tx + 16 * u, a.window, a.sinks);
          P[(ty * RT + i) * kPStride + tx + 16 * u] = see ? p : -1.0f;
        }
        l[i] = l[i] * f + half_sum(sum);
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            o[i][u][e].x *= f;
            o[i][u][e].y *= f;
          }
      }
      if (it + 1 < g.it1) filled<1>();
      else filled<0>();
      __syncthreads();  // V is there (the rows of P that a half-warp reads are its own)
      auto accumulate = [&](auto masked) {
#pragma unroll 1
        for (int k4 = 0; k4 < kGenKeys; k4 += 4) {
          float4 p[RT];
#pragma unroll
          for (int i = 0; i < RT; ++i) p[i] = *reinterpret_cast<const float4*>(P + (ty * RT + i) * kPStride + k4);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int u = 0; u < NU; ++u) {
              const int c4 = tx + 16 * u;
              if (c4 * 4 >= DP) continue;
              const float4 v = *reinterpret_cast<const float4*>(V + tile_at(k4 + kk, c4, DP));
#pragma unroll
              for (int i = 0; i < RT; ++i) {
                const float pk = kk == 0 ? p[i].x : kk == 1 ? p[i].y : kk == 2 ? p[i].z : p[i].w;
                if (decltype(masked)::value && pk < 0.0f) continue;
                const float2 p2 = make_float2(pk, pk);
                o[i][u][0] = ffma2(p2, make_float2(v.x, v.y), o[i][u][0]);
                o[i][u][1] = ffma2(p2, make_float2(v.z, v.w), o[i][u][1]);
              }
            }
        }
      };
      if (whole) accumulate(std::false_type{});
      else accumulate(std::true_type{});
      if (it + 1 < g.it1) {
        __syncthreads();  // V is read
        fill(V, a.c.values, it + 1);
      }
    }
    // copies to one place are in no order: those of a segment without tiles (its
    // rows) have to land before the next segment's start
    filled<0>();
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int r = ty * RT + i;
      if (r >= rows) continue;
      const int t = (g.row0 + r) / a.group, hq = g.head * a.group + (g.row0 + r) % a.group;
      const size_t at = (size_t)(q0 + t) * Hq + hq;
      const bool none = l[i] == 0.0f;
      const float inv = none ? 0.0f : 1.0f / l[i];
      if (tx == 0) {
        if (g.part >= 0) {
          float* ml = a.part_ml + ((size_t)g.part * BR + r) * 2;
          ml[0] = m[i];
          ml[1] = l[i];
        } else if (a.lse) {
          a.lse[at] = none ? -INFINITY : (m[i] + log2f(l[i])) * (float)M_LN2;
        }
      }
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = 4 * (tx + 16 * u) + e;
          if (c >= D) continue;
          const float x = e & 1 ? o[i][u][e >> 1].y : o[i][u][e >> 1].x;
          if (g.part >= 0) a.part_o[((size_t)g.part * BR + r) * D + c] = x;
          else static_cast<T*>(a.out)[at * D + c] = from_float<T>(none ? 0.0f : x * inv);
        }
    }
  }
}

// The same for more than 64 rows and head dims up to 128, in tiles of 128 rows by
// 128 slots: a thread's 8 x 8 scores (then 8 rows by 8 columns) take 16 loads of
// 16 bytes from shared memory per 256 multiply-adds, where the 4 x 4 of the tiles
// above take 8 per 64. K and V do not fit beside Q and P whole: they pass through
// a ring of four slabs (128 slots by 32 of the head dim, or 32 slots by the head
// dim), each loaded while the three before it are worked on, with one barrier per
// slab. The head dim is filled up to 64 or 128 so that offsets are constants.
// 500 f32 tokens on 1548, 32 heads of 128: 495 us, 30 TFLOP/s of the products, with
// 64-row tiles 639; 100 tokens on 1100, 8 heads: 51 against 63 in all; only a single
// tile is no faster (42 against 40). Bound by issue: two warps a scheduler, an
// instruction issued in half of the cycles, two thirds of them multiply-adds (loads
// from shared memory take a third of their pipe). Scalar multiply-adds for P V
// instead of paired ones: 4 % slower; two steps of the inner loop at once: 3 %.
template <typename T, int DP>
__global__ void __launch_bounds__(kGenThreads, 1) k_paged_attn_long(PagedAttn a, const PagedSeg* __restrict__ segs,
                                                                    const int* __restrict__ first, bool wide,
                                                                    bool wide_q) {
  constexpr int BR = kGenRowsLong, BK = kGenKeysLong, NU = DP / 64;
  extern __shared__ float4 sm4[];
  float* Q = reinterpret_cast<float*>(sm4);  // [BR][DP]
  float* P = Q + BR * DP;                    // [BR][kPStrideLong]
  float* ring = P + BR * kPStrideLong;       // kSlabs of kSlabFloats
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;  // rows ty + 16 i, slots tx + 16 u
  const int D = a.c.dim, Hq = a.c.heads * a.group;
  const int k_slabs = (D + 31) / 32, per = k_slabs + BK / 32;
  const int s1 = __ldg(first + blockIdx.x + 1);
  for (int si = __ldg(first + blockIdx.x); si < s1; ++si) {
    const PagedSeg g = segs[si];
    const int n = __ldg(a.s.kv_len + g.seq), q0 = __ldg(a.s.q_start + g.seq);
    const int nq = __ldg(a.s.q_start + g.seq + 1) - q0, rows = min(BR, nq * a.group - g.row0);
    const int* table = a.s.table + (size_t)g.seq * a.s.stride;
    const PagedSpan span = paged_span(g.row0, BR, a.group, n, nq, a.window, a.sinks, BK);
    __syncthreads();  // the previous segment's tiles are read
    fill_tile<T>(Q, BR, DP, D, wide_q, [&](int r) -> const T* {
      if (r >= rows) return nullptr;
      const int t = (g.row0 + r) / a.group, hq = g.head * a.group + (g.row0 + r) % a.group;
      return static_cast<const T*>(a.q) + (size_t)(q0 + t) * a.q_token + (size_t)hq * a.q_head;
    });
    float m[8], l[8];
    float2 o[8][NU][2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.0f;
#pragma unroll
      for (int u = 0; u < NU; ++u) o[i][u][0] = o[i][u][1] = make_float2(0.0f, 0.0f);
    }
    const int pa = n - nq + g.row0 / a.group, pb = n - nq + (g.row0 + rows - 1) / a.group;
    auto slot0 = [&](int it) { return (it < span.nsink ? it : span.first + it - span.nsink) * BK; };
    // the next slab of the segment into its place (nothing behind the last one,
    // but a group all the same, so that every step waits for the same number)
    int load_it = g.it0, load_x = 0, load_at = 0;
    auto load = [&] {
      if (load_it < g.it1) {
        const int j0 = slot0(load_it);
        // slots that no row of the tile sees are zeros here
        auto row = [&](const void* pool, int j) -> const T* {
          if (j > pb || (a.window && j <= pa - a.window && j >= a.sinks)) return nullptr;
          return static_cast<const T*>(pool) + paged_row(table, a.c, g.head, j);
        };
        float* to = ring + load_at * kSlabFloats;
        if (load_x < k_slabs) {
          const int d0 = 32 * load_x;
          fill_tile<T>(to, BK, 32, D - d0, wide, [&](int r) -> const T* {
            const T* p = row(a.c.keys, j0 + r);
            return p ? p + d0 : nullptr;
          });
        } else {
          const int r0 = j0 + 32 * (load_x - k_slabs);
          fill_tile<T>(to, 32, DP, D, wide, [&](int r) { return row(a.c.values, r0 + r); });
        }
        if (++load_x == per) {
          load_x = 0;
          ++load_it;
        }
      } else {
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
      load_at = (load_at + 1) % kSlabs;
    };
    int at = 0;
    auto next = [&] {  // the next slab to work on; the one before it makes room
      filled<kSlabs - 2>();
      __syncthreads();
      load();
      const float* p = ring + at * kSlabFloats;
      at = (at + 1) % kSlabs;
      return p;
    };
#pragma unroll 1
    for (int k = 0; k < kSlabs - 1; ++k) load();
    for (int it = g.it0; it < g.it1; ++it) {
      const int j0 = slot0(it);
      float s[8][8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int u = 0; u < 8; ++u) s[i][u] = 0.0f;
#pragma unroll 1
      for (int x = 0; x < k_slabs; ++x) {
        const float* kp = next() + tx * 32;
        const float* qp = Q + ty * DP + 32 * x;
#pragma unroll 1
        for (int c = 0; c < 8; ++c) {
          // (rows 16 apart have the same permutation of their pieces)
          const int qc = (c ^ (ty & 7)) << 2, kc = (c ^ (tx & 7)) << 2;
          float4 q[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) q[i] = *reinterpret_cast<const float4*>(qp + 16 * i * DP + qc);
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const float4 k = *reinterpret_cast<const float4*>(kp + 16 * u * 32 + kc);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              s[i][u] = fmaf(q[i].x, k.x, s[i][u]);
              s[i][u] = fmaf(q[i].y, k.y, s[i][u]);
              s[i][u] = fmaf(q[i].z, k.z, s[i][u]);
              s[i][u] = fmaf(q[i].w, k.w, s[i][u]);
            }
          }
        }
      }
      const bool whole = j0 + BK - 1 <= pa && (!a.window || j0 > pb - a.window || j0 + BK <= a.sinks);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        unsigned see = 0xffu;  // which of its eight slots the row sees
        if (!whole) {
          const int pos = n - nq + (g.row0 + ty + 16 * i) / a.group;
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (!paged_sees(pos, j0 + tx + 16 * u, a.window, a.sinks)) see ^= 1u << u;
        }
        float mx = m[i];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          s[i][u] = (see >> u & 1) ? s[i][u] * a.scale2 : -INFINITY;
          mx = fmaxf(mx, s[i][u]);
        }
        mx = half_max(mx);
        const float mu = mx == -INFINITY ? 0.0f : mx;  // nothing seen yet: all terms are 0
        const float f = exp2f(m[i] - mu);
        m[i] = mx;
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float p = exp2f(s[i][u] - mu);
          sum += p;
          // a slot that the row does not see is marked, see above
          P[(ty + 16 * i) * kPStrideLong + tx + 16 * u] = (see >> u & 1) ? p : -1.0f;
        }
        l[i] = l[i] * f + half_sum(sum);
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            o[i][u][e].x *= f;
            o[i][u][e].y *= f;
          }
      }
      __syncwarp();  // a half-warp reads its own rows of P only
      auto accumulate = [&](const float* v_slab, const float* pp, auto masked) {
#pragma unroll 1
        for (int k4 = 0; k4 < 32; k4 += 4) {
          float4 p[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) p[i] = *reinterpret_cast<const float4*>(pp + 16 * i * kPStrideLong + k4);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int u = 0; u < NU; ++u) {
              const float4 v = *reinterpret_cast<const float4*>(v_slab + tile_at(k4 + kk, tx + 16 * u, DP));
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float pk = kk == 0 ? p[i].x : kk == 1 ? p[i].y : kk == 2 ? p[i].z : p[i].w;
                if (decltype(masked)::value && pk < 0.0f) continue;
                const float2 p2 = make_float2(pk, pk);
                o[i][u][0] = ffma2(p2, make_float2(v.x, v.y), o[i][u][0]);
                o[i][u][1] = ffma2(p2, make_float2(v.z, v.w), o[i][u][1]);
              }
            }
        }
      };
#pragma unroll 1
      for (int x = 0; x < BK / 32; ++x) {
        const float* v = next();
        if (j0 + 32 * x > pb) continue;
        const float* pp = P + ty * kPStrideLong + 32 * x;
        if (whole) accumulate(v, pp, std::false_type{});
        else accumulate(v, pp, std::true_type{});
      }
    }
    filled<0>();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = ty + 16 * i;
      if (r >= rows) continue;
      const int t = (g.row0 + r) / a.group, hq = g.head * a.group + (g.row0 + r) % a.group;
      const size_t to = (size_t)(q0 + t) * Hq + hq;
      const bool none = l[i] == 0.0f;
      const float inv = none ? 0.0f : 1.0f / l[i];
      if (tx == 0) {
        if (g.part >= 0) {
          float* ml = a.part_ml + ((size_t)g.part * BR + r) * 2;
          ml[0] = m[i];
          ml[1] = l[i];
        } else if (a.lse) {
          a.lse[to] = none ? -INFINITY : (m[i] + log2f(l[i])) * (float)M_LN2;
        }
      }
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = 4 * (tx + 16 * u) + e;
          if (c >= D) continue;
          const float x = e & 1 ? o[i][u][e >> 1].y : o[i][u][e >> 1].x;
          if (g.part >= 0) a.part_o[((size_t)g.part * BR + r) * D + c] = x;
          else static_cast<T*>(a.out)[to * D + c] = from_float<T>(none ? 0.0f : x * inv);
        }
    }
  }
}

// Joins the parts of cut tiles: one warp per row, lanes over the columns. All
// it needs of the plan is read before it waits for the attention to end, and the
// first parts' sums and maxima are loaded together; bound by that one latency
// for short lists, and by reading the parts from L2 for long ones (4.4 us for one
// sequence of 2048 slots, most of it the wait; 16 for two chunks of 1000 tokens).
constexpr int kJoinWarps = 4, kJoinAhead = 4;
template <typename T, int NC>  // NC: columns per lane
__global__ void __launch_bounds__(32 * kJoinWarps) k_paged_join(PagedAttn a, const PagedJoin* __restrict__ joins,
                                                                int row_tile) {
  const PagedJoin g = joins[blockIdx.x];
  const int r = blockIdx.y * kJoinWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int D = a.c.dim;
  wait_for_previous();
  if (r >= g.rows) return;
  const size_t row = (size_t)g.part0 * row_tile + r;
  const float* ml = a.part_ml + row * 2;
  const float* po = a.part_o + row * D;
  float m = -INFINITY, l = 0.0f, acc[NC];
#pragma unroll
  for (int u = 0; u < NC; ++u) acc[u] = 0.0f;
  // as in the attention itself, over parts instead of tiles
  for (int p0 = 0; p0 < g.parts; p0 += kJoinAhead) {
    float2 y[kJoinAhead];
    float x[kJoinAhead][NC];
#pragma unroll
    for (int k = 0; k < kJoinAhead; ++k) {
      const size_t at = (size_t)(p0 + k) * row_tile;
      y[k] = make_float2(-INFINITY, 0.0f);
      if (p0 + k < g.parts) y[k] = *reinterpret_cast<const float2*>(ml + at * 2);
#pragma unroll
      for (int u = 0; u < NC; ++u) {
        x[k][u] = 0.0f;
        if (p0 + k < g.parts && lane + 32 * u < D) x[k][u] = po[at * D + lane + 32 * u];
      }
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < kJoinAhead; ++k) top = fmaxf(top, y[k].x);
    const float mu = top == -INFINITY ? 0.0f : top, f = exp2f(m - mu);
    m = top;
    l *= f;
#pragma unroll
    for (int u = 0; u < NC; ++u) acc[u] *= f;
#pragma unroll
    for (int k = 0; k < kJoinAhead; ++k) {
      if (p0 + k >= g.parts) continue;
      const float w = exp2f(y[k].x - mu);
      l = fmaf(w, y[k].y, l);
#pragma unroll
      for (int u = 0; u < NC; ++u) acc[u] = fmaf(w, x[k][u], acc[u]);
    }
  }
  const int t = (g.row0 + r) / a.group, hq = g.head * a.group + (g.row0 + r) % a.group;
  const size_t at = (size_t)(g.token0 + t) * (a.c.heads * a.group) + hq;
  const bool none = l == 0.0f;
  if (lane == 0 && a.lse) a.lse[at] = none ? -INFINITY : (m + log2f(l)) * (float)M_LN2;
  const float inv = none ? 0.0f : 1.0f / l;
#pragma unroll
  for (int u = 0; u < NC; ++u) {
    const int c = lane + 32 * u;
    if (c < D) static_cast<T*>(a.out)[at * D + c] = from_float<T>(none ? 0.0f : acc[u] * inv);
  }
}

// Attention weight of 64 slots of one (sequence, head): the column sums of
// the softmax over all rows that may see them, each row's sum known from lse.
// A CTA owns its slots and adds its rows in a fixed order: no atomics. Rows come
// in tiles of 16 RT: 16 where no sequence has more, 128 otherwise (f32, 500 tokens
// on 1548 with 32 heads of 128: 336 us, 356 in tiles of 64 rows; of 256: 686 and
// 898). Bound as the attention itself: shared-memory loads and multiply-adds.
template <typename T, int RT>
__global__ void __launch_bounds__(kGenThreads) k_paged_weights(PagedAttn a, const PagedSlots* __restrict__ tiles,
                                                               float decay, int DP, bool wide, bool wide_q) {
  constexpr int BR = 16 * RT;
  extern __shared__ float4 sm4[];
  float* K = reinterpret_cast<float*>(sm4);  // [64][DP]
  float* Q = K + kGenKeys * DP;              // [BR][DP]
  __shared__ float lse2[BR];
  __shared__ float sums[16][kGenKeys];
  const PagedSlots g = tiles[blockIdx.x];
  const int h = blockIdx.y, tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int D = a.c.dim, Hq = a.c.heads * a.group;
  const int n = __ldg(a.s.kv_len + g.seq), q0 = __ldg(a.s.q_start + g.seq);
  const int nq = __ldg(a.s.q_start + g.seq + 1) - q0;
  const int* table = a.s.table + (size_t)g.seq * a.s.stride;
  const int j0 = g.slot0, j1 = min(j0 + kGenKeys, n);
  fill_tile<T>(K, kGenKeys, DP, D, wide, [&](int r) -> const T* {
    return j0 + r < j1 ? static_cast<const T*>(a.c.keys) + paged_row(table, a.c, h, j0 + r) : nullptr;
  });
  // tokens that may see any of the slots: from slot j0 on, to the window's end
  // behind the last slot unless some of the slots are sinks
  const int ta = max(0, j0 - (n - nq));
  const int tb = (a.window && j0 >= a.sinks) ? (int)min((long long)nq, (long long)j1 - 1 + a.window - (n - nq)) : nq;
  float w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int row0 = ta * a.group; row0 < tb * a.group; row0 += BR) {
    const int rows = min(BR, tb * a.group - row0);
    __syncthreads();
    fill_tile<T>(Q, BR, DP, D, wide_q, [&](int r) -> const T* {
      if (r >= rows) return nullptr;
      const int t = (row0 + r) / a.group, hq = h * a.group + (row0 + r) % a.group;
      return static_cast<const T*>(a.q) + (size_t)(q0 + t) * a.q_token + (size_t)hq * a.q_head;
    });
    for (int r = tid; r < rows; r += kGenThreads) {
      const int t = (row0 + r) / a.group, hq = h * a.group + (row0 + r) % a.group;
      lse2[r] = a.lse[(size_t)(q0 + t) * Hq + hq] * (float)M_LOG2E;
    }
    filled<0>();
    __syncthreads();
    float s[RT][4];
    scores<RT>(Q, K, DP, ty, tx, s);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int r = ty * RT + i;
      if (r >= rows) continue;
      const float z = lse2[r];
      if (z == -INFINITY) continue;  // a row that sees nothing
      const int pos = n - nq + (row0 + r) / a.group;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (paged_sees(pos, j0 + tx + 16 * u, a.window, a.sinks)) w[u] += exp2f(fmaf(s[i][u], a.scale2, -z));
    }
  }
  filled<0>();  // K, where no row sees the slots
#pragma unroll
  for (int u = 0; u < 4; ++u) sums[ty][tx + 16 * u] = w[u];
  __syncthreads();
  if (tid < j1 - j0) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += sums[i][tid];
    const int j = j0 + tid;
    const int page = __ldg(table + (j >> a.c.page_shift));
    float* p = a.c.weights + (((size_t)page * a.c.heads + h) << a.c.page_shift) + (j & ((1 << a.c.page_shift) - 1));
    *p = decay == 0.0f ? t : fmaf(decay, *p, t);
  }
}

// rows may be read 16 bytes at a time
template <typename T>
bool wide_rows(const PagedAttn& a) {
  return a.c.dim * sizeof(T) % 16 == 0;
}
template <typename T>
bool wide_query(const PagedAttn& a) {
  return a.c.dim * sizeof(T) % 16 == 0 && (a.q_token | a.q_head) * sizeof(T) % 16 == 0 && aligned(a.q, 16);
}

template <typename T, int RT, int NU>
cudaError_t attn_launch(const PagedAttn& a, const PagedWork& w, cudaStream_t st) {
  const int DP = (a.c.dim + 31) / 32 * 32;
  auto bytes = [](size_t dp) { return ((16 * RT + 2 * kGenKeys) * dp + 16 * RT * kPStride) * sizeof(float); };
  const size_t smem = bytes(DP);
  auto kern = k_paged_attn<T, RT, NU>;
  static OptInOnce done;
  cudaError_t e = opt_in_once(done, kern, bytes(64 * NU));
  if (e != cudaSuccess) return e;
  kern<<<w.ctas, kGenThreads, smem, st>>>(a, w.segs, w.first, DP, wide_rows<T>(a), wide_query<T>(a));
  note_launches(1);
  return cudaGetLastError();
}

template <typename T, int DP>
cudaError_t attn_long_launch(const PagedAttn& a, const PagedWork& w, cudaStream_t st) {
  constexpr size_t smem = ((size_t)kGenRowsLong * (DP + kPStrideLong) + kSlabs * kSlabFloats) * sizeof(float);
  auto kern = k_paged_attn_long<T, DP>;
  static OptInOnce done;
  cudaError_t e = opt_in_once(done, kern, smem);
  if (e != cudaSuccess) return e;
  kern<<<w.ctas, kGenThreads, smem, st>>>(a, w.segs, w.first, wide_rows<T>(a), wide_query<T>(a));
  note_launches(1);
  return cudaGetLastError();
}

template <typename T>
cudaError_t attn_typed(const PagedAttn& a, const PagedWork& w, cudaStream_t st) {
  if (w.row_tile == kGenRowsLong)
    return a.c.dim <= 64 ? attn_long_launch<T, 64>(a, w, st) : attn_long_launch<T, kGenDimLong>(a, w, st);
  const int nu = (a.c.dim + 63) / 64;
  if (w.row_tile == kGenRows)
    return nu == 1 ? attn_launch<T, 4, 1>(a, w, st) : nu == 2 ? attn_launch<T, 4, 2>(a, w, st)
                                                              : attn_launch<T, 4, 4>(a, w, st);
  return nu == 1 ? attn_launch<T, 1, 1>(a, w, st) : nu == 2 ? attn_launch<T, 1, 2>(a, w, st)
                                                            : attn_launch<T, 1, 4>(a, w, st);
}

template <typename T>
cudaError_t join_typed(const PagedAttn& a, const PagedWork& w, cudaStream_t st) {
  const dim3 grid((unsigned)w.joins_n, (unsigned)((w.row_tile + kJoinWarps - 1) / kJoinWarps));
  note_launches(1);
  auto kern = a.c.dim <= 64 ? k_paged_join<T, 2> : a.c.dim <= 128 ? k_paged_join<T, 4> : k_paged_join<T, 8>;
  return launch_behind(kern, grid, 32 * kJoinWarps, 0, st, a, w.joins, w.row_tile);
}

template <typename T, int RT>
cudaError_t weights_launch(const PagedAttn& a, const PagedSlots* tiles, size_t ntiles, float decay, cudaStream_t st) {
  const int DP = (a.c.dim + 31) / 32 * 32;
  auto bytes = [](size_t dp) { return (16 * RT + kGenKeys) * dp * sizeof(float); };
  const size_t smem = bytes(DP);
  auto kern = k_paged_weights<T, RT>;
  static OptInOnce done;
  cudaError_t e = opt_in_once(done, kern, bytes(kGenDimMost));
  if (e != cudaSuccess) return e;
  kern<<<dim3((unsigned)ntiles, (unsigned)a.c.heads), kGenThreads, smem, st>>>(a, tiles, decay, DP, wide_rows<T>(a),
                                                                              wide_query<T>(a));
  note_launches(1);
  return cudaGetLastError();
}

template <typename T>
cudaError_t weights_typed(const PagedAttn& a, const PagedSlots* tiles, size_t ntiles, bool few_rows, float decay,
                          cudaStream_t st) {
  return few_rows ? weights_launch<T, 1>(a, tiles, ntiles, decay, st)
                  : weights_launch<T, 8>(a, tiles, ntiles, decay, st);
}

}  // namespace

cudaError_t launch_paged_attn_generic(const PagedAttn& a, const PagedWork& w, cudaStream_t st) {
  if (w.ctas == 0) return cudaSuccess;
  if (a.c.dtype == KVF_IN_F32) return attn_typed<float>(a, w, st);
  if (a.c.dtype == KVF_IN_F16) return attn_typed<__half>(a, w, st);
  return attn_typed<__nv_bfloat16>(a, w, st);
}

cudaError_t launch_paged_join(const PagedAttn& a, const PagedWork& w, cudaStream_t st) {
  if (w.joins_n == 0) return cudaSuccess;
  if (a.c.dtype == KVF_IN_F32) return join_typed<float>(a, w, st);
  if (a.c.dtype == KVF_IN_F16) return join_typed<__half>(a, w, st);
  return join_typed<__nv_bfloat16>(a, w, st);
}

cudaError_t launch_paged_weights_generic(const PagedAttn& a, const PagedSlots* tiles, size_t ntiles, bool few_rows,
                                         float decay, cudaStream_t st) {
  if (ntiles == 0) return cudaSuccess;
  if (a.c.dtype == KVF_IN_F32) return weights_typed<float>(a, tiles, ntiles, few_rows, decay, st);
  if (a.c.dtype == KVF_IN_F16) return weights_typed<__half>(a, tiles, ntiles, few_rows, decay, st);
  return weights_typed<__nv_bfloat16>(a, tiles, ntiles, few_rows, decay, st);
}

}  // namespace kvf
