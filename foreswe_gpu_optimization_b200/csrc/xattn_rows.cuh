// Cross attention for a few query rows per key head (G * Nq <= 8: single tokens, a handful of sites): both types, one
// pass over K and V forward, and one over K, V, dK and dV backward. In fp32 also for up to 32 queries per head
// forward, 8 rows per CTA, and for the queries behind the last whole tile where there are as few.
//
// Such calls are bound by reading K and V; a tile of 64 or 128 query rows would be mostly padding. 16 lanes hold one
// key's row of K and V (4 columns per lane and 64 of the head dim) straight from global memory, no shared memory
// between; a half-warp takes KB keys at a time. The R * KB scores of a step are summed across the 16 lanes by a transposing
// reduction (each round halves the values a lane still carries), so that every lane ends with one (row, key) score and
// works out its exponential, its dropout bit and its dS; shuffles hand them back for the second products. The rows of Q
// and dO (the few there are) stay in shared memory, O and dQ in registers, all sums in fp32.
// Measured: fp32, 32 x 16 heads, 1 query, 4096 keys of 128: 331 us (6.5 TB/s); 8 queries, 64 x 16 heads, 4096 keys of
// 64: 702 us (3.1 TB/s: past 4 rows the shuffles and products of a key take longer than its bytes). bf16, 1 x 16 heads,
// 512 keys of 128: 11 us, latency. fp32 forward and backward, 64 x 15 / 5 heads, 2 queries, 11785 keys of 64 with
// dropout: 2.3 ms for 3.9 GB. The next step's rows are fetched during the products (8 rows, 64 x 16 heads, bf16: 694 ->
// 489 us), except backward at 8 rows and head dims above 64, whose registers are full with dQ.
// Backward needs no scratch: dK and dV of a key are complete within its half-warp, and dS goes to memory only for the
// bias table's gradient.
#pragma once
#include <type_traits>

#include "sm100.cuh"
#include "xattn_common.cuh"

namespace geoattn {

constexpr int kRowThreads = 256, kRowWarps = kRowThreads / 32, kRowLanes = 16;
constexpr int kRowMax = 8;  // query rows of a key head's group

template <int NV, int R>
struct RowCfg {
  static constexpr int DP = NV * 64;
  static constexpr int KB = NV == 1 && R < 8 ? 4 : 2;  // keys of a half-warp's step
  static constexpr int NVAL = R * KB;
  static constexpr int LOG = NVAL == 2 ? 1 : NVAL == 4 ? 2 : NVAL == 8 ? 3 : 4;
  static constexpr int REP = kRowLanes >> LOG;  // lanes that end with the same value
  static constexpr int STEP = 2 * kRowWarps * KB;
  static_assert(NVAL >= 2 && NVAL <= kRowLanes, "");
};

// Four columns of a row, as two pairs of fp32.
struct Cols {
  uint64_t x[2];
};
__device__ __forceinline__ Cols cols_of(float4 v) { return {{f2(v.x, v.y), f2(v.z, v.w)}}; }

template <class E>
__device__ __forceinline__ bool row_vec(const XTensor& t) {
  return (reinterpret_cast<uintptr_t>(t.p) & (4 * sizeof(E) - 1)) == 0 && t.s[0] % 4 == 0 && t.s[1] % 4 == 0 &&
         t.s[2] % 4 == 0;
}
template <class E>
__device__ __forceinline__ E* row_at(const XTensor& t, int b, int h, int i) {
  return reinterpret_cast<E*>(t.p) + b * t.s[0] + h * t.s[1] + i * t.s[2];
}
// Four columns as they lie in memory.
template <class E>
using Raw4 = std::conditional_t<sizeof(E) == 4, float4, uint2>;
__device__ __forceinline__ float4 widen(float4 v) { return v; }
__device__ __forceinline__ float4 widen(uint2 w) {
  return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
                     __uint_as_float(w.y & 0xFFFF0000u));
}
template <class E>
__device__ __forceinline__ Raw4<E> raw4(const E* row, int d, int D, bool vec) {
  if (vec && d + 4 <= D) return *reinterpret_cast<const Raw4<E>*>(row + d);
  Raw4<E> v{};
  E* e = reinterpret_cast<E*>(&v);
#pragma unroll
  for (int x = 0; x < 4; ++x)
    if (d + x < D) e[x] = row[d + x];
  return v;
}
template <class E>
__device__ __forceinline__ float4 load4(const E* row, int d, int D, bool vec) {
  return widen(raw4(row, d, D, vec));
}
template <class E>
__device__ __forceinline__ void store4(E* row, int d, int D, bool vec, float4 v) {
  if (vec && d + 4 <= D) {
    if constexpr (sizeof(E) == 4) {
      *reinterpret_cast<float4*>(row + d) = v;
    } else {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
      *reinterpret_cast<uint2*>(row + d) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
  } else {
    if (d < D) row[d] = from_f<E>(v.x);
    if (d + 1 < D) row[d + 1] = from_f<E>(v.y);
    if (d + 2 < D) row[d + 2] = from_f<E>(v.z);
    if (d + 3 < D) row[d + 3] = from_f<E>(v.w);
  }
}

// The sums over 16 lanes of N values: lane l ends with value l >> (4 - log2 N).
template <int N>
__device__ __forceinline__ float transpose_sum(float (&v)[N], int lane) {
  int w = 8;
#pragma unroll
  for (int n = N; n > 1; n /= 2, w /= 2) {
    const bool up = lane & w;
#pragma unroll
    for (int x = 0; x < n / 2; ++x) {
      const float mine = up ? v[x + n / 2] : v[x], other = up ? v[x] : v[x + n / 2];
      v[x] = mine + __shfl_xor_sync(0xffffffffu, other, w);
    }
  }
#pragma unroll
  for (int k = 8 / N; k > 0; k /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], k);
  return v[0];
}

// A half-warp's next KB keys on their way from memory: fetched while the step before is worked on. Absent keys are
// zeros, whatever lies there.
template <class E, int NV, int KB>
struct KeyStep {
  Raw4<E> k[KB][NV], v[KB][NV];
  uint32_t live;  // bit y: key y exists

  __device__ __forceinline__ void get(const XParams& p, const E* K, const E* V, int b, int n, int j0, int lane, bool vk,
                                      bool vv) {
    live = 0;
#pragma unroll
    for (int y = 0; y < KB; ++y) live |= (uint32_t)key_live(p, b, j0 + y, n) << y;
    const bool wide = vk && vv && p.D % 4 == 0;
#pragma unroll
    for (int y = 0; y < KB; ++y)
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        const int d = (c * kRowLanes + lane) * 4;
        k[y][c] = v[y][c] = Raw4<E>{};
        if ((live >> y & 1) && d < p.D) {
          const E *kr = K + (j0 + y) * p.k.s[2], *vr = V + (j0 + y) * p.v.s[2];
          if (wide) {
            k[y][c] = *reinterpret_cast<const Raw4<E>*>(kr + d);
            v[y][c] = *reinterpret_cast<const Raw4<E>*>(vr + d);
          } else {
            k[y][c] = raw4(kr, d, p.D, vk);
            v[y][c] = raw4(vr, d, p.D, vv);
          }
        }
      }
  }
};

// Products of the half-warp's KB keys with the R rows in shared memory, summed over the head dim.
template <int NV, int R, int KB>
__device__ __forceinline__ float row_scores(const float4 (*rows)[NV * kRowLanes], const Cols (&k)[KB][NV], int lane) {
  float v[R * KB];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    Cols q[NV];
#pragma unroll
    for (int c = 0; c < NV; ++c) q[c] = cols_of(rows[r][c * kRowLanes + lane]);
#pragma unroll
    for (int y = 0; y < KB; ++y) {
      uint64_t s = mul2(q[0].x[0], k[y][0].x[0]);
      s = fma2(q[0].x[1], k[y][0].x[1], s);
#pragma unroll
      for (int c = 1; c < NV; ++c) s = fma2(q[c].x[1], k[y][c].x[1], fma2(q[c].x[0], k[y][c].x[0], s));
      float e, o;
      unf2(s, e, o);
      v[r * KB + y] = e + o;
    }
  }
  return transpose_sum(v, lane);
}

// Adds the warps' sums of R rows; warp 0 (both half-warps) ends with the total. Called by every thread.
template <int NV, int R>
__device__ __forceinline__ void join_warps(Cols (&acc)[R][NV], float4 (*slot)[R][NV * kRowLanes], int warp, int lane,
                                           int half) {
#pragma unroll
  for (int w = kRowWarps / 2; w; w /= 2) {
    __syncthreads();  // the slots' last readers are done
    if (half == 0 && warp >= w && warp < 2 * w) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < NV; ++c) {
          float4 v;
          unf2(acc[r][c].x[0], v.x, v.y);
          unf2(acc[r][c].x[1], v.z, v.w);
          slot[warp - w][r][c * kRowLanes + lane] = v;
        }
    }
    __syncthreads();
    if (warp < w) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < NV; ++c) {
          const Cols v = cols_of(slot[warp][r][c * kRowLanes + lane]);
          acc[r][c].x[0] = add2(acc[r][c].x[0], v.x[0]);
          acc[r][c].x[1] = add2(acc[r][c].x[1], v.x[1]);
        }
    }
  }
}
template <int NV, int R>
__device__ __forceinline__ void join_halves(Cols (&acc)[R][NV]) {
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        acc[r][c].x[e] = add2(acc[r][c].x[e], __shfl_xor_sync(0xffffffffu, (unsigned long long)acc[r][c].x[e], 16));
}

// Keys of split `s`: whole steps, so that a split's bounds do not depend on the lengths.
__device__ __forceinline__ void row_range(const XParams& p, int splits, int s, int& k0, int& k1) {
  const int per = ((p.Nk + splits - 1) / splits + 63) / 64 * 64;
  const long long a = (long long)per * s, e = a + per;
  k0 = a < p.Nk ? (int)a : p.Nk;
  k1 = e < p.Nk ? (int)e : p.Nk;
}

template <class E, int NV, int R>
__device__ __forceinline__ void stage_rows(const XParams& p, const XTensor& t, int b, int kh, int first,
                                           float4 (*dst)[NV * kRowLanes]) {
  const bool vec = row_vec<E>(t);
  for (int x = threadIdx.x; x < R * NV * kRowLanes; x += kRowThreads) {
    const int r = x / (NV * kRowLanes), d = x % (NV * kRowLanes) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    const int g = first + r;  // row of the group
    if (g < p.G * p.rq)
      v = load4<E>(row_at<const E>(t, b, kh * p.G + g / p.rq, p.q0 + g % p.rq), d, p.D, vec);
    dst[r][d / 4] = v;
  }
}
// Bias tables of the kRowMax heads from `first` on, as far as they belong to the group.
__device__ __forceinline__ void stage_tables(const XParams& p, int kh, int first, float (*tab)[kMaxBuckets]) {
  if (p.ids)
    for (int x = threadIdx.x; x < kRowMax * kMaxBuckets; x += kRowThreads) {
      const int g = x / kMaxBuckets, t = x % kMaxBuckets;
      if (first + g < p.G) tab[g][t] = table_log2(p, kh * p.G + first + g, t);
    }
}

// One CTA per (R rows of the group, batch, key head, key split).
template <class E, int NV, int R>
__global__ void __launch_bounds__(kRowThreads) xattn_rows_fwd_kernel(const XParams p) {
  using C = RowCfg<NV, R>;
  constexpr int KB = C::KB;
  __shared__ float4 qs[R][NV * kRowLanes];
  __shared__ float4 slot[kRowWarps / 2][R][NV * kRowLanes];
  __shared__ float tab[kRowMax][kMaxBuckets];
  __shared__ float sm_m[kRowWarps][R], sm_l[kRowWarps][R];
  const int rows = p.G * p.rq, parts = (rows + R - 1) / R, first = blockIdx.x % parts * R;
  const int units = p.B * p.Hkv, unit = blockIdx.x / parts % units, split = blockIdx.x / parts / units;
  const int b = unit / p.Hkv, kh = unit % p.Hkv;
  const int warp = threadIdx.x / 32, half = threadIdx.x / 16 % 2, lane = threadIdx.x % 16;
  const int idx = lane / C::REP, y0 = idx % KB, r0 = idx / KB;  // this lane's key of the step and row
  const bool row = first + r0 < rows;
  const int hg = row ? (first + r0) / p.rq : 0, h = kh * p.G + hg, i = p.q0 + (row ? (first + r0) % p.rq : 0);
  if (blockIdx.x + threadIdx.x == 0) *p.status = kDevOk;
  const AttnDrop drop = attn_drop(p.rng, p.drop_thr, p.drop_scale);
  const int n = key_count(p, b);
  int k0, k1;
  row_range(p, p.splits, split, k0, k1);
  k1 = min(k1, n);
  stage_rows<E, NV, R>(p, p.q, b, kh, first, qs);
  stage_tables(p, kh, first / p.rq, tab);
  __syncthreads();
  const E *K = row_at<const E>(p.k, b, kh, 0), *V = row_at<const E>(p.v, b, kh, 0);
  const bool vk = row_vec<E>(p.k), vv = row_vec<E>(p.v);
  const auto from = [&](int r) { return half * 16 + r * KB * C::REP; };  // lane of (row r, key 0)
  float m = -INFINITY, l = 0.f;  // of this lane's row; l over this lane's keys
  Cols acc[R][NV] = {};
  KeyStep<E, NV, KB> step;
  const int j_first = k0 + (warp * 2 + half) * KB;
  step.get(p, K, V, b, k1, j_first, lane, vk, vv);

  for (int j0 = j_first; j0 - half * KB < k1; j0 += C::STEP) {  // the same number of steps in both halves
    Cols k[KB][NV], v[KB][NV];
#pragma unroll
    for (int y = 0; y < KB; ++y)
#pragma unroll
      for (int c = 0; c < NV; ++c) k[y][c] = cols_of(widen(step.k[y][c])), v[y][c] = cols_of(widen(step.v[y][c]));
    const uint32_t there = step.live;
    step.get(p, K, V, b, k1, j0 + C::STEP, lane, vk, vv);
    const int j = j0 + y0;
    const bool live = row && (there >> y0 & 1);
    float x = row_scores<NV, R, KB>(qs, k, lane) * p.scale_log2;
    if (p.ids && live) {
      const int id = p.ids[i * p.ids_ld + j];
      x += id < p.T ? tab[hg - first / p.rq][id] : -INFINITY;
    }
    if (!live) x = -INFINITY;
    float top = x;
#pragma unroll
    for (int w = C::REP; w < C::REP * KB; w *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    // the maximum moves only when it grows by 2^8: a weight stays below 2^8 and the sums far from overflow
    if (__any_sync(0xffffffffu, top > m + 8.f)) {
      const float next = fmaxf(m, top), f = next == -INFINITY ? 1.f : xex2(m - next);
      m = next;
      l *= f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float g = __shfl_sync(0xffffffffu, f, from(r));
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e) acc[r][c].x[e] = mul2(acc[r][c].x[e], f2(g, g));
      }
    }
    float pr = xex2(x - (m == -INFINITY ? 0.f : m));  // m = -inf: x is -inf (or NaN, which stays)
    l += pr;
    if (drop.thr && !(drop.keep8(i, j >> 3, b * p.H + h) >> (j & 7) & 1)) pr = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int y = 0; y < KB; ++y) {
        const float a = __shfl_sync(0xffffffffu, pr, from(r) + y * C::REP);
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e) acc[r][c].x[e] = fma2(f2(a, a), v[y][c].x[e], acc[r][c].x[e]);
      }
  }

  // join the lanes' sums, then the sixteen half-warps
#pragma unroll
  for (int w = C::REP; w < C::REP * KB; w *= 2) l += __shfl_xor_sync(0xffffffffu, l, w);
  float top = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
  float ls = l * (m == -INFINITY ? 0.f : xex2(m - top));
  ls += __shfl_xor_sync(0xffffffffu, ls, 16);
  if (half == 0 && idx % KB == 0 && lane % C::REP == 0) sm_m[warp][r0] = top, sm_l[warp][r0] = ls;
  __syncthreads();
  top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, sm_m[w][r0]);
  const float f = m == -INFINITY ? 0.f : xex2(m - top);
  ls = 0.f;
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) ls += sm_l[w][r0] * (sm_m[w][r0] == -INFINITY ? 0.f : xex2(sm_m[w][r0] - top));
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float g = __shfl_sync(0xffffffffu, f, from(r));
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) acc[r][c].x[e] = mul2(acc[r][c].x[e], f2(g, g));
  }
  join_halves<NV, R>(acc);
  join_warps<NV, R>(acc, slot, warp, lane, half);
  if (warp) return;
  const bool vo = row_vec<E>(p.o);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float lr = __shfl_sync(0xffffffffu, ls, from(r)), mr = __shfl_sync(0xffffffffu, top, from(r));
    if (first + r >= rows || half) continue;
    const int hr = kh * p.G + (first + r) / p.rq, ir = p.q0 + (first + r) % p.rq;
    const long long at = (long long)(b * p.H + hr) * p.Nq + ir;
    const float inv = p.splits > 1 ? 1.f : lr == 0.f ? 0.f : (p.drop_thr ? p.drop_scale : 1.f) / lr;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const int d = (c * kRowLanes + lane) * 4;
      float4 o;
      unf2(acc[r][c].x[0], o.x, o.y);
      unf2(acc[r][c].x[1], o.z, o.w);
      o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
      if (p.splits > 1)
        store4(p.part_o + ((long long)split * p.B * p.H * p.Nq + at) * p.D, d, p.D, p.D % 4 == 0, o);
      else
        store4(row_at<E>(p.o, b, hr, ir), d, p.D, vo, o);
    }
    if (lane == 0) {
      if (p.splits > 1)
        reinterpret_cast<float2*>(p.part_ml)[(long long)split * p.B * p.H * p.Nq + at] = make_float2(mr, lr);
      else if (p.stats)
        p.stats[at] = row_stats(mr, lr);
    }
  }
}

// One CTA per (unit of the launch, key split). Writes every dK and dV row of its keys (zeros for absent ones).
template <class E, int NV, int R>
__global__ void __launch_bounds__(kRowThreads) xattn_rows_bwd_kernel(const XParams p, int units) {
  using C = RowCfg<NV, R>;
  constexpr int KB = C::KB;
  constexpr bool AHEAD = NV == 1 || R < 8;  // keys of the next step in registers, where they fit
  __shared__ float4 qs[R][NV * kRowLanes], gs[R][NV * kRowLanes];
  __shared__ float4 slot[kRowWarps / 2][R][NV * kRowLanes];
  __shared__ float tab[kRowMax][kMaxBuckets];
  __shared__ float delta[R];
  const int ul = blockIdx.x % units, split = blockIdx.x / units, unit = p.u0 + ul;
  const int b = unit / p.Hkv, kh = unit % p.Hkv;
  const int warp = threadIdx.x / 32, half = threadIdx.x / 16 % 2, lane = threadIdx.x % 16;
  const int idx = lane / C::REP, y0 = idx % KB, r0 = idx / KB;
  const bool row = r0 < p.G * p.Nq;
  const int h = kh * p.G + (row ? r0 / p.Nq : 0), i = row ? r0 % p.Nq : 0;
  if (blockIdx.x + threadIdx.x == 0) *p.status = kDevOk;
  const AttnDrop drop = attn_drop(p.rng, p.drop_thr, p.drop_scale);
  const int n = key_count(p, b);
  int k0, k1;
  row_range(p, p.splits, split, k0, k1);
  stage_rows<E, NV, R>(p, p.q, b, kh, 0, qs);
  stage_rows<E, NV, R>(p, p.dout, b, kh, 0, gs);
  stage_tables(p, kh, 0, tab);
  __syncthreads();
  {
    const bool vo = row_vec<E>(p.o);
    for (int r = threadIdx.x / 16; r < R; r += kRowThreads / 16) {  // warp-uniform: R = 1 leaves half a warp idle
      float s = 0.f;
      if (r < p.G * p.Nq) {
        const E* O = row_at<const E>(p.o, b, kh * p.G + r / p.Nq, r % p.Nq);
#pragma unroll
        for (int c = 0; c < NV; ++c) {
          const float4 o = load4(O, (c * kRowLanes + lane) * 4, p.D, vo), g = gs[r][c * kRowLanes + lane];
          s = fmaf(o.x, g.x, fmaf(o.y, g.y, fmaf(o.z, g.z, fmaf(o.w, g.w, s))));
        }
      }
      const uint32_t lanes = 0xFFFFu << half * 16;
#pragma unroll
      for (int w = 8; w; w /= 2) s += __shfl_xor_sync(lanes, s, w);
      if (lane == 0) delta[r] = s;
    }
  }
  __syncthreads();
  const float2 st = row ? p.stats[(long long)(b * p.H + h) * p.Nq + i] : make_float2(0.f, 0.f);
  const float dl = delta[r0];
  const E *K = row_at<const E>(p.k, b, kh, 0), *V = row_at<const E>(p.v, b, kh, 0);
  E *dK = row_at<E>(p.dk, b, kh, 0), *dV = row_at<E>(p.dv, b, kh, 0);
  const bool vk = row_vec<E>(p.k), vv = row_vec<E>(p.v), vdk = row_vec<E>(p.dk), vdv = row_vec<E>(p.dv);
  E* ds_out = reinterpret_cast<E*>(p.ds) + (long long)(ul * p.G + (row ? r0 / p.Nq : 0)) * p.nkp * p.nqp + i;
  Cols acc[R][NV] = {};  // dQ
  const int kl = min(k1, n);
  KeyStep<E, NV, KB> step;
  const int j_first = k0 + (warp * 2 + half) * KB;
  if (AHEAD) step.get(p, K, V, b, kl, j_first, lane, vk, vv);

  for (int j0 = j_first; j0 - half * KB < k1; j0 += C::STEP) {  // the same number of steps in both halves
    if (!AHEAD) step.get(p, K, V, b, kl, j0, lane, vk, vv);
    Cols k[KB][NV], v[KB][NV];
#pragma unroll
    for (int y = 0; y < KB; ++y)
#pragma unroll
      for (int c = 0; c < NV; ++c) k[y][c] = cols_of(widen(step.k[y][c])), v[y][c] = cols_of(widen(step.v[y][c]));
    const uint32_t there = step.live;
    if (AHEAD) step.get(p, K, V, b, kl, j0 + C::STEP, lane, vk, vv);
    const int j = j0 + y0;
    const bool live = row && (there >> y0 & 1);
    float x = row_scores<NV, R, KB>(qs, k, lane) * p.scale_log2;
    float g = row_scores<NV, R, KB>(gs, v, lane);
    if (p.ids && live) {
      const int id = p.ids[i * p.ids_ld + j];
      x += id < p.T ? tab[r0 / p.Nq][id] : -INFINITY;
    }
    const float pr = live ? xex2(x - st.x) * st.y : 0.f;
    float a = pr;
    if (drop.thr) {
      const bool keep = drop.keep8(i, j >> 3, b * p.H + h) >> (j & 7) & 1;
      a = keep ? pr * drop.scale : 0.f;
      g = keep ? g * drop.scale : 0.f;
    }
    const float ds = live ? pr * (g - dl) : 0.f;
    if (p.ids && row && j < kl && lane % C::REP == 0)
      ds_out[(long long)(j / 64) * (p.nqp / 8) * 512 + j % 64 * 8] = from_f<E>(ds);
    Cols dk[KB][NV] = {}, dv[KB][NV] = {};
#pragma unroll
    for (int r = 0; r < R; ++r) {
      Cols q[NV], go[NV];
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        q[c] = cols_of(qs[r][c * kRowLanes + lane]);
        go[c] = cols_of(gs[r][c * kRowLanes + lane]);
      }
#pragma unroll
      for (int y = 0; y < KB; ++y) {
        const int src = half * 16 + (r * KB + y) * C::REP;
        const float s1 = __shfl_sync(0xffffffffu, ds, src), a1 = __shfl_sync(0xffffffffu, a, src);
        const uint64_t s2 = f2(s1, s1), a2 = f2(a1, a1);
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            dk[y][c].x[e] = fma2(s2, q[c].x[e], dk[y][c].x[e]);
            dv[y][c].x[e] = fma2(a2, go[c].x[e], dv[y][c].x[e]);
            acc[r][c].x[e] = fma2(s2, k[y][c].x[e], acc[r][c].x[e]);
          }
      }
    }
#pragma unroll
    for (int y = 0; y < KB; ++y) {
      if (j0 + y >= k1) continue;
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        const int d = (c * kRowLanes + lane) * 4;
        float4 o;
        unf2(dk[y][c].x[0], o.x, o.y);
        unf2(dk[y][c].x[1], o.z, o.w);
        o = make_float4(o.x * p.scale, o.y * p.scale, o.z * p.scale, o.w * p.scale);
        store4(dK + (j0 + y) * p.dk.s[2], d, p.D, vdk, o);
        unf2(dv[y][c].x[0], o.x, o.y);
        unf2(dv[y][c].x[1], o.z, o.w);
        store4(dV + (j0 + y) * p.dv.s[2], d, p.D, vdv, o);
      }
    }
  }
  join_halves<NV, R>(acc);
  join_warps<NV, R>(acc, slot, warp, lane, half);
  if (warp || half) return;
  const bool vq = row_vec<E>(p.dq);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= p.G * p.Nq) continue;
    const int hr = kh * p.G + r / p.Nq, ir = r % p.Nq;
    const long long at = (long long)(b * p.H + hr) * p.Nq + ir;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const int d = (c * kRowLanes + lane) * 4;
      float4 o;
      unf2(acc[r][c].x[0], o.x, o.y);
      unf2(acc[r][c].x[1], o.z, o.w);
      o = make_float4(o.x * p.scale, o.y * p.scale, o.z * p.scale, o.w * p.scale);
      if (p.splits > 1)
        store4(p.part_o + ((long long)split * p.B * p.H * p.Nq + at) * p.D, d, p.D, p.D % 4 == 0, o);
      else
        store4(row_at<E>(p.dq, b, hr, ir), d, p.D, vq, o);
    }
  }
}

// dQ of the key splits, summed in order: one thread per element.
template <class E>
__global__ void __launch_bounds__(256) xattn_rows_dq_sum_kernel(const XParams p) {
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x, total = (long long)p.B * p.H * p.Nq * p.D;
  if (x >= total) return;
  float s = 0.f;
#pragma unroll 4
  for (int k = 0; k < p.splits; ++k) s += p.part_o[k * total + x];
  const int d = (int)(x % p.D), i = (int)(x / p.D % p.Nq);
  const long long bh = x / p.D / p.Nq;
  reinterpret_cast<E*>(p.dq.p)[bh / p.H * p.dq.s[0] + bh % p.H * p.dq.s[1] + i * p.dq.s[2] + d] = from_f<E>(s);
}

}  // namespace geoattn
