// Kernels around the cross attention: bucket ids by distance, their transpose, the bias table's gradient, dropout on
// hidden states, and the generator state.
#pragma once
#include "xattn_common.cuh"

namespace geoattn {

// ids[i][j] = number of edges <= the great-circle distance (km) of site i and station j; kNoPair beyond max_km.
// Haversine in float64 on the 6371 km sphere, as the geo prior's (extended_dl_forecasting.py:305-318).
__global__ void __launch_bounds__(256) distance_buckets_kernel(int nq, const double* __restrict__ lat_q,
                                                               const double* __restrict__ lon_q, int nk,
                                                               const double* __restrict__ lat_k,
                                                               const double* __restrict__ lon_k,
                                                               const double* __restrict__ edges, int nedges,
                                                               double max_km, uint8_t* __restrict__ ids) {
  __shared__ double edge[kMaxBuckets];
  if (threadIdx.x < nedges) edge[threadIdx.x] = edges[threadIdx.x];
  __syncthreads();
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;
  if (x >= (long long)nq * nk) return;
  const int i = (int)(x / nk), j = (int)(x % nk);
  const double d2r = 0.017453292519943295;
  const double li = lat_q[i] * d2r, lj = lat_k[j] * d2r;
  const double s1 = sin(0.5 * (li - lj)), s2 = sin(0.5 * (lon_q[i] * d2r - lon_k[j] * d2r));
  const double a = s1 * s1 + cos(li) * cos(lj) * s2 * s2;
  const double km = 2.0 * asin(sqrt(a > 1.0 ? 1.0 : a)) * 6371.0;
  int n = 0;
  for (int e = 0; e < nedges; ++e) n += km >= edge[e];
  ids[x] = km > max_km ? (uint8_t)kNoPair : (uint8_t)n;
}

// out[i][j] = ids[i][j], rows padded to `ldo` (a multiple of 16) with kNoPair: what 16-byte loads need.
__global__ void __launch_bounds__(256) ids_pad_kernel(const uint8_t* __restrict__ ids, long long ld, int nq, int nk,
                                                      int ldo, uint8_t* __restrict__ out) {
  const long long x = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (x >= (long long)nq * ldo) return;
  const long long i = x / ldo;
  const int j = (int)(x % ldo);
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) w |= (uint32_t)(j + e < nk ? ids[i * ld + j + e] : (uint8_t)kNoPair) << (8 * e);
  *reinterpret_cast<uint32_t*>(out + x) = w;
}

// idsT[j][i] = ids[i][j], padded to [nkp][nqp] with kNoPair.
__global__ void __launch_bounds__(256) ids_transpose_kernel(const uint8_t* __restrict__ ids, long long ld, int nq,
                                                            int nk, int nqp, uint8_t* __restrict__ idsT) {
  __shared__ uint8_t tile[64][65];
  const int i0 = blockIdx.x * 64, j0 = blockIdx.y * 64;
  for (int x = threadIdx.x; x < 64 * 64; x += 256) {
    const int r = x / 64, c = x % 64;
    tile[r][c] = i0 + r < nq && j0 + c < nk ? ids[(long long)(i0 + r) * ld + j0 + c] : (uint8_t)kNoPair;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < 64 * 16; x += 256) {
    const int r = x / 16, c = (x % 16) * 4;
    const uint32_t w = tile[c][r] | tile[c + 1][r] << 8 | tile[c + 2][r] << 16 | (uint32_t)tile[c + 3][r] << 24;
    *reinterpret_cast<uint32_t*>(idsT + (long long)(j0 + r) * nqp + i0 + c) = w;
  }
}

// Bias gradient of one launch's units: part[h][chunk][t] = sum of dS over the chunk's pairs of bucket t and the
// launch's batches. A thread sums its pairs over the batch first and then adds them to its own column of the
// shared histogram (hist[t][thread]: no atomics, no bank conflicts, a fixed order). Bound by reading dS once.
template <class S>
__global__ void __launch_bounds__(256) table_grad_kernel(const XParams p, int units, float* __restrict__ part) {
  constexpr int VEC = 16 / (int)sizeof(S);
  extern __shared__ float hist[];  // [T][256]
  const int h = blockIdx.y, kh = h / p.G, chunks = gridDim.x;
  for (int t = 0; t < p.T; ++t) hist[t * 256 + threadIdx.x] = 0.f;
  const long long per_row = p.nqp / VEC, total = (long long)p.Nk * per_row;
  const long long c0 = total * blockIdx.x / chunks, c1 = total * (blockIdx.x + 1) / chunks;
  const long long slab = (long long)p.nkp * p.nqp;
  const int first = (kh - p.u0 % p.Hkv + p.Hkv) % p.Hkv;  // first local unit of this key head
  for (long long x = c0 + threadIdx.x; x < c1; x += 256) {
    const int j = (int)(x / per_row);
    const long long at = (long long)j * p.nqp + (x % per_row) * VEC;
    float sum[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = 0.f;
#pragma unroll 4
    for (int ul = first; ul < units; ul += p.Hkv) {
      if (p.lens && j >= key_count(p, (p.u0 + ul) / p.Hkv)) continue;  // rows that the key pass left out
      const S* s = reinterpret_cast<const S*>(p.ds) + (long long)(ul * p.G + h % p.G) * slab + at;
      const uint4 w = *reinterpret_cast<const uint4*>(s);
      const S* v = reinterpret_cast<const S*>(&w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] += to_f(v[e]);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int t = p.idsT[at + e];
      if (t < p.T) hist[t * 256 + threadIdx.x] += sum[e];
    }
  }
  __syncthreads();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int t = warp; t < p.T; t += 8) {
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) x += hist[t * 256 + e * 32 + lane];
#pragma unroll
    for (int w = 16; w; w /= 2) x += __shfl_xor_sync(0xffffffffu, x, w);
    if (lane == 0) part[((long long)h * chunks + blockIdx.x) * p.T + t] = x;
  }
}

// dtable[h][t] = sum of the partials of every launch and chunk, in float64 and a fixed order: one warp per entry.
__global__ void __launch_bounds__(32) table_grad_sum_kernel(const float* __restrict__ part, int launches, int H,
                                                            int chunks, int T, void* out, int out_bf16) {
  const int h = blockIdx.x / T, t = blockIdx.x % T;
  double x = 0.0;
  for (int c = threadIdx.x; c < launches * chunks; c += 32)
    x += part[(((long long)(c / chunks) * H + h) * chunks + c % chunks) * T + t];
#pragma unroll
  for (int w = 16; w; w /= 2) x += __shfl_xor_sync(0xffffffffu, x, w);
  if (threadIdx.x) return;
  if (out_bf16) reinterpret_cast<__nv_bfloat16*>(out)[blockIdx.x] = __float2bfloat16_rn((float)x);
  else reinterpret_cast<float*>(out)[blockIdx.x] = (float)x;
}

// y = keep ? scale x : 0 (+ residual), kept by bit e % 8 of counter (e / 8 low, e / 8 high, offset low, offset high)
// under the key (seed low, seed high); eight elements, one Philox call, per thread. A dropped element is 0 whatever x
// holds. One pass over memory: bound by HBM.
template <class E, bool RES>
__global__ void __launch_bounds__(256) dropout_kernel(const E* __restrict__ x, const E* __restrict__ res,
                                                      E* __restrict__ y, long long n, const long long* __restrict__ rng,
                                                      int thr, float scale, int vec) {
  const long long blk = (long long)blockIdx.x * 256 + threadIdx.x, e0 = blk * 8;
  if (e0 >= n) return;
  const unsigned long long seed = (unsigned long long)rng[0], off = (unsigned long long)rng[1];
  const PhiloxKey key{(uint32_t)seed, (uint32_t)(seed >> 32)};
  const uint32_t keep =
      keep_bits8(philox7((uint32_t)blk, (uint32_t)((unsigned long long)blk >> 32), (uint32_t)off,
                         (uint32_t)(off >> 32), key),
                 (uint32_t)thr);
  constexpr int W = sizeof(E) * 8 / 16;  // 16-byte words of eight elements
  if (vec && e0 + 8 <= n) {
    uint4 a[W], r[W], o[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      a[w] = reinterpret_cast<const uint4*>(x + e0)[w];
      if (RES) r[w] = reinterpret_cast<const uint4*>(res + e0)[w];
    }
    const E *av = reinterpret_cast<const E*>(a), *rv = reinterpret_cast<const E*>(r);
    E* ov = reinterpret_cast<E*>(o);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = (keep >> e) & 1 ? to_f(av[e]) * scale : 0.f;
      ov[e] = from_f<E>(RES ? d + to_f(rv[e]) : d);
    }
#pragma unroll
    for (int w = 0; w < W; ++w) reinterpret_cast<uint4*>(y + e0)[w] = o[w];
  } else {
    for (int e = 0; e < 8 && e0 + e < n; ++e) {
      const float d = (keep >> e) & 1 ? to_f(x[e0 + e]) * scale : 0.f;
      y[e0 + e] = from_f<E>(RES ? d + to_f(res[e0 + e]) : d);
    }
  }
}

// Hands out the generator's (seed, offset) and moves the offset on, in stream order, so that a captured call draws
// new masks at every replay.
__global__ void rng_take_kernel(long long* state, long long* out) {
  out[0] = state[0];
  out[1] = state[1];
  state[1] += 1;
}

}  // namespace geoattn
