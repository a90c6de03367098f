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

// Tiled copy of the bucket ids for the tensor-core kernels, out[row / 64][col / 8][row % 64][8], rows and columns padded:
// a warp whose lanes are consecutive rows reads 8 columns as one contiguous block (row-major rows cost a cache line per
// lane). An entry is the byte offset of its bucket in a table of T fp32 values and -inf behind them (kNoPairOffset for
// ids that exclude their pair), so that a kernel spends one instruction per id. TRANS: rows are the keys and columns the
// queries (backward), else the other way round. A 64 x 64 tile per CTA.
template <bool TRANS>
__global__ void __launch_bounds__(256) ids_tile_kernel(const uint8_t* __restrict__ ids, long long ld, int nq, int nk,
                                                       int cols_p, int T, uint16_t* __restrict__ out) {
  __shared__ uint8_t tile[64][68];  // [query][key]
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  const int i0 = TRANS ? c0 : r0, j0 = TRANS ? r0 : c0;
  for (int x = threadIdx.x; x < 64 * 64; x += 256) {
    const int i = x / 64, j = x % 64;
    tile[i][j] = i0 + i < nq && j0 + j < nk ? ids[(long long)(i0 + i) * ld + j0 + j] : (uint8_t)kNoPair;
  }
  __syncthreads();
  uint4* dst = reinterpret_cast<uint4*>(out) + ((long long)blockIdx.y * (cols_p / 8) + c0 / 8) * 64;
  for (int x = threadIdx.x; x < 64 * 8; x += 256) {
    const int r = x % 64, g = x / 64;
    if (c0 + g * 8 >= cols_p) break;
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t o[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = g * 8 + k * 2 + e, id = TRANS ? tile[c][r] : tile[r][c];
        o[e] = id < T ? 4 * id : kNoPairOffset;
      }
      w[k] = o[0] | o[1] << 16;
    }
    dst[(long long)g * 64 + r] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Bias gradient of one launch's units: part[h][chunk][t] = sum of dS over the chunk's pairs of bucket t and the
// launch's batches. dS lies as the ids do, [key / 64][query / 8][key % 64][8] per head; a thread takes 16 bytes of it,
// sums them over the batch first (8 loads in flight) and then adds them to its own column of the shared histogram
// (hist[t][thread]: no atomics, no bank conflicts, a fixed order). Bound by reading dS
// once: 256 x 16 heads x 512 x 512 in bf16 317 us, 6.8 TB/s (part of it still in L2).
template <class S>
__global__ void __launch_bounds__(256) table_grad_kernel(const XParams p, int units, float* __restrict__ part) {
  constexpr int VEC = 16 / (int)sizeof(S);
  extern __shared__ float hist[];  // [T][256]
  const int h = blockIdx.y, kh = h / p.G, chunks = gridDim.x;
  for (int t = 0; t < p.T; ++t) hist[t * 256 + threadIdx.x] = 0.f;
  const long long slab = (long long)p.nkp * p.nqp, total = slab / VEC;
  const long long c0 = total * blockIdx.x / chunks, c1 = total * (blockIdx.x + 1) / chunks;
  const int first = (kh - p.u0 % p.Hkv + p.Hkv) % p.Hkv;  // first local unit of this key head
  const long long step = (long long)p.Hkv * p.G * slab;
  for (long long x = c0 + threadIdx.x; x < c1; x += 256) {
    const long long at = x * VEC;
    const int j = (int)(at / (64ll * p.nqp)) * 64 + (int)(at / 8 % 64);
    if ((int)(at / 512 % (p.nqp / 8)) * 8 >= p.Nq) continue;  // granules without a query hold nothing
    const S* src = reinterpret_cast<const S*>(p.ds) + (long long)(first * p.G + h % p.G) * slab + at;
    float sum[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = 0.f;
    for (int ul = first; ul < units; ul += 8 * p.Hkv) {
      uint4 w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int u = ul + k * p.Hkv;
        // keys that the key pass left out hold nothing
        w[k] = u < units && j < key_count(p, (p.u0 + u) / p.Hkv) ? __ldcs(reinterpret_cast<const uint4*>(src + k * step))
                                                                 : make_uint4(0, 0, 0, 0);
      }
      src += 8 * step;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const S* v = reinterpret_cast<const S*>(&w[k]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum[e] += to_f(v[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int o = p.idsT[at + e];  // 4 * bucket
      if (o != kNoPairOffset) hist[o * 64 + threadIdx.x] += sum[e];
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
// holds. One pass over memory, bound by HBM: 131072 x 2048 bf16 with the residual 244 us (6.6 TB/s), without 212 us (5.1);
// 18907 x 1000 fp32 35 and 24 us.
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
