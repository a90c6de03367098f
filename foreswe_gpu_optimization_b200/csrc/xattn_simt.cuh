// Cross attention on the FMA pipe: fp32 storage. The tensor cores take fp32 operands only as TF32 (10 mantissa bits);
// these kernels keep every product and sum in fp32, so the results carry fp32 accuracy.
//
// Tiles sit in shared memory head-dim-major ([d][row], rows padded by 4 floats), so that a thread's 4 or 8 rows (or
// keys) are one or two 16-byte loads per d; each of the 256 threads (16 x 16) owns a register block of the product and
// works on it two values at a time (fma.rn.f32x2). Weights go through shared memory between the two products, in
// 16-byte chunks whose place is XORed with the writing lane so that neither side meets a bank conflict.
// Bound by shared memory's return path (one 32-bit word per lane and clock: longer than the products themselves) and,
// above D = 64, by the latency that 8 warps per SM cannot hide. 32 x 8 heads x 512 x 512 x 64 with the bias: forward
// 542 us (32 TFLOP/s of 74), key pass 1120 us (31), dQ 290 us (30); 8 x 16 / 2 heads, 415 x 1441 of 175 with dropout and
// the bias: forward 2.1 ms (26), key pass 4.8 ms (22). Fetching the next query tile during the products changed nothing
// there.
#pragma once
#include <type_traits>

#include "sm100.cuh"
#include "xattn_common.cuh"

namespace geoattn {

constexpr int kSimtThreads = 256;

// One thread's share of a tile of ROWS rows x DP columns, 4 consecutive d at a time, on its way from global to shared
// memory: `at` gives its x-th (row, d), `get` fetches them (zero where d >= D or ok(row) is false), so that a tile can
// be fetched while another is worked on.
template <int ROWS, int DP, int NT = kSimtThreads>
struct SimtTile {
  static constexpr int N = ROWS * DP / 4 / NT;
  float4 v[N];
  // head-dim-major tiles: a warp takes 16 rows x 8 d, whole 32-byte sectors in and 32 different banks out
  static __device__ __forceinline__ void at_t(int x, int& r, int& d) {
    static_assert(ROWS % 16 == 0, "");
    const int y = x / 32;
    r = y % (ROWS / 16) * 16 + x % 16, d = y / (ROWS / 16) * 8 + x % 32 / 16 * 4;
  }
  // row-major tiles
  static __device__ __forceinline__ void at_n(int x, int& r, int& d) { r = x / (DP / 4), d = x % (DP / 4) * 4; }

  template <bool T, class OK>
  __device__ __forceinline__ void get(const float* src, long long ld, int D, bool vec, OK ok) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      int r, d;
      if (T) at_t(threadIdx.x + k * NT, r, d);
      else at_n(threadIdx.x + k * NT, r, d);
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (d < D && ok(r)) {
        const float* s = src + (long long)r * ld + d;
        if (vec) {
          v[k] = *reinterpret_cast<const float4*>(s);
        } else {
          v[k].x = s[0];
          if (d + 1 < D) v[k].y = s[1];
          if (d + 2 < D) v[k].z = s[2];
          if (d + 3 < D) v[k].w = s[3];
        }
      }
    }
  }
  template <int ST>
  __device__ __forceinline__ void put_t(float* dst) const {
    static_assert(4 * ST % 32 == 16, "");
#pragma unroll
    for (int k = 0; k < N; ++k) {
      int r, d;
      at_t(threadIdx.x + k * NT, r, d);
      dst[d * ST + r] = v[k].x, dst[(d + 1) * ST + r] = v[k].y;
      dst[(d + 2) * ST + r] = v[k].z, dst[(d + 3) * ST + r] = v[k].w;
    }
  }
  __device__ __forceinline__ void put_n(float* dst) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      int r, d;
      at_n(threadIdx.x + k * NT, r, d);
      *reinterpret_cast<float4*>(dst + r * DP + d) = v[k];
    }
  }
};

__device__ __forceinline__ bool simt_vec(const XTensor& t, int D) {
  return D % 4 == 0 && (reinterpret_cast<uintptr_t>(t.p) & 15) == 0 && t.s[0] % 4 == 0 &&
         t.s[1] % 4 == 0 && t.s[2] % 4 == 0;
}

// ---------------------------------------------------------------------------------------------------------------
// Forward: one CTA per (128 query rows, head, key split). Online softmax: running max and sum per row, the rows'
// 64 columns spread over 16 lanes.
// ---------------------------------------------------------------------------------------------------------------
template <int DP>
struct SimtFwd {
  // 16 x XT threads of 8 rows and CT columns. (8 x 8 blocks load less from shared memory per FMA, but leave 4 warps per
  // CTA, which cannot hide the softmax between the products: 579 against 538 us at 32 x 8 x 512 x 64.)
  static constexpr int XT = 16, NT = 16 * XT, CT = 64 / XT, CO = DP / XT;
  static constexpr int BM = 128, BN = 64, SQ = BM + 4, SK = BN + 4;
  static constexpr int FLOATS = DP * SQ + DP * SK + BN * BM + 256 + BN;
  static constexpr int SMEM = FLOATS * 4;
};

template <int DP>
__global__ void __launch_bounds__(SimtFwd<DP>::NT, DP == 64 ? 2 : 1) xattn_simt_fwd_kernel(const XParams p) {
  using C = SimtFwd<DP>;
  constexpr int XT = C::XT, CT = C::CT, CO = C::CO;
  extern __shared__ float4 simt_smem[];
  float* qt = reinterpret_cast<float*>(simt_smem);
  float* kv = qt + DP * C::SQ;
  float* pt = kv + DP * C::SK;
  float* tab = pt + C::BN * C::BM;
  float* live = tab + 256;
  const int qt_i = blockIdx.x % p.tiles, rest = blockIdx.x / p.tiles;
  const int h = rest % p.H, b = (rest / p.H) % p.B, split = rest / p.H / p.B;
  const int kh = h / p.G, i0 = qt_i * C::BM, bh = b * p.H + h;
  const int ty = threadIdx.x / XT, tx = threadIdx.x % XT;
  const auto col = [&](int c) { return c / 4 * (XT * 4) + tx * 4 + c % 4; };  // this thread's columns
  const int n = key_count(p, b);
  const int ntiles = (n + C::BN - 1) / C::BN;
  const int t0 = (int)((long long)ntiles * split / p.splits), t1 = (int)((long long)ntiles * (split + 1) / p.splits);
  const float* Q = reinterpret_cast<const float*>(p.q.p) + b * p.q.s[0] + h * p.q.s[1];
  const float* K = reinterpret_cast<const float*>(p.k.p) + b * p.k.s[0] + kh * p.k.s[1];
  const float* V = reinterpret_cast<const float*>(p.v.p) + b * p.v.s[0] + kh * p.v.s[1];
  const bool vq = simt_vec(p.q, p.D), vk = simt_vec(p.k, p.D), vv = simt_vec(p.v, p.D);
  if (blockIdx.x + threadIdx.x == 0) *p.status = kDevOk;
  const AttnDrop drop = attn_drop(p.rng, p.drop_thr, p.drop_scale);

  if (p.ids)
    for (int t = threadIdx.x; t < 256; t += C::NT) tab[t] = table_log2(p, h, t);
  {
    SimtTile<C::BM, DP, C::NT> q;
    q.template get<true>(Q + (long long)i0 * p.q.s[2], p.q.s[2], p.D, vq, [&](int r) { return i0 + r < p.Nq; });
    q.template put_t<C::SQ>(qt);
  }
  SimtTile<C::BN, DP, C::NT> next;  // the next K, then V tile, fetched a product ahead
  auto fetch = [&](const XTensor& x, const float* src, bool vec, auto t, int j0) {
    next.template get<decltype(t)::value>(src + (long long)j0 * x.s[2], x.s[2], p.D, vec,
                                          [&](int r) { return key_live(p, b, j0 + r, n); });
  };
  if (t0 < t1) fetch(p.k, K, vk, std::true_type{}, t0 * C::BN);

  float m[8], l[8];
  uint64_t acc[4][CO];  // pairs of rows
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < CO; ++c) acc[r / 2][c] = 0;
  }
  for (int t = t0; t < t1; ++t) {
    const int j0 = t * C::BN;
    __syncthreads();  // the last tile's products have read kv, pt and live
    if (threadIdx.x < C::BN) live[threadIdx.x] = key_live(p, b, j0 + threadIdx.x, n) ? 0.f : -INFINITY;
    next.template put_t<C::SK>(kv);
    __syncthreads();
    fetch(p.v, V, vv, std::false_type{}, j0);
    uint64_t s2[4][CT] = {};
#pragma unroll 4
    for (int d = 0; d < DP; ++d) {
      const ulonglong2 a0 = *reinterpret_cast<const ulonglong2*>(qt + d * C::SQ + ty * 8);
      const ulonglong2 a1 = *reinterpret_cast<const ulonglong2*>(qt + d * C::SQ + ty * 8 + 4);
      const uint64_t a[4] = {a0.x, a0.y, a1.x, a1.y};
#pragma unroll
      for (int c = 0; c < CT; c += 4) {
        const float4 k4 = *reinterpret_cast<const float4*>(kv + d * C::SK + col(c));
        const uint64_t kk[4] = {f2(k4.x, k4.x), f2(k4.y, k4.y), f2(k4.z, k4.z), f2(k4.w, k4.w)};
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) s2[r][c + e] = fma2(a[r], kk[e], s2[r][c + e]);
      }
    }
    __syncthreads();  // every thread has read K
    next.put_n(kv);
    if (t + 1 < t1) fetch(p.k, K, vk, std::true_type{}, j0 + C::BN);
    float s[8][CT];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < CT; ++c) unf2(s2[r][c], s[2 * r][c], s[2 * r + 1][c]);
    float corr[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int i = i0 + ty * 8 + r;
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const int j = j0 + col(c);
        float x = s[r][c] * p.scale_log2;
        if (p.ids && i < p.Nq && j < p.Nk) x += tab[p.ids[i * p.ids_ld + j]];
        s[r][c] = live[col(c)] == 0.f ? x : -INFINITY;
        mx = fmaxf(mx, s[r][c]);
      }
#pragma unroll
      for (int w = 1; w < XT; w *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float mn = fmaxf(m[r], mx), base = mn == -INFINITY ? 0.f : mn;
      corr[r] = xex2(m[r] - base);
      m[r] = mn;
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        s[r][c] = xex2(s[r][c] - base);
        sum += s[r][c];
      }
#pragma unroll
      for (int w = 1; w < XT; w *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      l[r] = l[r] * corr[r] + sum;
      if (drop.thr) {
#pragma unroll
        for (int c = 0; c < CT; c += 4) {
          const uint32_t kb = drop.keep8(i, (j0 + col(c)) >> 3, bh) >> ((tx & 1) * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[r][c + e] = (kb >> e) & 1 ? s[r][c + e] : 0.f;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < CO; ++c) acc[r][c] = mul2(acc[r][c], f2(corr[2 * r], corr[2 * r + 1]));
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      float* dst = pt + col(c) * C::BM;
      *reinterpret_cast<float4*>(dst + ((ty * 2) ^ (tx & 7)) * 4) = make_float4(s[0][c], s[1][c], s[2][c], s[3][c]);
      *reinterpret_cast<float4*>(dst + ((ty * 2 + 1) ^ (tx & 7)) * 4) = make_float4(s[4][c], s[5][c], s[6][c], s[7][c]);
    }
    __syncthreads();
#pragma unroll 4
    for (int j = 0; j < C::BN; ++j) {
      const int w = (j >> 2) & 7;
      const ulonglong2 a0 = *reinterpret_cast<const ulonglong2*>(pt + j * C::BM + ((ty * 2) ^ w) * 4);
      const ulonglong2 a1 = *reinterpret_cast<const ulonglong2*>(pt + j * C::BM + ((ty * 2 + 1) ^ w) * 4);
      const uint64_t a[4] = {a0.x, a0.y, a1.x, a1.y};
#pragma unroll
      for (int c = 0; c < CO; c += 4) {
        const float4 v4 = *reinterpret_cast<const float4*>(kv + j * DP + col(c));
        const uint64_t v[4] = {f2(v4.x, v4.x), f2(v4.y, v4.y), f2(v4.z, v4.z), f2(v4.w, v4.w)};
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[r][c + e] = fma2(a[r], v[e], acc[r][c + e]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int i = i0 + ty * 8 + r;
    if (i >= p.Nq) continue;
    float out[CO];
#pragma unroll
    for (int c = 0; c < CO; ++c) {
      float a, d;
      unf2(acc[r / 2][c], a, d);
      out[c] = r & 1 ? d : a;
    }
    const long long row = (long long)bh * p.Nq + i;
    if (p.splits > 1) {
      const long long at = (long long)split * p.B * p.H * p.Nq + row;
#pragma unroll
      for (int c = 0; c < CO; ++c) {
        const int d = col(c);
        if (d < p.D) p.part_o[at * p.D + d] = out[c];
      }
      if (tx == 0) {
        p.part_ml[at * 2] = m[r];
        p.part_ml[at * 2 + 1] = l[r];
      }
    } else {
      const float inv = l[r] == 0.f ? 0.f : (drop.thr ? drop.scale : 1.f) / l[r];
      float* O = reinterpret_cast<float*>(p.o.p) + b * p.o.s[0] + h * p.o.s[1] + i * p.o.s[2];
#pragma unroll
      for (int c = 0; c < CO; ++c) {
        const int d = col(c);
        if (d < p.D) O[d] = out[c] * inv;
      }
      if (tx == 0 && p.stats) p.stats[row] = row_stats(m[r], l[r]);
    }
  }
}

// Join the key splits of each row: one warp per row. The splits' weights are worked out by the lanes side by side (32
// at a time) and handed round; a lane sums 4 consecutive columns. 16 x 32 heads x 4 rows of 128, 5 splits: 6 us.
template <class E>
__global__ void __launch_bounds__(256) xattn_combine_kernel(const XParams p) {
  const long long rows = (long long)p.B * p.H * p.Nq;
  const long long row = (long long)blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (row >= rows) return;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + row;
  float m = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, ml[s * rows].x);
#pragma unroll
  for (int w = 16; w; w /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
  const float base = m == -INFINITY ? 0.f : m;
  const int i = (int)(row % p.Nq), bh = (int)(row / p.Nq), h = bh % p.H, b = bh / p.H;
  E* O = reinterpret_cast<E*>(p.o.p) + b * p.o.s[0] + h * p.o.s[1] + i * p.o.s[2];
  const bool vec = p.D % 4 == 0;
  float l = 0.f;
  for (int d0 = 0; d0 < p.D; d0 += 128) {
    const int d = d0 + lane * 4;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < p.splits; s0 += 32) {
      const float2 mine = s0 + lane < p.splits ? ml[(s0 + lane) * rows] : make_float2(-INFINITY, 0.f);
      const float weight = xex2(mine.x - base);
      if (d0 == 0) l += mine.y * weight;
      const int n = p.splits - s0 < 32 ? p.splits - s0 : 32;
#pragma unroll 4
      for (int s = 0; s < n; ++s) {
        const float w = __shfl_sync(0xffffffffu, weight, s);
        const float* src = p.part_o + ((s0 + s) * rows + row) * p.D + d;
        if (vec && d < p.D) {
          const float4 v = *reinterpret_cast<const float4*>(src);
          x[0] = fmaf(v.x, w, x[0]), x[1] = fmaf(v.y, w, x[1]), x[2] = fmaf(v.z, w, x[2]), x[3] = fmaf(v.w, w, x[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < p.D) x[e] = fmaf(src[e], w, x[e]);
        }
      }
    }
    if (d0 == 0) {
#pragma unroll
      for (int w = 16; w; w /= 2) l += __shfl_xor_sync(0xffffffffu, l, w);
    }
    const float inv = l == 0.f ? 0.f : (p.drop_thr ? p.drop_scale : 1.f) / l;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < p.D) O[d + e] = from_f<E>(x[e] * inv);
  }
  if (lane == 0 && p.stats) p.stats[row] = row_stats(m, l);
}

// delta_i = dO_i . O_i: 8 lanes per row, 4 rows per warp.
__global__ void __launch_bounds__(256) xattn_delta_kernel(const XParams p) {
  const long long rows = (long long)p.B * p.H * p.Nq;
  const long long row = (long long)blockIdx.x * 32 + threadIdx.x / 8;
  const int lane = threadIdx.x % 8;
  if (blockIdx.x + threadIdx.x == 0) *p.status = kDevOk;
  float x = 0.f;
  if (row < rows) {
    const int i = (int)(row % p.Nq), bh = (int)(row / p.Nq), h = bh % p.H, b = bh / p.H;
    const float* O = reinterpret_cast<const float*>(p.o.p) + b * p.o.s[0] + h * p.o.s[1] + i * p.o.s[2];
    const float* G = reinterpret_cast<const float*>(p.dout.p) + b * p.dout.s[0] + h * p.dout.s[1] + i * p.dout.s[2];
    if (simt_vec(p.o, p.D) && simt_vec(p.dout, p.D)) {
#pragma unroll 2
      for (int d = lane * 4; d < p.D; d += 32) {
        const float4 u = *reinterpret_cast<const float4*>(O + d), v = *reinterpret_cast<const float4*>(G + d);
        x = fmaf(u.x, v.x, fmaf(u.y, v.y, fmaf(u.z, v.z, fmaf(u.w, v.w, x))));
      }
    } else {
      for (int d = lane; d < p.D; d += 8) x = fmaf(O[d], G[d], x);
    }
  }
#pragma unroll
  for (int w = 4; w; w /= 2) x += __shfl_xor_sync(0xffffffffu, x, w);
  if (lane == 0 && row < rows) p.delta[row] = x;
}

// ---------------------------------------------------------------------------------------------------------------
// Backward, key pass: one CTA per (TK keys, key head, batch); loops over the heads that share the key head and their
// 64-row query tiles. dK and dV stay in registers (no atomics: fixed order); dS^T goes to the scratch.
// Half of the threads form the scores and the others dP, in blocks of 8 x 4 (4 x 4 above D = 128), and exchange them
// through the weights' place in shared memory: fewer words per product than both in every thread's blocks of half the
// size (173 heads, 327 x 40 of 158: 343 -> 277 us; 32 x 8 heads x 512 x 512 x 64: 1163 -> 1120 us).
// ---------------------------------------------------------------------------------------------------------------
template <int DP>
struct SimtBwd {
  static constexpr int TK = DP <= 128 ? 64 : 32, KT = TK / 16, BQ = 64, SK = TK + 4, SQ = BQ + 4;
  static constexpr int QR = TK / 8;         // a thread's queries in the first products, by 4 keys
  static constexpr int XN = 16 * 64 / TK;   // threads across the columns in the second ones, 4 keys each
  static constexpr int FLOATS = 2 * DP * SK + 2 * DP * SQ + 2 * TK * BQ + 256 + TK + 3 * BQ;
  static constexpr int SMEM = FLOATS * 4;
};

template <int DP>
__global__ void __launch_bounds__(kSimtThreads, DP == 64 ? 2 : 1) xattn_simt_bwd_keys_kernel(const XParams p) {
  using C = SimtBwd<DP>;
  constexpr int KT = C::KT, XN = C::XN, NC = DP / XN, QR = C::QR;
  extern __shared__ float4 simt_smem[];
  float* kt = reinterpret_cast<float*>(simt_smem);
  float* vt = kt + DP * C::SK;
  float* qt = vt + DP * C::SK;
  float* gt = qt + DP * C::SQ;
  float* pt = gt + DP * C::SQ;
  float* st = pt + C::TK * C::BQ;
  float* tab = st + C::TK * C::BQ;
  float* live = tab + 256;
  float* mx = live + C::TK;
  float* inv = mx + C::BQ;
  float* del = inv + C::BQ;
  const int nkt = (p.Nk + C::TK - 1) / C::TK;
  const int kt_i = blockIdx.x % nkt, ul = blockIdx.x / nkt, unit = p.u0 + ul;
  const int b = unit / p.Hkv, kh = unit % p.Hkv, j0 = kt_i * C::TK;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int n = key_count(p, b);
  const AttnDrop drop = attn_drop(p.rng, p.drop_thr, p.drop_scale);
  // first products: half of the threads form the scores, the others dP
  const int part = threadIdx.x / 128, py = threadIdx.x % 128 / (C::TK / 4), px = threadIdx.x % (C::TK / 4);
  const float *rows = part ? gt : qt, *cols = part ? vt : kt;
  const int ny = threadIdx.x / XN, nx = threadIdx.x % XN;  // second products: keys 4 ny .., columns nx + XN c
  uint64_t ak[4][NC], av[4][NC];  // sums over even and odd queries
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int c = 0; c < NC; ++c) ak[x][c] = av[x][c] = 0;

  if (j0 < n) {
    if (threadIdx.x < C::TK) live[threadIdx.x] = key_live(p, b, j0 + threadIdx.x, n) ? 0.f : -INFINITY;
    __syncthreads();
    const float* K = reinterpret_cast<const float*>(p.k.p) + b * p.k.s[0] + kh * p.k.s[1] + (long long)j0 * p.k.s[2];
    const float* V = reinterpret_cast<const float*>(p.v.p) + b * p.v.s[0] + kh * p.v.s[1] + (long long)j0 * p.v.s[2];
    {
      SimtTile<C::TK, DP> x;
      const auto ok = [&](int r) { return live[r] == 0.f; };
      x.template get<true>(K, p.k.s[2], p.D, simt_vec(p.k, p.D), ok);
      x.template put_t<C::SK>(kt);
      x.template get<true>(V, p.v.s[2], p.D, simt_vec(p.v, p.D), ok);
      x.template put_t<C::SK>(vt);
    }
    const int nqt = (p.Nq + C::BQ - 1) / C::BQ;
    const bool vq = simt_vec(p.q, p.D), vg = simt_vec(p.dout, p.D);
    for (int it = 0; it < nqt * p.G; ++it) {
      const int h = kh * p.G + it / nqt, i0 = (it % nqt) * C::BQ, bh = b * p.H + h;
      const float* Q = reinterpret_cast<const float*>(p.q.p) + b * p.q.s[0] + h * p.q.s[1] + (long long)i0 * p.q.s[2];
      const float* G = reinterpret_cast<const float*>(p.dout.p) + b * p.dout.s[0] + h * p.dout.s[1] + (long long)i0 * p.dout.s[2];
      __syncthreads();  // the last tile's products have read qt, gt, pt, st
      if (p.ids && it % nqt == 0) tab[threadIdx.x] = table_log2(p, h, threadIdx.x);
      if (threadIdx.x < C::BQ) {
        const int i = i0 + threadIdx.x;
        const float2 st = i < p.Nq ? p.stats[(long long)bh * p.Nq + i] : make_float2(0.f, 0.f);
        mx[threadIdx.x] = st.x;
        inv[threadIdx.x] = st.y;
        del[threadIdx.x] = i < p.Nq ? p.delta[(long long)bh * p.Nq + i] : 0.f;
      }
      {
        SimtTile<C::BQ, DP> x, y;
        const auto ok = [&](int r) { return i0 + r < p.Nq; };
        x.template get<true>(Q, p.q.s[2], p.D, vq, ok);
        y.template get<true>(G, p.dout.s[2], p.D, vg, ok);
        x.template put_t<C::SQ>(qt);
        y.template put_t<C::SQ>(gt);
      }
      __syncthreads();
      {
        uint64_t x2[QR / 2][4] = {};  // pairs of queries
#pragma unroll 4
        for (int d = 0; d < DP; ++d) {
          uint64_t a[QR / 2];
#pragma unroll
          for (int u = 0; u < QR / 4; ++u) {
            const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(rows + d * C::SQ + py * QR + u * 4);
            a[2 * u] = v.x, a[2 * u + 1] = v.y;
          }
          const float4 k4 = *reinterpret_cast<const float4*>(cols + d * C::SK + px * 4);
          const uint64_t kk[4] = {f2(k4.x, k4.x), f2(k4.y, k4.y), f2(k4.z, k4.z), f2(k4.w, k4.w)};
#pragma unroll
          for (int u = 0; u < QR / 2; ++u)
#pragma unroll
            for (int c = 0; c < 4; ++c) x2[u][c] = fma2(a[u], kk[c], x2[u][c]);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int key = px * 4 + c;
          float* dst = (part ? st : pt) + key * C::BQ;
#pragma unroll
          for (int u = 0; u < QR / 4; ++u) {
            float4 v;
            unf2(x2[2 * u][c], v.x, v.y);
            unf2(x2[2 * u + 1][c], v.z, v.w);
            *reinterpret_cast<float4*>(dst + ((py * (QR / 4) + u) ^ (key / KT & 7)) * 4) = v;
          }
        }
      }
      __syncthreads();
      float s[4][KT], dp[4][KT];
#pragma unroll
      for (int c = 0; c < KT; ++c) {
        const int at = (tx * KT + c) * C::BQ + (ty ^ (tx & 7)) * 4;
        const float4 u = *reinterpret_cast<const float4*>(pt + at), v = *reinterpret_cast<const float4*>(st + at);
        s[0][c] = u.x, s[1][c] = u.y, s[2][c] = u.z, s[3][c] = u.w;
        dp[0][c] = v.x, dp[1][c] = v.y, dp[2][c] = v.z, dp[3][c] = v.w;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = i0 + ty * 4 + r;
        const float m = mx[ty * 4 + r], il = inv[ty * 4 + r], dl = del[ty * 4 + r];
        const uint32_t kb = drop.thr ? drop.keep8(i, (j0 + tx * KT) >> 3, bh) >> ((j0 + tx * KT) & 7) : 0;
#pragma unroll
        for (int c = 0; c < KT; ++c) {
          const int j = j0 + tx * KT + c;
          float x = s[r][c] * p.scale_log2;
          if (p.ids && i < p.Nq && j < p.Nk) x += tab[p.ids[i * p.ids_ld + j]];
          const float pr = live[tx * KT + c] == 0.f ? xex2(x - m) * il : 0.f;
          float a = pr, g = dp[r][c];
          if (drop.thr) {
            const bool keep = (kb >> c) & 1;
            a = keep ? pr * drop.scale : 0.f;
            g = keep ? g * drop.scale : 0.f;
          }
          s[r][c] = a;
          dp[r][c] = live[tx * KT + c] == 0.f ? pr * (g - dl) : 0.f;
        }
      }
#pragma unroll
      for (int c = 0; c < KT; ++c) {
        const int at = (tx * KT + c) * C::BQ + (ty ^ (tx & 7)) * 4;
        *reinterpret_cast<float4*>(pt + at) = make_float4(s[0][c], s[1][c], s[2][c], s[3][c]);
        *reinterpret_cast<float4*>(st + at) = make_float4(dp[0][c], dp[1][c], dp[2][c], dp[3][c]);
      }
      __syncthreads();
      float* ds = reinterpret_cast<float*>(p.ds) + (long long)(ul * p.G + it / nqt) * p.nkp * p.nqp +
                  ((long long)(j0 / 64) * (p.nqp / 8) + i0 / 8) * 512 + j0 % 64 * 8;
#pragma unroll 2
      for (int x = threadIdx.x; x < C::TK * 16; x += kSimtThreads) {  // granules of 8 queries, keys side by side
        const int g = x / (2 * C::TK), key = x / 2 % C::TK, half = x % 2;
        *reinterpret_cast<float4*>(ds + g * 512 + key * 8 + half * 4) =
            *reinterpret_cast<const float4*>(st + key * C::BQ + ((2 * g + half) ^ (key / KT & 7)) * 4);
      }
#pragma unroll 2
      for (int r = 0; r < C::BQ / 4; ++r) {
        ulonglong2 pp[4], ss[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int key = ny * 4 + x, at = key * C::BQ + (r ^ (key / KT & 7)) * 4;
          pp[x] = *reinterpret_cast<const ulonglong2*>(pt + at);
          ss[x] = *reinterpret_cast<const ulonglong2*>(st + at);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const ulonglong2 g2 = *reinterpret_cast<const ulonglong2*>(gt + (nx + XN * c) * C::SQ + r * 4);
          const ulonglong2 q2 = *reinterpret_cast<const ulonglong2*>(qt + (nx + XN * c) * C::SQ + r * 4);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            av[x][c] = fma2(pp[x].x, g2.x, fma2(pp[x].y, g2.y, av[x][c]));
            ak[x][c] = fma2(ss[x].x, q2.x, fma2(ss[x].y, q2.y, ak[x][c]));
          }
        }
      }
    }
  }
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int j = j0 + ny * 4 + x;
    if (j >= p.Nk) continue;
    float* dK = reinterpret_cast<float*>(p.dk.p) + b * p.dk.s[0] + kh * p.dk.s[1] + (long long)j * p.dk.s[2];
    float* dV = reinterpret_cast<float*>(p.dv.p) + b * p.dv.s[0] + kh * p.dv.s[1] + (long long)j * p.dv.s[2];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = nx + XN * c;
      if (d < p.D) {
        float e, o;
        unf2(ak[x][c], e, o);
        dK[d] = (e + o) * p.scale;
        unf2(av[x][c], e, o);
        dV[d] = e + o;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// dQ = scale dS K from the dS^T scratch: one CTA per (64 query rows, head of the launch's units).
// ---------------------------------------------------------------------------------------------------------------
template <int DP>
struct SimtDq {
  static constexpr int BQ = 64, BK = 32;
  static constexpr int SMEM = (BK * BQ + BK * DP) * 4;
};

template <int DP>
__global__ void __launch_bounds__(kSimtThreads) xattn_simt_bwd_dq_kernel(const XParams p) {
  using C = SimtDq<DP>;
  extern __shared__ float4 simt_smem[];
  float* ds = reinterpret_cast<float*>(simt_smem);
  float* kn = ds + C::BK * C::BQ;
  const int nqt = (p.Nq + C::BQ - 1) / C::BQ;
  const int i0 = (blockIdx.x % nqt) * C::BQ, ul = blockIdx.x / nqt;  // ul: local (unit, head of the group)
  const int unit = p.u0 + ul / p.G, b = unit / p.Hkv, kh = unit % p.Hkv, h = kh * p.G + ul % p.G;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int n = key_count(p, b);
  const bool vk = simt_vec(p.k, p.D);
  const float* K = reinterpret_cast<const float*>(p.k.p) + b * p.k.s[0] + kh * p.k.s[1];
  const float* S = reinterpret_cast<const float*>(p.ds) + (long long)ul * p.nkp * p.nqp;
  uint64_t acc[2][DP / 16];  // pairs of queries
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) acc[r][c] = 0;
  for (int j0 = 0; j0 < n; j0 += C::BK) {
    __syncthreads();
    for (int x = threadIdx.x; x < C::BK * C::BQ / 4; x += kSimtThreads) {
      const int r = x / (C::BQ / 4), c = (x % (C::BQ / 4)) * 4;
      *reinterpret_cast<float4*>(ds + r * C::BQ + c) =
          j0 + r < n ? *reinterpret_cast<const float4*>(
                           S + ((long long)((j0 + r) / 64) * (p.nqp / 8) + (i0 + c) / 8) * 512 + (j0 + r) % 64 * 8 + c % 8)
                     : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    {
      SimtTile<C::BK, DP> x;
      x.template get<false>(K + (long long)j0 * p.k.s[2], p.k.s[2], p.D, vk, [&](int r) { return key_live(p, b, j0 + r, n); });
      x.put_n(kn);
    }
    __syncthreads();
#pragma unroll 4
    for (int j = 0; j < C::BK; ++j) {
      const ulonglong2 a2 = *reinterpret_cast<const ulonglong2*>(ds + j * C::BQ + ty * 4);
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        const float4 k4 = *reinterpret_cast<const float4*>(kn + j * DP + c * 64 + tx * 4);
        const uint64_t k[4] = {f2(k4.x, k4.x), f2(k4.y, k4.y), f2(k4.z, k4.z), f2(k4.w, k4.w)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[0][c * 4 + e] = fma2(a2.x, k[e], acc[0][c * 4 + e]);
          acc[1][c * 4 + e] = fma2(a2.y, k[e], acc[1][c * 4 + e]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = i0 + ty * 4 + r;
    if (i >= p.Nq) continue;
    float* dQ = reinterpret_cast<float*>(p.dq.p) + b * p.dq.s[0] + h * p.dq.s[1] + (long long)i * p.dq.s[2];
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      const int d = (c / 4) * 64 + tx * 4 + c % 4;
      float e, o;
      unf2(acc[r / 2][c], e, o);
      if (d < p.D) dQ[d] = (r & 1 ? o : e) * p.scale;
    }
  }
}

}  // namespace geoattn
