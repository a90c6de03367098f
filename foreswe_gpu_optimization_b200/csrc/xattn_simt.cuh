// Cross attention on the FMA pipe: fp32 storage. The tensor cores take fp32 operands only as TF32 (10 mantissa bits);
// these kernels keep every product and sum in fp32, so the results carry fp32 accuracy.
//
// Tiles sit in shared memory head-dim-major ([d][row], rows padded by 4 floats), so that a thread's 4 or 8 rows (or
// keys) are one or two 16-byte loads per d; each of the 256 threads (16 x 16) owns a register block of the product.
// Bound by the FMA pipe: per d a warp issues 32 (forward) or 32 (S and dP together) FMAs against 4-5 shared-memory
// wavefronts.
#pragma once
#include "xattn_common.cuh"

namespace geoattn {

constexpr int kSimtThreads = 256;

// dst[d][r] = row r of `src` (zero where r >= n, d >= D or !live[r]); 4 consecutive d per load where `vec`.
template <int ROWS, int DP, int ST>
__device__ __forceinline__ void simt_load_t(float* dst, const float* src, long long ld, int n, int D, bool vec,
                                            const float* live) {
  for (int x = threadIdx.x; x < ROWS * (DP / 4); x += kSimtThreads) {
    const int r = x % ROWS, d = (x / ROWS) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (r < n && d < D && (!live || live[r] == 0.f)) {
      const float* s = src + (long long)r * ld + d;
      if (vec) {
        const float4 f = *reinterpret_cast<const float4*>(s);
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (d + i < D) v[i] = s[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[(d + i) * ST + r] = v[i];
  }
}

// dst[r][d], row stride DP, as above.
template <int ROWS, int DP>
__device__ __forceinline__ void simt_load_n(float* dst, const float* src, long long ld, int n, int D, bool vec,
                                            const float* live) {
  for (int x = threadIdx.x; x < ROWS * (DP / 4); x += kSimtThreads) {
    const int r = x / (DP / 4), d = (x % (DP / 4)) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (r < n && d < D && (!live || live[r] == 0.f)) {
      const float* s = src + (long long)r * ld + d;
      if (vec) {
        const float4 f = *reinterpret_cast<const float4*>(s);
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (d + i < D) v[i] = s[i];
      }
    }
    *reinterpret_cast<float4*>(dst + r * DP + d) = make_float4(v[0], v[1], v[2], v[3]);
  }
}

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
  static constexpr int BM = 128, BN = 64, SQ = BM + 4, SK = BN + 4;
  static constexpr int FLOATS = DP * SQ + DP * SK + BN * SQ + 256 + BN;
  static constexpr int SMEM = FLOATS * 4;
};

template <int DP>
__global__ void __launch_bounds__(kSimtThreads) xattn_simt_fwd_kernel(const XParams p) {
  using C = SimtFwd<DP>;
  extern __shared__ float4 simt_smem[];
  float* qt = reinterpret_cast<float*>(simt_smem);
  float* kv = qt + DP * C::SQ;
  float* pt = kv + DP * C::SK;
  float* tab = pt + C::BN * C::SQ;
  float* live = tab + 256;
  const int nqt = (p.Nq + C::BM - 1) / C::BM;
  const int qt_i = blockIdx.x % nqt, rest = blockIdx.x / nqt;
  const int h = rest % p.H, b = (rest / p.H) % p.B, split = rest / p.H / p.B;
  const int kh = h / p.G, i0 = qt_i * C::BM, bh = b * p.H + h;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int n = key_count(p, b);
  const int ntiles = (n + C::BN - 1) / C::BN;
  const int t0 = (int)((long long)ntiles * split / p.splits), t1 = (int)((long long)ntiles * (split + 1) / p.splits);
  const float* Q = reinterpret_cast<const float*>(p.q.p) + b * p.q.s[0] + h * p.q.s[1];
  const float* K = reinterpret_cast<const float*>(p.k.p) + b * p.k.s[0] + kh * p.k.s[1];
  const float* V = reinterpret_cast<const float*>(p.v.p) + b * p.v.s[0] + kh * p.v.s[1];
  const bool vq = simt_vec(p.q, p.D), vk = simt_vec(p.k, p.D), vv = simt_vec(p.v, p.D);
  const AttnDrop drop = attn_drop(p.rng, p.drop_thr, p.drop_scale);

  if (p.ids) tab[threadIdx.x] = table_log2(p, h, threadIdx.x);
  simt_load_t<C::BM, DP, C::SQ>(qt, Q + (long long)i0 * p.q.s[2], p.q.s[2], p.Nq - i0, p.D, vq, nullptr);

  float m[8], l[8], acc[8][DP / 16];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) acc[r][c] = 0.f;
  }
  for (int t = t0; t < t1; ++t) {
    const int j0 = t * C::BN;
    __syncthreads();  // the last tile's products have read kv and pt; the first time: tab
    if (threadIdx.x < C::BN) live[threadIdx.x] = key_live(p, b, j0 + threadIdx.x, n) ? 0.f : -INFINITY;
    __syncthreads();
    simt_load_t<C::BN, DP, C::SK>(kv, K + (long long)j0 * p.k.s[2], p.k.s[2], n - j0, p.D, vk, live);
    __syncthreads();
    float s[8][4] = {};
#pragma unroll 4
    for (int d = 0; d < DP; ++d) {
      const float4 a0 = *reinterpret_cast<const float4*>(qt + d * C::SQ + ty * 8);
      const float4 a1 = *reinterpret_cast<const float4*>(qt + d * C::SQ + ty * 8 + 4);
      const float4 k4 = *reinterpret_cast<const float4*>(kv + d * C::SK + tx * 4);
      const float a[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w}, kk[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[r][c] = fmaf(a[r], kk[c], s[r][c]);
    }
    __syncthreads();  // every thread has read K
    simt_load_n<C::BN, DP>(kv, V + (long long)j0 * p.v.s[2], p.v.s[2], n - j0, p.D, vv, live);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int i = i0 + ty * 8 + r;
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = j0 + tx * 4 + c;
        float x = s[r][c] * p.scale_log2;
        if (p.ids && i < p.Nq && j < p.Nk) x += tab[p.ids[i * p.ids_ld + j]];
        s[r][c] = live[tx * 4 + c] == 0.f ? x : -INFINITY;
        mx = fmaxf(mx, s[r][c]);
      }
#pragma unroll
      for (int w = 1; w < 16; w *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float mn = fmaxf(m[r], mx), base = mn == -INFINITY ? 0.f : mn;
      const float corr = xex2(m[r] - base);
      m[r] = mn;
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[r][c] = xex2(s[r][c] - base);
        sum += s[r][c];
      }
#pragma unroll
      for (int w = 1; w < 16; w *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      l[r] = l[r] * corr + sum;
      if (drop.thr) {
        const uint32_t kb = drop.keep8(i, (j0 + tx * 4) >> 3, bh) >> ((tx & 1) * 4);
#pragma unroll
        for (int c = 0; c < 4; ++c) s[r][c] = (kb >> c) & 1 ? s[r][c] : 0.f;
      }
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) acc[r][c] *= corr;
#pragma unroll
      for (int c = 0; c < 4; ++c) pt[(tx * 4 + c) * C::SQ + ty * 8 + r] = s[r][c];
    }
    __syncthreads();
#pragma unroll 2
    for (int j = 0; j < C::BN; ++j) {
      const float4 a0 = *reinterpret_cast<const float4*>(pt + j * C::SQ + ty * 8);
      const float4 a1 = *reinterpret_cast<const float4*>(pt + j * C::SQ + ty * 8 + 4);
      const float a[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        const float4 v4 = *reinterpret_cast<const float4*>(kv + j * DP + c * 64 + tx * 4);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          acc[r][c * 4 + 0] = fmaf(a[r], v4.x, acc[r][c * 4 + 0]);
          acc[r][c * 4 + 1] = fmaf(a[r], v4.y, acc[r][c * 4 + 1]);
          acc[r][c * 4 + 2] = fmaf(a[r], v4.z, acc[r][c * 4 + 2]);
          acc[r][c * 4 + 3] = fmaf(a[r], v4.w, acc[r][c * 4 + 3]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int i = i0 + ty * 8 + r;
    if (i >= p.Nq) continue;
    const long long row = (long long)bh * p.Nq + i;
    if (p.splits > 1) {
      const long long at = (long long)split * p.B * p.H * p.Nq + row;
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        const int d = (c / 4) * 64 + tx * 4 + c % 4;
        if (d < p.D) p.part_o[at * p.D + d] = acc[r][c];
      }
      if (tx == 0) {
        p.part_ml[at * 2] = m[r];
        p.part_ml[at * 2 + 1] = l[r];
      }
    } else {
      const float inv = l[r] == 0.f ? 0.f : (drop.thr ? drop.scale : 1.f) / l[r];
      float* O = reinterpret_cast<float*>(p.o.p) + b * p.o.s[0] + h * p.o.s[1] + i * p.o.s[2];
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        const int d = (c / 4) * 64 + tx * 4 + c % 4;
        if (d < p.D) O[d] = acc[r][c] * inv;
      }
      if (tx == 0 && p.stats) p.stats[row] = row_stats(m[r], l[r]);
    }
  }
}

// Join the key splits of each row: one warp per row.
template <class E>
__global__ void __launch_bounds__(256) xattn_combine_kernel(const XParams p) {
  const long long rows = (long long)p.B * p.H * p.Nq;
  const long long row = (long long)blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (row >= rows) return;
  float m = -INFINITY;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.part_ml[(s * rows + row) * 2]);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const float* ml = p.part_ml + (s * rows + row) * 2;
    l += ml[1] * xex2(ml[0] - base);
  }
  const float inv = l == 0.f ? 0.f : (p.drop_thr ? p.drop_scale : 1.f) / l;
  const int i = (int)(row % p.Nq), bh = (int)(row / p.Nq), h = bh % p.H, b = bh / p.H;
  E* O = reinterpret_cast<E*>(p.o.p) + b * p.o.s[0] + h * p.o.s[1] + i * p.o.s[2];
  for (int d = lane; d < p.D; d += 32) {
    float x = 0.f;
    for (int s = 0; s < p.splits; ++s)
      x += p.part_o[(s * rows + row) * p.D + d] * xex2(p.part_ml[(s * rows + row) * 2] - base);
    O[d] = from_f<E>(x * inv);
  }
  if (lane == 0 && p.stats) p.stats[row] = row_stats(m, l);
}

// delta_i = dO_i . O_i, one warp per row.
__global__ void __launch_bounds__(256) xattn_delta_kernel(const XParams p) {
  const long long rows = (long long)p.B * p.H * p.Nq;
  const long long row = (long long)blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (row >= rows) return;
  const int i = (int)(row % p.Nq), bh = (int)(row / p.Nq), h = bh % p.H, b = bh / p.H;
  const float* O = reinterpret_cast<const float*>(p.o.p) + b * p.o.s[0] + h * p.o.s[1] + i * p.o.s[2];
  const float* G = reinterpret_cast<const float*>(p.dout.p) + b * p.dout.s[0] + h * p.dout.s[1] + i * p.dout.s[2];
  float x = 0.f;
  for (int d = lane; d < p.D; d += 32) x = fmaf(O[d], G[d], x);
#pragma unroll
  for (int w = 16; w; w /= 2) x += __shfl_xor_sync(0xffffffffu, x, w);
  if (lane == 0) p.delta[row] = x;
}

// ---------------------------------------------------------------------------------------------------------------
// Backward, key pass: one CTA per (TK keys, key head, batch); loops over the heads that share the key head and their
// 64-row query tiles. dK and dV stay in registers (no atomics: fixed order); dS^T goes to the scratch.
// ---------------------------------------------------------------------------------------------------------------
template <int DP>
struct SimtBwd {
  static constexpr int TK = DP <= 128 ? 64 : 32, KT = TK / 16, BQ = 64, SK = TK + 4, SQ = BQ + 4;
  static constexpr int FLOATS = 2 * DP * SK + 2 * DP * SQ + 2 * TK * SQ + 256 + TK + 3 * BQ;
  static constexpr int SMEM = FLOATS * 4;
};

template <int DP>
__global__ void __launch_bounds__(kSimtThreads) xattn_simt_bwd_keys_kernel(const XParams p) {
  using C = SimtBwd<DP>;
  constexpr int KT = C::KT, NC = DP / 16;
  extern __shared__ float4 simt_smem[];
  float* kt = reinterpret_cast<float*>(simt_smem);
  float* vt = kt + DP * C::SK;
  float* qt = vt + DP * C::SK;
  float* gt = qt + DP * C::SQ;
  float* pt = gt + DP * C::SQ;
  float* st = pt + C::TK * C::SQ;
  float* tab = st + C::TK * C::SQ;
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
  float ak[KT][NC], av[KT][NC];
#pragma unroll
  for (int x = 0; x < KT; ++x)
#pragma unroll
    for (int c = 0; c < NC; ++c) ak[x][c] = av[x][c] = 0.f;

  if (j0 < n) {
    if (threadIdx.x < C::TK) live[threadIdx.x] = key_live(p, b, j0 + threadIdx.x, n) ? 0.f : -INFINITY;
    __syncthreads();
    const float* K = reinterpret_cast<const float*>(p.k.p) + b * p.k.s[0] + kh * p.k.s[1] + (long long)j0 * p.k.s[2];
    const float* V = reinterpret_cast<const float*>(p.v.p) + b * p.v.s[0] + kh * p.v.s[1] + (long long)j0 * p.v.s[2];
    simt_load_t<C::TK, DP, C::SK>(kt, K, p.k.s[2], n - j0, p.D, simt_vec(p.k, p.D), live);
    simt_load_t<C::TK, DP, C::SK>(vt, V, p.v.s[2], n - j0, p.D, simt_vec(p.v, p.D), live);
    const int nqt = (p.Nq + C::BQ - 1) / C::BQ;
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
      simt_load_t<C::BQ, DP, C::SQ>(qt, Q, p.q.s[2], p.Nq - i0, p.D, simt_vec(p.q, p.D), nullptr);
      simt_load_t<C::BQ, DP, C::SQ>(gt, G, p.dout.s[2], p.Nq - i0, p.D, simt_vec(p.dout, p.D), nullptr);
      __syncthreads();
      float s[4][KT] = {}, dp[4][KT] = {};
#pragma unroll 4
      for (int d = 0; d < DP; ++d) {
        const float4 q4 = *reinterpret_cast<const float4*>(qt + d * C::SQ + ty * 4);
        const float4 g4 = *reinterpret_cast<const float4*>(gt + d * C::SQ + ty * 4);
        const float a[4] = {q4.x, q4.y, q4.z, q4.w}, g[4] = {g4.x, g4.y, g4.z, g4.w};
        float kk[KT], vv[KT];
#pragma unroll
        for (int c = 0; c < KT; c += 2) {
          const float2 k2 = *reinterpret_cast<const float2*>(kt + d * C::SK + tx * KT + c);
          const float2 v2 = *reinterpret_cast<const float2*>(vt + d * C::SK + tx * KT + c);
          kk[c] = k2.x, kk[c + 1] = k2.y, vv[c] = v2.x, vv[c + 1] = v2.y;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < KT; ++c) {
            s[r][c] = fmaf(a[r], kk[c], s[r][c]);
            dp[r][c] = fmaf(g[r], vv[c], dp[r][c]);
          }
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
      float* ds = reinterpret_cast<float*>(p.ds) + (long long)(ul * p.G + it / nqt) * p.nkp * p.nqp +
                  ((long long)(j0 / 64) * (p.nqp / 8) + (i0 + ty * 4) / 8) * 512 + (ty & 1) * 4;
#pragma unroll
      for (int c = 0; c < KT; ++c) {
        const float4 a4 = make_float4(s[0][c], s[1][c], s[2][c], s[3][c]);
        const float4 d4 = make_float4(dp[0][c], dp[1][c], dp[2][c], dp[3][c]);
        *reinterpret_cast<float4*>(pt + (tx * KT + c) * C::SQ + ty * 4) = a4;
        *reinterpret_cast<float4*>(st + (tx * KT + c) * C::SQ + ty * 4) = d4;
        *reinterpret_cast<float4*>(ds + (j0 % 64 + tx * KT + c) * 8) = d4;
      }
      __syncthreads();
#pragma unroll 2
      for (int r = 0; r < C::BQ; r += 4) {
        float4 pp[KT], ss[KT];
#pragma unroll
        for (int x = 0; x < KT; ++x) {
          pp[x] = *reinterpret_cast<const float4*>(pt + (ty * KT + x) * C::SQ + r);
          ss[x] = *reinterpret_cast<const float4*>(st + (ty * KT + x) * C::SQ + r);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float4 g4 = *reinterpret_cast<const float4*>(gt + (tx + 16 * c) * C::SQ + r);
          const float4 q4 = *reinterpret_cast<const float4*>(qt + (tx + 16 * c) * C::SQ + r);
#pragma unroll
          for (int x = 0; x < KT; ++x) {
            av[x][c] = fmaf(pp[x].x, g4.x, fmaf(pp[x].y, g4.y, fmaf(pp[x].z, g4.z, fmaf(pp[x].w, g4.w, av[x][c]))));
            ak[x][c] = fmaf(ss[x].x, q4.x, fmaf(ss[x].y, q4.y, fmaf(ss[x].z, q4.z, fmaf(ss[x].w, q4.w, ak[x][c]))));
          }
        }
      }
    }
  }
#pragma unroll
  for (int x = 0; x < KT; ++x) {
    const int j = j0 + ty * KT + x;
    if (j >= p.Nk) continue;
    float* dK = reinterpret_cast<float*>(p.dk.p) + b * p.dk.s[0] + kh * p.dk.s[1] + (long long)j * p.dk.s[2];
    float* dV = reinterpret_cast<float*>(p.dv.p) + b * p.dv.s[0] + kh * p.dv.s[1] + (long long)j * p.dv.s[2];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = tx + 16 * c;
      if (d < p.D) {
        dK[d] = ak[x][c] * p.scale;
        dV[d] = av[x][c];
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
  static constexpr int SMEM = (BK * BQ + BK * DP + BK) * 4;
};

template <int DP>
__global__ void __launch_bounds__(kSimtThreads) xattn_simt_bwd_dq_kernel(const XParams p) {
  using C = SimtDq<DP>;
  extern __shared__ float4 simt_smem[];
  float* ds = reinterpret_cast<float*>(simt_smem);
  float* kn = ds + C::BK * C::BQ;
  float* live = kn + C::BK * DP;
  const int nqt = (p.Nq + C::BQ - 1) / C::BQ;
  const int i0 = (blockIdx.x % nqt) * C::BQ, ul = blockIdx.x / nqt;  // ul: local (unit, head of the group)
  const int unit = p.u0 + ul / p.G, b = unit / p.Hkv, kh = unit % p.Hkv, h = kh * p.G + ul % p.G;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int n = key_count(p, b);
  const float* K = reinterpret_cast<const float*>(p.k.p) + b * p.k.s[0] + kh * p.k.s[1];
  const float* S = reinterpret_cast<const float*>(p.ds) + (long long)ul * p.nkp * p.nqp;
  float acc[4][DP / 16];
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) acc[r][c] = 0.f;
  for (int j0 = 0; j0 < n; j0 += C::BK) {
    __syncthreads();
    if (threadIdx.x < C::BK) live[threadIdx.x] = key_live(p, b, j0 + threadIdx.x, n) ? 0.f : -INFINITY;
    for (int x = threadIdx.x; x < C::BK * C::BQ / 4; x += kSimtThreads) {
      const int r = x / (C::BQ / 4), c = (x % (C::BQ / 4)) * 4;
      *reinterpret_cast<float4*>(ds + r * C::BQ + c) =
          j0 + r < n ? *reinterpret_cast<const float4*>(
                           S + ((long long)((j0 + r) / 64) * (p.nqp / 8) + (i0 + c) / 8) * 512 + (j0 + r) % 64 * 8 + c % 8)
                     : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
    simt_load_n<C::BK, DP>(kn, K + (long long)j0 * p.k.s[2], p.k.s[2], n - j0, p.D, simt_vec(p.k, p.D), live);
    __syncthreads();
#pragma unroll 4
    for (int j = 0; j < C::BK; ++j) {
      const float4 a4 = *reinterpret_cast<const float4*>(ds + j * C::BQ + ty * 4);
      const float a[4] = {a4.x, a4.y, a4.z, a4.w};
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        const float4 k4 = *reinterpret_cast<const float4*>(kn + j * DP + c * 64 + tx * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          acc[r][c * 4 + 0] = fmaf(a[r], k4.x, acc[r][c * 4 + 0]);
          acc[r][c * 4 + 1] = fmaf(a[r], k4.y, acc[r][c * 4 + 1]);
          acc[r][c * 4 + 2] = fmaf(a[r], k4.z, acc[r][c * 4 + 2]);
          acc[r][c * 4 + 3] = fmaf(a[r], k4.w, acc[r][c * 4 + 3]);
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
      if (d < p.D) dQ[d] = acc[r][c] * p.scale;
    }
  }
}

}  // namespace geoattn
