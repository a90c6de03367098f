// Cross attention on the tensor cores (bf16): TMA-fed 128-byte-swizzled tiles, tcgen05 products with fp32 accumulators
// in tensor memory. Shared-memory tiles are regions of rows x 128 bytes (64 head-dim columns), one region per 64
// columns of the padded head dim DP (64, 128, 192); TMA fills rows and columns past the tensor with zeros.
//
// Every product has M = 128 (the rows of a tile sit in the 128 lanes of tensor memory, one thread per row), and the
// CTAs are sized so that two share an SM (at most 256 tensor-memory columns and 113 KB each): one CTA's element-wise
// work overlaps the other's products, loads, prologue and epilogue.
#pragma once
#include "sm100.cuh"
#include "xattn_common.cuh"

namespace geoattn {
namespace xa {

extern __shared__ __align__(1024) uint8_t xsmem[];

struct XMaps {
  CUtensorMap q, k, v, dout, ds;
};

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const WaitCtx& ctx) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, ctx));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// NKB regions of `rows` x 128 bytes.
template <int DP>
__device__ __forceinline__ void load_rows(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int region, int row,
                                          int h, int b) {
#pragma unroll
  for (int kb = 0; kb < DP / 64; ++kb) tma_load_4d(dst + kb * region, map, bar, kb * 64, row, h, b);
}

// acc[128 x 64] = A[128 x DP] B[64 x DP]^T, both K-major: the score-shaped product.
template <int DP>
__device__ __forceinline__ void mma_scores(uint32_t acc, uint32_t a, uint32_t b) {
  constexpr uint32_t idesc = instr_desc(1, 0, 0, 128, 64);
#pragma unroll
  for (int kb = 0; kb < DP / 64; ++kb)
#pragma unroll
    for (int s = 0; s < 4; ++s)
      mma_ss<Kind::kF16>(acc, smem_desc_sw128(a + kb * (128 * 128) + s * 32, 16, 1024),
                         smem_desc_sw128(b + kb * (64 * 128) + s * 32, 16, 1024), idesc, kb + s > 0);
}

// acc[128 x DP] (+)= A[128 x 64] B[64 x DP]: A in tensor memory (two bf16 per column), B with its rows along K.
template <int DP>
__device__ __forceinline__ void mma_weights(uint32_t acc, uint32_t a, uint32_t b, bool accumulate) {
  constexpr uint32_t idesc = instr_desc(1, 0, 1, 128, DP);
#pragma unroll
  for (int s = 0; s < 4; ++s)
    mma_ts<Kind::kF16>(acc, a + s * 8, smem_desc_sw128(b + s * 16 * 128, 64 * 128, 1024), idesc, accumulate || s > 0);
}

// Set row `r` of a 64-row tile to zero.
template <int DP>
__device__ __forceinline__ void clear_row(uint8_t* tile, int r) {
#pragma unroll
  for (int kb = 0; kb < DP / 64; ++kb)
#pragma unroll
    for (int c = 0; c < 8; ++c)
      *reinterpret_cast<uint4*>(tile + kb * (64 * 128) + r * 128 + c * 16) = make_uint4(0, 0, 0, 0);
}

// Liveness of 64 keys from j0 on as two words, the same in every lane of the warp.
__device__ __forceinline__ void live_words(const XParams& p, int b, int j0, int n, uint32_t (&w)[2]) {
  const int lane = threadIdx.x & 31;
  w[0] = __ballot_sync(0xffffffffu, key_live(p, b, j0 + lane, n));
  w[1] = __ballot_sync(0xffffffffu, key_live(p, b, j0 + 32 + lane, n));
}

template <int N>
__device__ __forceinline__ void store_row(__nv_bfloat16* dst, const float (&v)[N], float f, int D, bool vec) {
  // N consecutive columns of one row, of which D exist
#pragma unroll
  for (int c = 0; c < N; c += 8) {
    if (vec && c + 8 <= D) {
      *reinterpret_cast<uint4*>(dst + c) =
          make_uint4(pack_bf16(v[c] * f, v[c + 1] * f), pack_bf16(v[c + 2] * f, v[c + 3] * f),
                     pack_bf16(v[c + 4] * f, v[c + 5] * f), pack_bf16(v[c + 6] * f, v[c + 7] * f));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < D) dst[c + e] = __float2bfloat16_rn(v[c + e] * f);
    }
  }
}
__device__ __forceinline__ bool vec_rows(const XTensor& t) {
  return ((reinterpret_cast<uintptr_t>(t.p) | (uintptr_t)(t.s[0] * 2) | (uintptr_t)(t.s[1] * 2) |
           (uintptr_t)(t.s[2] * 2)) & 15) == 0;
}

// ---------------------------------------------------------------------------------------------------------------
// Forward. One CTA per (128 query rows, head, batch, key split), keys in chunks of 64:
//   MMA warp   S(c + 1) = Q K^T into the other score buffer, then O += P(c) V(c)
//   4 warps    P(c) = 2^(t - m), a row per thread; bf16, written over its scores
// The running maximum moves only when it would grow by more than 2^kLazy (P stays below that, l and O are fp32), so O
// is rescaled rarely; it then waits for O's product c - 1, the only one that can be in flight there (S(c) was issued
// after product c - 2).
// Few queries of heads that share a key head (G * Nq <= 128) are packed into one tile's rows.
// DP = 192 has room for one score buffer and one chunk of K and V; S(c + 1) then follows O's product c.
// ---------------------------------------------------------------------------------------------------------------
template <int DP>
struct FwdCfg {
  static constexpr int NSB = DP == 192 ? 1 : 2;              // score buffers
  static constexpr int NKV = DP == 192 ? 1 : DP == 128 ? 2 : 4;  // chunks of K, and of V, in flight
  static constexpr int Q_BYTES = DP / 64 * 128 * 128, KV_BYTES = DP / 64 * 64 * 128;
  static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + NKV * KV_BYTES, OFF_TAB = OFF_V + NKV * KV_BYTES;
  static constexpr int SMEM = OFF_TAB + 1024;
  static constexpr int TM_S = 0, TM_O = NSB * 64, TM_COLS = 256;
  static constexpr int THREADS = 192, TMA_WARP = 4, MMA_WARP = 5;
};
constexpr float kLazy = 8.f;

template <int DP, bool BIAS>
__global__ void __launch_bounds__(192, 2) xattn_fwd_kernel(const __grid_constant__ XMaps maps, const XParams p) {
  using C = FwdCfg<DP>;
  constexpr int NKV = C::NKV, NSB = C::NSB;
  __shared__ uint64_t bar_q, bar_kfull[NKV], bar_kempty[NKV], bar_vfull[NKV], bar_vempty[NKV], bar_s[NSB], bar_p[NSB], bar_pv[2];
  __shared__ uint32_t tmem_sh;
  __shared__ int abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const bool pack = p.pack != 0;
  const int nqt = pack ? 1 : (p.Nq + 127) / 128, nh = pack ? p.Hkv : p.H;
  const int qt = blockIdx.x % nqt, rest = blockIdx.x / nqt;
  const int hx = rest % nh, b = (rest / nh) % p.B, split = rest / nh / p.B;
  const int kh = pack ? hx : hx / p.G;
  const int n = key_count(p, b);
  const int all = (n + 63) / 64;
  const int c0 = (int)((long long)all * split / p.splits), nc = (int)((long long)all * (split + 1) / p.splits) - c0;
  WaitCtx ctx{&abort_flag, p.status};

  if (threadIdx.x == 0) {
    // a wait gives up after 2 s at the earliest, long after the first CTA has started
    if (blockIdx.x == 0) *p.status = kDevOk;
    abort_flag = 0;
    mbar_init(&bar_q, 1);
    for (int i = 0; i < NKV; ++i) {
      mbar_init(&bar_kfull[i], 1);
      mbar_init(&bar_kempty[i], 1);
      mbar_init(&bar_vfull[i], 1);
      mbar_init(&bar_vempty[i], 1);
    }
    for (int i = 0; i < NSB; ++i) {
      mbar_init(&bar_s[i], 1);
      mbar_init(&bar_p[i], 128);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&bar_pv[i], 1);
    fence_barrier_init();
  }
  if (warp == C::MMA_WARP) {
    tmem_alloc(&tmem_sh, C::TM_COLS);
    tmem_relinquish();
  }
  float* tab = reinterpret_cast<float*>(xsmem + C::OFF_TAB);
  if (BIAS)
    for (int t = threadIdx.x; t < 256; t += C::THREADS) tab[t] = table_log2(p, hx, t);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_sh, sbase = smem_u32(xsmem);

  if (warp == C::TMA_WARP) {
    if (lane == 0 && nc > 0) {
      if (pack) {
        mbar_arrive_expect_tx(&bar_q, DP / 64 * p.G * p.Nq * 128);
        load_rows<DP>(xsmem, &maps.q, &bar_q, 128 * 128, 0, kh * p.G, b);
      } else {
        mbar_arrive_expect_tx(&bar_q, C::Q_BYTES);
        load_rows<DP>(xsmem, &maps.q, &bar_q, 128 * 128, qt * 128, hx, b);
      }
      for (int c = 0; c < nc; ++c) {
        const int st = c % NKV;
        const uint32_t par = ((c / NKV) & 1) ^ 1;
        if (!mbar_wait(&bar_kempty[st], par, ctx)) break;
        mbar_arrive_expect_tx(&bar_kfull[st], C::KV_BYTES);
        load_rows<DP>(xsmem + C::OFF_K + st * C::KV_BYTES, &maps.k, &bar_kfull[st], 64 * 128, (c0 + c) * 64, kh, b);
        if (!mbar_wait(&bar_vempty[st], par, ctx)) break;
        mbar_arrive_expect_tx(&bar_vfull[st], C::KV_BYTES);
        load_rows<DP>(xsmem + C::OFF_V + st * C::KV_BYTES, &maps.v, &bar_vfull[st], 64 * 128, (c0 + c) * 64, kh, b);
      }
    }
  } else if (warp == C::MMA_WARP) {
    if (lane == 0 && nc > 0) {
      bool ok = mbar_wait(&bar_q, 0, ctx);
      auto scores = [&](int c) {
        const int st = c % NKV;
        if (!(ok = ok && mbar_wait(&bar_kfull[st], (c / NKV) & 1, ctx))) return;
        tc_fence_after();
        mma_scores<DP>(tmem + C::TM_S + (c % NSB) * 64, sbase, sbase + C::OFF_K + st * C::KV_BYTES);
        mma_commit(&bar_s[c % NSB]);
        mma_commit(&bar_kempty[st]);
      };
      scores(0);
      for (int c = 0; c < nc && ok; ++c) {
        if (NSB == 2 && c + 1 < nc) scores(c + 1);
        const int st = c % NKV;
        if (!(ok = ok && mbar_wait(&bar_p[c % NSB], (c / NSB) & 1, ctx) && mbar_wait(&bar_vfull[st], (c / NKV) & 1, ctx))) break;
        tc_fence_after();
        mma_weights<DP>(tmem + C::TM_O, tmem + C::TM_S + (c % NSB) * 64, sbase + C::OFF_V + st * C::KV_BYTES, c > 0);
        mma_commit(&bar_vempty[st]);
        mma_commit(&bar_pv[c & 1]);
        if (NSB == 1 && c + 1 < nc) scores(c + 1);
      }
    }
  } else {
    const int r = warp * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    const int i = pack ? r % p.Nq : qt * 128 + r;
    const int h = pack ? kh * p.G + r / p.Nq : hx;
    const bool row = pack ? r < p.G * p.Nq : i < p.Nq;
    const bool any_row = __any_sync(0xffffffffu, row);
    const int bh = b * p.H + h;
    const AttnDrop drop = attn_drop(p.rng, p.drop_thr, p.drop_scale);
    const uint8_t* idrow = BIAS ? p.ids + (long long)(row ? i : 0) * p.ids_ld : nullptr;
    const bool check_keys = p.kmask != nullptr;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int c = 0; c < nc; ++c) {
      const int j0 = (c0 + c) * 64;
      uint32_t live[2] = {~0u, ~0u};
      if (check_keys || j0 + 64 > n) live_words(p, b, j0, n, live);
      uint4 id4[4];
      if (BIAS) {  // 16 ids per load; the last ones of a row may lie past Nk: excluded
#pragma unroll
        for (int x = 0; x < 4; ++x)
          id4[x] = j0 + x * 16 < p.Nk ? __ldg(reinterpret_cast<const uint4*>(idrow + j0) + x)
                                      : make_uint4(~0u, ~0u, ~0u, ~0u);
      }
      const uint32_t sbuf = lanes + C::TM_S + (c % NSB) * 64;
      if (ok) ok = warp_wait(&bar_s[c % NSB], (c / NSB) & 1, ctx);
      if (!ok) break;
      tc_fence_after();
      if (any_row) {
        uint32_t lo[32], hi[32];
        tmem_ld32_issue(sbuf, lo);
        tmem_ld32_issue(sbuf + 32, hi);
        tmem_wait32(lo);
        tmem_pin32(hi);
        float x[64];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          x[e] = __uint_as_float(lo[e]);
          x[e + 32] = __uint_as_float(hi[e]);
        }
        if (BIAS) {
          const uint32_t* w = reinterpret_cast<const uint32_t*>(id4);
#pragma unroll
          for (int e = 0; e < 64; ++e) x[e] = fmaf(x[e], p.scale_log2, tab[(w[e / 4] >> (8 * (e % 4))) & 255]);
        }
        if ((live[0] & live[1]) != ~0u) {
#pragma unroll
          for (int e = 0; e < 64; ++e)
            if (!((live[e / 32] >> (e % 32)) & 1)) x[e] = -INFINITY;
        }
        float mx = x[0];
#pragma unroll
        for (int e = 1; e < 64; ++e) mx = fmaxf(mx, x[e]);
        if (!BIAS) mx *= p.scale_log2;  // x is still the raw product (scale > 0: the order and -inf stay)
        const bool grow = mx > m + kLazy || (m == -INFINITY && mx > m);
        if (__any_sync(0xffffffffu, grow && l > 0.f)) {  // O holds something to rescale
          if (!(ok = warp_wait(&bar_pv[(c - 1) & 1], ((c - 1) >> 1) & 1, ctx))) break;
          tc_fence_after();
          const float f = grow ? xex2(m - mx) : 1.f;
          l *= f;
#pragma unroll 1
          for (int d = 0; d < DP; d += 16) {
            uint32_t o[16];
            tmem_ld16_issue(lanes + C::TM_O + d, o);
            tmem_wait16(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st16(lanes + C::TM_O + d, o);
          }
          tmem_wait_st();
        }
        if (grow) m = mx;
        const float base = m == -INFINITY ? 0.f : m;
        float sum = 0.f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t w[16];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float t = x[half * 32 + g * 8 + e];
              v[e] = xex2(BIAS ? t - base : fmaf(t, p.scale_log2, -base));
              sum += v[e];
            }
            if (drop.thr) {
              const uint32_t keep = drop.keep8(i, (j0 >> 3) + half * 4 + g, bh);
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = (keep >> e) & 1 ? v[e] : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) w[g * 4 + e] = pack_bf16(v[2 * e], v[2 * e + 1]);
          }
          tmem_st16(sbuf + half * 16, w);
        }
        l += sum;
        tmem_wait_st();
      }
      if ((live[0] & live[1]) != ~0u) {  // what absent keys hold must not reach the product: 0 * NaN
        if (!(ok = warp_wait(&bar_vfull[c % NKV], (c / NKV) & 1, ctx))) break;
        if (r < 64 && !((live[r / 32] >> (r % 32)) & 1)) {
          clear_row<DP>(xsmem + C::OFF_V + (c % NKV) * C::KV_BYTES, r);
          fence_proxy_async_smem();
        }
      }
      tc_fence_before();
      mbar_arrive(&bar_p[c % NSB]);
    }
    if (ok && nc > 0) ok = warp_wait(&bar_pv[(nc - 1) & 1], ((nc - 1) >> 1) & 1, ctx);
    tc_fence_after();
    const long long stat = (long long)bh * p.Nq + i;
    const long long part = (long long)split * p.B * p.H * p.Nq + stat;
    const float f = l == 0.f ? 0.f : (p.drop_thr ? p.drop_scale : 1.f) / l;
    const bool vec = vec_rows(p.o);
    if (ok && any_row) {
#pragma unroll 1
      for (int d = 0; d < DP; d += 32) {
        float o[32];
        if (nc > 0) {
          tmem_ld32(lanes + C::TM_O + d, o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
        }
        if (!row || d >= p.D) continue;
        if (p.splits > 1) {
          float* dst = p.part_o + part * p.D + d;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (d + e < p.D) dst[e] = l == 0.f ? 0.f : o[e];
        } else {
          __nv_bfloat16* dst =
              reinterpret_cast<__nv_bfloat16*>(p.o.p) + b * p.o.s[0] + h * p.o.s[1] + (long long)i * p.o.s[2] + d;
          if (l == 0.f) {  // a row with nothing left
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
          store_row(dst, o, f, p.D - d, vec);
        }
      }
      if (row && p.splits > 1) {
        p.part_ml[part * 2] = m;
        p.part_ml[part * 2 + 1] = l;
      } else if (row && p.stats) {
        p.stats[stat] = row_stats(m, l);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::MMA_WARP) tmem_dealloc(tmem, C::TM_COLS);
}

}  // namespace xa
}  // namespace geoattn
