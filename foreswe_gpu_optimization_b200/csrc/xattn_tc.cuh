// Cross attention on the tensor cores (bf16): TMA-fed 128-byte-swizzled tiles, tcgen05 products with fp32 accumulators
// in tensor memory. Shared-memory tiles are regions of rows x 128 bytes (64 head-dim columns), one region per 64
// columns of the padded head dim DP (64, 128, 192); TMA fills rows and columns past the tensor with zeros.
//
// Every product has M = 128 (the rows of a tile sit in the 128 lanes of tensor memory, one thread per row). The CTAs of
// the forward and of dQ are sized so that two share an SM (at most 256 tensor-memory columns and 113 KB each): one CTA's
// element-wise work overlaps the other's products, loads, prologue and epilogue. The key pass fills tensor memory with
// one CTA and is persistent instead.
//
// Times are of single launches at the burst clock; BxHxNqxNkxD gives the sizes.
#pragma once
#include "sm100.cuh"
#include "xattn_common.cuh"

namespace geoattn {
namespace xa {

extern __shared__ __align__(1024) uint8_t xsmem[];

struct XMaps {
  CUtensorMap q, k, v, dout, o, dq, dk, dv;
};

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const WaitCtx& ctx) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, ctx));
}

// Barrier `id` among `threads` threads.
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Barrier `id` among `threads` threads that also tells each whether any of them said yes.
__device__ __forceinline__ bool named_any(int id, int threads, bool yes) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbarrier.cta.red.or.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"((uint32_t)yes)
      : "memory");
  return r != 0;
}

// The bias of the pair with byte offset `id`, from the table at `off` in shared memory.
__device__ __forceinline__ float table_at(int off, uint32_t id) { return *reinterpret_cast<const float*>(xsmem + off + id); }
__device__ __forceinline__ uint64_t table_pair(int off, uint32_t w) {
  return f2(table_at(off, w & 0xFFFF), table_at(off, w >> 16));
}

// NKB regions of `rows` x 128 bytes.
template <int DP>
__device__ __forceinline__ void load_rows(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int region, int row,
                                          int h, int b) {
#pragma unroll
  for (int kb = 0; kb < DP / 64; ++kb) tma_load_4d(dst + kb * region, map, bar, kb * 64, row, h, b);
}

// Descriptor of an operand without swizzle, M or N contiguous: 8 x 8 matrices of 8 rows (along K) x 16 bytes, `lbo`
// bytes apart along K and `sbo` along M or N.
__device__ __forceinline__ uint64_t smem_desc_plain(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)((lbo >> 4) & 0x3FFF) << 16 |
         (uint64_t)((sbo >> 4) & 0x3FFF) << 32 | (uint64_t)1 << 46;
}

// acc[128 x N] = A[128 x DP] B[N x DP]^T, both K-major: the score-shaped product. An instruction reads its operands from
// shared memory at 128 bytes per clock (A 4 KB, B 32 N bytes for K = 16), so N = 64 takes 48 clocks and N = 128 takes 64.
template <int DP, int N>
__device__ __forceinline__ void mma_scores(uint32_t acc, uint32_t a, uint32_t b) {
  constexpr uint32_t idesc = instr_desc(1, 0, 0, 128, N);
#pragma unroll
  for (int kb = 0; kb < DP / 64; ++kb)
#pragma unroll
    for (int s = 0; s < 4; ++s)
      mma_ss<Kind::kF16>(acc, smem_desc_sw128(a + kb * (128 * 128) + s * 32, 16, 1024),
                         smem_desc_sw128(b + kb * (N * 128) + s * 32, 16, 1024), idesc, kb + s > 0);
}

// acc[128 x DP] (+)= A[128 x K] B[K x DP]: A in tensor memory (two bf16 per column), each piece of PIECE (16 or 32)
// columns at the start of the score columns that it replaces (another warpgroup may still read its own); B with its rows
// along K.
template <int DP, int K, int PIECE>
__device__ __forceinline__ void mma_pieces(uint32_t acc, uint32_t a, uint32_t b, bool accumulate) {
  constexpr uint32_t idesc = instr_desc(1, 0, 1, 128, DP);
#pragma unroll
  for (int s = 0; s < K / 16; ++s)
    mma_ts<Kind::kF16>(acc, a + (s * 16 / PIECE) * PIECE + (s * 16 % PIECE) / 2, smem_desc_sw128(b + s * 16 * 128, K * 128, 1024), idesc,
                       accumulate || s > 0);
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
// 32 columns d0 .. d0 + 31 of row r, in bf16, into a 128-row tile for a TMA store (regions of 64 columns).
__device__ __forceinline__ void stage_row32(uint8_t* tile, int r, int d0, const float (&v)[32], float f) {
  uint8_t* dst = tile + (d0 / 64) * (128 * 128) + (r >> 3) * 1024 + (r & 7) * 128;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *reinterpret_cast<uint4*>(dst + ((((d0 % 64) / 8 + c) ^ (r & 7)) << 4)) =
        make_uint4(pack_bf16(v[8 * c] * f, v[8 * c + 1] * f), pack_bf16(v[8 * c + 2] * f, v[8 * c + 3] * f),
                   pack_bf16(v[8 * c + 4] * f, v[8 * c + 5] * f), pack_bf16(v[8 * c + 6] * f, v[8 * c + 7] * f));
}
// The staged tile leaves (one thread, after a barrier of the threads that staged it and their proxy fence).
template <int DP>
__device__ __forceinline__ void store_tile(const CUtensorMap* map, const uint8_t* tile, int D, int row, int h, int b) {
  for (int kb = 0; kb < DP / 64 && kb * 64 < D; ++kb)
    tma_store_4d(map, tile + kb * (128 * 128), kb * 64, row, h, b);
  bulk_commit();
}

__device__ __forceinline__ bool vec_rows(const XTensor& t) {
  return ((reinterpret_cast<uintptr_t>(t.p) | (uintptr_t)(t.s[0] * 2) | (uintptr_t)(t.s[1] * 2) |
           (uintptr_t)(t.s[2] * 2)) & 15) == 0;
}

// ---------------------------------------------------------------------------------------------------------------
// Forward. One CTA per (128 query rows, head, batch, key split), keys in chunks of 64:
//   MMA warp       S(c + 1) = Q K^T into the other score buffer, then O += P(c) V(c)
//   2 warpgroups   P(c) = 2^(t - m): thread r of warpgroup w has row r and keys 32 w .. 32 w + 31 of the chunk; P goes
//                  in bf16 over the scores it came from
// m is one per row and moves only when a chunk would pass it by more than kLazy (P stays below 2^kLazy; l and O are
// fp32): one barrier per chunk tells the two warps of 32 rows whether any of them has to move, and only then do they
// exchange their maxima and rescale O, after O's product c - 1 (the only one that can be in flight: S(c) was issued
// after c - 2).
// Few queries of heads that share a key head (G * Nq <= 128) are packed into one tile's rows, each with its head's bias
// table.
// DP = 192 has room for one score buffer and one chunk of K and V; S(c + 1) then follows O's product c.
// Measured: 256x16x512x512x128 with the bias 886 us (620 TFLOP/s, 2.8x its products' time), 32x16x700x512x64 with the
// bias and a mask 192 us, 1x8x4096x8192x128 160 us (859 TFLOP/s; 237 with dropout), 32x16x512x512x192 with bias and
// dropout 255 us: bound by the products' operand feed (a 64-key score product reads as many shared-memory bytes as it has
// time for) and the chain from scores to weights. 16x(32/8)x4x16384x128 with lengths 146 us: 5.3 TB/s of K and V.
// 128-key chunks, one warpgroup per tile, a barrier per half of P, and maxima exchanged a chunk ahead were built and were
// 5 to 25 % slower at D = 128.
// ---------------------------------------------------------------------------------------------------------------
template <int DP>
struct FwdCfg {
  static constexpr int NSB = DP == 192 ? 1 : 2;                  // score buffers
  static constexpr int NKV = DP == 192 ? 1 : DP == 128 ? 2 : 4;  // chunks of K, and of V, in flight
  static constexpr int Q_BYTES = DP / 64 * 128 * 128, KV_BYTES = DP / 64 * 64 * 128;
  static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + NKV * KV_BYTES, OFF_TAB = OFF_V + NKV * KV_BYTES;
  static constexpr int OFF_ROW = OFF_TAB + 4224;                 // [2][128] floats: what the warpgroups exchange
  static constexpr int SMEM = OFF_ROW + 1024;
  static constexpr int TM_S = 0, TM_O = NSB * 64, TM_COLS = 256;
  static constexpr int EWT = 256, THREADS = EWT + 64, TMA_WARP = 8, MMA_WARP = 9;
};
constexpr float kLazy = 8.f;
constexpr int kPackTables = 16;                     // heads of a packed tile that has a bias
constexpr int kTableBytes = (kMaxBuckets + 1) * 4;  // -inf behind the buckets
static_assert(kPackTables * kTableBytes <= 4224, "");

// BIAS: 0 none, 1 the head's table, 2 a packed tile's tables (a row has its head's)
template <int DP, int BIAS, bool DROP>
__global__ void __launch_bounds__(320, 2) xattn_fwd_kernel(const __grid_constant__ XMaps maps, const XParams p) {
  using C = FwdCfg<DP>;
  constexpr int NKV = C::NKV, NSB = C::NSB;
  __shared__ uint64_t bar_q, bar_kfull[NKV], bar_kempty[NKV], bar_vfull[NKV], bar_vempty[NKV], bar_s[NSB], bar_p[NSB],
      bar_pv[2];
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
      mbar_init(&bar_p[i], C::EWT);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&bar_pv[i], 1);
    fence_barrier_init();
  }
  if (warp == C::MMA_WARP) {
    tmem_alloc(&tmem_sh, C::TM_COLS);
    tmem_relinquish();
  }
  if (BIAS)
    for (int x = threadIdx.x; x < (BIAS == 2 ? p.G : 1) * (kMaxBuckets + 1); x += C::THREADS)
      reinterpret_cast<float*>(xsmem + C::OFF_TAB)[x] =
          table_log2(p, BIAS == 2 ? kh * p.G + x / (kMaxBuckets + 1) : hx, x % (kMaxBuckets + 1));
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
        mma_scores<DP, 64>(tmem + C::TM_S + (c % NSB) * 64, sbase, sbase + C::OFF_K + st * C::KV_BYTES);
        mma_commit(&bar_s[c % NSB]);
        mma_commit(&bar_kempty[st]);
      };
      scores(0);
      for (int c = 0; c < nc && ok; ++c) {
        if (NSB == 2 && c + 1 < nc) scores(c + 1);
        const int st = c % NKV;
        if (!(ok = ok && mbar_wait(&bar_p[c % NSB], (c / NSB) & 1, ctx) && mbar_wait(&bar_vfull[st], (c / NKV) & 1, ctx)))
          break;
        tc_fence_after();
        mma_pieces<DP, 64, 32>(tmem + C::TM_O, tmem + C::TM_S + (c % NSB) * 64, sbase + C::OFF_V + st * C::KV_BYTES, c > 0);
        mma_commit(&bar_vempty[st]);
        mma_commit(&bar_pv[c & 1]);
        if (NSB == 1 && c + 1 < nc) scores(c + 1);
      }
    }
  } else {
    const int wg = warp / 4, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int i = pack ? r % p.Nq : qt * 128 + r;
    const int h = pack ? kh * p.G + r / p.Nq : hx;
    const bool row = pack ? r < p.G * p.Nq : i < p.Nq;
    const bool any_row = __any_sync(0xffffffffu, row);
    const int tab = C::OFF_TAB + (BIAS == 2 && row ? r / p.Nq * kTableBytes : 0);
    const int bh = b * p.H + h;
    const AttnDrop drop = attn_drop(p.rng, DROP ? p.drop_thr : 0, p.drop_scale);
    const uint32_t thr2 = drop.pair();
    // rows past nqp (in a last tile of 64) read the tile's other half
    const uint4* idrow = reinterpret_cast<const uint4*>(p.idsQ) +
                         ((long long)((i < p.nqp ? i : i - 64) / 64) * (p.nkp / 8) + c0 * 8 + wg * 4) * 64 + i % 64;
    float* xrow = reinterpret_cast<float*>(xsmem + C::OFF_ROW);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    // this thread's 32 ids and this lane's key of the next chunk, fetched a chunk ahead
    uint4 id[4];
    bool live_next = true;
    auto fetch = [&](int c) {
      if (p.kmask || (c0 + c + 1) * 64 > n) live_next = key_live(p, b, (c0 + c) * 64 + wg * 32 + lane, n);
      if (BIAS) {
#pragma unroll
        for (int x = 0; x < 4; ++x) id[x] = __ldg(idrow + c * 512 + x * 64);
      }
    };
    if (nc > 0) fetch(0);
    for (int c = 0; c < nc; ++c) {
      const int j0 = (c0 + c) * 64 + wg * 32;
      const uint32_t live = __ballot_sync(0xffffffffu, live_next);
      const uint32_t sbuf = lanes + C::TM_S + (c % NSB) * 64 + wg * 32;
      if (ok) ok = warp_wait(&bar_s[c % NSB], (c / NSB) & 1, ctx);
      tc_fence_after();
      float x[32];
      float mx = -INFINITY;
      if (ok && any_row) {
        tmem_ld32(sbuf, x);
        if (BIAS) {
          const uint32_t* w = reinterpret_cast<const uint32_t*>(id);
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const uint32_t o = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xFFFF;
            x[e] = fmaf(x[e], p.scale_log2, table_at(BIAS == 2 ? tab : C::OFF_TAB, o));
          }
        }
        if (live != ~0u) {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = (live >> e) & 1 ? x[e] : -INFINITY;
        }
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[e] = max3(x[e], x[e + 4], x[e + 8]);
          y[e] = max3(y[e], x[e + 12], x[e + 16]);
          y[e] = max3(y[e], x[e + 20], x[e + 24]);
          y[e] = fmaxf(y[e], x[e + 28]);
        }
        mx = fmaxf(max3(y[0], y[1], y[2]), y[3]);
        if (!BIAS) mx *= p.scale_log2;  // x is still the raw product (scale > 0: the order and -inf stay)
      }
      if (c + 1 < nc) fetch(c + 1);
      if (named_any(1 + (warp & 3), 64, row && (mx > m + kLazy || (m == -INFINITY && mx > m)))) {
        xrow[wg * 128 + r] = mx;
        named_sync(1 + (warp & 3), 64);
        const float top = fmaxf(mx, xrow[(wg ^ 1) * 128 + r]);
        const bool grow = top > m + kLazy || (m == -INFINITY && top > m);
        const float f = grow ? xex2(m - top) : 1.f;
        l *= f;
        m = grow ? top : m;
        if (c > 0) {
          if (ok) ok = warp_wait(&bar_pv[(c - 1) & 1], ((c - 1) >> 1) & 1, ctx);
          tc_fence_after();
          if (ok && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
            for (int d = wg * (DP / 2); d < (wg + 1) * (DP / 2); d += 16) {
              uint32_t o[16];
              tmem_ld16_issue(lanes + C::TM_O + d, o);
              tmem_wait16(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st16(lanes + C::TM_O + d, o);
            }
          }
        }
      }
      if (ok && any_row) {
        const float base = m == -INFINITY ? 0.f : m;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t w[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            float a = x[8 * g + e], d = x[8 * g + e + 1];
            a = xex2(BIAS ? a - base : fmaf(a, p.scale_log2, -base));
            d = xex2(BIAS ? d - base : fmaf(d, p.scale_log2, -base));
            sum[e & 2] += a, sum[(e & 2) + 1] += d;
            w[g * 4 + e / 2] = pack_bf16(a, d);
          }
          if (DROP) {
            const uint4 u = drop.words(i, (j0 >> 3) + g, bh);
            w[g * 4] &= spread_pair(keep_pair(u.x, thr2));
            w[g * 4 + 1] &= spread_pair(keep_pair(u.y, thr2));
            w[g * 4 + 2] &= spread_pair(keep_pair(u.z, thr2));
            w[g * 4 + 3] &= spread_pair(keep_pair(u.w, thr2));
          }
        }
        tmem_st16(sbuf, w);
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_wait_st();
      }
      if (live != ~0u) {  // what absent keys hold must not reach the product: 0 * NaN
        if (ok) ok = warp_wait(&bar_vfull[c % NKV], (c / NKV) & 1, ctx);
        if (ok && (warp & 3) == 0 && !((live >> lane) & 1)) {
          clear_row<DP>(xsmem + C::OFF_V + (c % NKV) * C::KV_BYTES, wg * 32 + lane);
          fence_proxy_async_smem();
        }
      }
      tc_fence_before();
      mbar_arrive(&bar_p[c % NSB]);
    }
    if (ok && nc > 0) ok = warp_wait(&bar_pv[(nc - 1) & 1], ((nc - 1) >> 1) & 1, ctx);
    tc_fence_after();
    named_sync(1 + (warp & 3), 64);  // the last exchange has been read
    xrow[wg * 128 + r] = l;
    named_sync(1 + (warp & 3), 64);
    l += xrow[(wg ^ 1) * 128 + r];
    const long long stat = (long long)bh * p.Nq + i;
    const long long part = (long long)split * p.B * p.H * p.Nq + stat;
    const float f = l == 0.f ? 0.f : (DROP ? p.drop_scale : 1.f) / l;
    const bool vec = vec_rows(p.o), tma = p.splits == 1 && p.out_tma;
    if (ok && any_row) {
#pragma unroll 1
      for (int d = wg * (DP / 2); d < (wg + 1) * (DP / 2); d += 32) {
        float o[32];
        if (nc > 0) tmem_ld32(lanes + C::TM_O + d, o);
        if (!tma && (!row || d >= p.D)) continue;
        if (l == 0.f) {  // a row with nothing left (or no chunk at all)
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
        }
        if (tma) {  // Q's tile is free: every product has completed
          stage_row32(xsmem, r, d, o, f);
        } else if (p.splits > 1) {
          float* dst = p.part_o + part * p.D + d;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (d + e < p.D) dst[e] = o[e];
        } else {
          __nv_bfloat16* dst =
              reinterpret_cast<__nv_bfloat16*>(p.o.p) + b * p.o.s[0] + h * p.o.s[1] + (long long)i * p.o.s[2] + d;
          store_row(dst, o, f, p.D - d, vec);
        }
      }
      if (row && wg == 0) {
        if (p.splits > 1) {
          p.part_ml[part * 2] = m;
          p.part_ml[part * 2 + 1] = l;
        } else if (p.stats) {
          p.stats[stat] = row_stats(m, l);
        }
      }
    }
    if (tma) {
      fence_proxy_async_smem();
      named_sync(5, C::EWT);
      if (threadIdx.x == 0 && ok) {
        if (pack) store_tile<DP>(&maps.o, xsmem, p.D, 0, kh * p.G, b);
        else store_tile<DP>(&maps.o, xsmem, p.D, qt * 128, hx, b);
        bulk_wait_read0();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::MMA_WARP) tmem_dealloc(tmem, C::TM_COLS);
}

// ---------------------------------------------------------------------------------------------------------------
// Backward, row records: chunks of 64 query rows, rec[b*h][chunk][3][64] floats:
//   without the bias  -(m + log2 l), unused, -delta       with it  -m, 1 / l, -delta (the bias may dwarf log2 l)
// so that P = 2^(t + rec0) or 2^(t + rec0) rec1; rows past Nq and rows with nothing left get P = 0. Bound by reading o
// and dO once: rows are taken in the order they lie in memory, with 8 loads of 16 bytes in flight per lane (256x16x512
// rows of 128: 197 us, 5.5 TB/s; 297 us with one or two loads in flight).
// ---------------------------------------------------------------------------------------------------------------
template <int LPR>  // lanes per row: 8 columns each
__global__ void __launch_bounds__(256) xattn_records_kernel(const XParams p, int heads_first) {
  constexpr int ROWS = 256 / LPR;  // rows of a step
  __shared__ float delta[256];
  if (threadIdx.x == 0 && blockIdx.x + blockIdx.y + blockIdx.z == 0) *p.status = kDevOk;
  // 256 rows: 16 rows of 16 heads, head by head in memory, or 256 rows of one head
  const int HB = heads_first ? 16 : 1, IB = 256 / HB;
  const int b = blockIdx.z, h0 = blockIdx.y * HB, i0 = blockIdx.x * IB;
  const int sub = threadIdx.x / LPR, c = threadIdx.x % LPR * 8;
  const bool vec = vec_rows(p.o) && vec_rows(p.dout);
  const __nv_bfloat16* O = reinterpret_cast<const __nv_bfloat16*>(p.o.p) + b * p.o.s[0] + c;
  const __nv_bfloat16* G = reinterpret_cast<const __nv_bfloat16*>(p.dout.p) + b * p.dout.s[0] + c;
#pragma unroll
  for (int s0 = 0; s0 < LPR; s0 += 4) {
    uint4 a[4], g[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int x = (s0 + u) * ROWS + sub, h = h0 + x % HB, i = i0 + x / HB;
      a[u] = g[u] = make_uint4(0, 0, 0, 0);
      if (h >= p.H || i >= p.Nq || c >= p.D) continue;
      const __nv_bfloat16 *o = O + h * p.o.s[1] + i * p.o.s[2], *d = G + h * p.dout.s[1] + i * p.dout.s[2];
      if (vec && c + 8 <= p.D) {
        a[u] = *reinterpret_cast<const uint4*>(o);
        g[u] = *reinterpret_cast<const uint4*>(d);
      } else {
        __nv_bfloat16 *av = reinterpret_cast<__nv_bfloat16*>(&a[u]), *gv = reinterpret_cast<__nv_bfloat16*>(&g[u]);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < p.D) av[e] = o[e], gv[e] = d[e];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const __nv_bfloat162 *av = reinterpret_cast<const __nv_bfloat162*>(&a[u]),
                           *gv = reinterpret_cast<const __nv_bfloat162*>(&g[u]);
      float d = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 s = __bfloat1622float2(av[e]), t = __bfloat1622float2(gv[e]);
        d = fmaf(s.x, t.x, fmaf(s.y, t.y, d));
      }
#pragma unroll
      for (int w = LPR / 2; w; w /= 2) d += __shfl_xor_sync(0xffffffffu, d, w);
      if (threadIdx.x % LPR == 0) delta[(s0 + u) * ROWS + sub] = d;
    }
  }
  __syncthreads();
  const int h = h0 + threadIdx.x / IB, i = i0 + threadIdx.x % IB;
  if (h >= p.H || i >= p.nqp) return;
  const long long bh = (long long)b * p.H + h;
  const float2 st = i < p.Nq ? p.stats[bh * p.Nq + i] : make_float2(0.f, 0.f);
  float* rec = p.rec + (bh * (p.nqp / 64) + i / 64) * 192 + i % 64;
  rec[0] = p.ids ? -st.x : st.y == 0.f ? -INFINITY : log2f(st.y) - st.x;
  rec[64] = st.y;
  rec[128] = -delta[threadIdx.x % IB * HB + threadIdx.x / IB];
}

// ---------------------------------------------------------------------------------------------------------------
// Backward, key pass. Tiles of (128 keys, key head, batch); loops over chunks of BQ queries of the heads that share the
// key head. Scores are formed transposed (keys in the lanes), so that P^T and dS^T are written over them in tensor
// memory as the A operands of
//   dV += P^T dO,  dK += dS^T Q
// and a thread owns one key's BQ / 4 queries; dS^T also goes to the scratch for dQ and the table's gradient.
//   MMA warp       dV(c), S^T(c + 1), dK(c), dP^T(c + 1), each as soon as what it reads is there and what it overwrites
//                  has been read by the product before it
//   4 warpgroups   P of chunk c while dK(c - 1) and dP^T(c) run, then dS of chunk c while dV(c) and S^T(c + 1) run
// Measured: 256x16x512x512x128 with the bias 1517 us (725 TFLOP/s), 1x8x4096x8192x128 with dropout 346 us (795),
// 32x16x512x512x192 with bias and dropout 328 us, 32x8x384x512x64 with dropout and lengths 73 us.
// Bound by the operand feed of the products (S and dP 64 clocks per 16 of the head dim and 128 queries, dV and dK as
// many per 16 queries at DP = 128): chunks of 128 queries, which halve K's and V's share of it, with one score buffer
// (S 128, dP 128, dK 128, dV 128 columns) beat chunks of 64 with two. DP = 192 has columns for 64 queries.
// One persistent CTA per SM (tensor memory is full): K and V of the next tile are loaded as soon as this one's last
// scores are formed, and the next tile's first scores run while dK and dV leave, from a stage of their own where shared
// memory has one, else from the slot of the tile's last chunk, which is refilled only then. (One CTA per tile spent 40 %
// of its time filling and draining at 512 queries.) Up to 64 queries per head run chunks of 64.
// Dropout: a Philox call covers one query and 8 keys. Each lane makes the calls of 2 or 4 queries for its octet of keys
// and the 8 x 8 bit blocks are transposed among 8 lanes (3 shuffles), so no call is made twice.
// ---------------------------------------------------------------------------------------------------------------
template <int DP, int BQ_>
struct KeysCfg {
  static constexpr int BQ = BQ_, QT = BQ / 4;  // queries per chunk and per thread
  static constexpr int NST = DP == 64 ? 4 : 2;  // chunks of Q, dO and records in flight
  static constexpr int K_BYTES = DP / 64 * 128 * 128, Q_BYTES = DP / 64 * BQ * 128, REC_BYTES = BQ * 12;
  static constexpr int STAGE = 2 * Q_BYTES;
  static constexpr bool OWN = DP == 64 || (DP == 128 && BQ == 64);  // dK and dV have a stage of their own
  static constexpr int OFF_V = K_BYTES, OFF_ST = 2 * K_BYTES, OFF_OUT = OFF_ST + NST * STAGE,
                       OFF_REC = OFF_OUT + (OWN ? 2 * K_BYTES : 0), OFF_TAB = OFF_REC + NST * REC_BYTES,
                       SMEM = OFF_TAB + 512;
  static constexpr int TM_DK = 0, TM_DV = DP, TM_S = 2 * DP, TM_DP = TM_S + BQ, TM_COLS = 512;
  static_assert(TM_DP + BQ <= 512 && SMEM + 1024 <= 227 * 1024, "");
  static constexpr int EWT = 512, THREADS = EWT + 64, TMA_WARP = 16, MMA_WARP = 17;
};

// Keep bits of 8 CALLS queries (i0 ..) for this lane's key j0 + lane: query 8 c + 2 i + e at bit 15 - (4 c + i) + 16 e. A
// lane makes the calls of queries 8 c + lane % 8 for keys 8 (lane / 8) ..; bit (c, i, e) there is key 2 i + e, and three
// exchanges transpose the 8 x 8 bits of each octet of lanes.
template <int CALLS>
__device__ __forceinline__ uint32_t keep_column(const AttnDrop& drop, uint32_t thr2, uint32_t i0, uint32_t j0,
                                                uint32_t bh) {
  const int lane = threadIdx.x & 31;
  uint32_t x = 0;
#pragma unroll
  for (int c = 0; c < CALLS; ++c) {
    const uint4 u = drop.words(i0 + 8 * c + (lane & 7), (j0 >> 3) + (lane >> 3), bh);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x |= (keep_pair(w[i], thr2) >> (4 * c + i)) & (0x80008000u >> (4 * c + i));
  }
  uint32_t y = __shfl_xor_sync(0xffffffffu, x, 1);
  x = lane & 1 ? (x & 0xFFFF0000u) | (y >> 16) : (x & 0x0000FFFFu) | (y << 16);
  y = __shfl_xor_sync(0xffffffffu, x, 2);
  x = lane & 2 ? (x & 0x55555555u) | ((y << 1) & 0xAAAAAAAAu) : (x & 0xAAAAAAAAu) | ((y >> 1) & 0x55555555u);
  y = __shfl_xor_sync(0xffffffffu, x, 4);
  return lane & 4 ? (x & 0x33333333u) | ((y << 2) & 0xCCCCCCCCu) : (x & 0xCCCCCCCCu) | ((y >> 2) & 0x33333333u);
}

template <int DP, int BQ_, bool BIAS, bool DROP>
__global__ void __launch_bounds__(KeysCfg<DP, BQ_>::THREADS, 1)
    xattn_bwd_keys_kernel(const __grid_constant__ XMaps maps, const XParams p) {
  using C = KeysCfg<DP, BQ_>;
  constexpr int NST = C::NST, BQ = C::BQ, QT = C::QT;
  __shared__ uint64_t bar_k, bar_kfree, bar_full[NST], bar_empty[NST], bar_s, bar_dp, bar_p, bar_ds, bar_done, bar_acc,
      bar_out;
  __shared__ uint32_t tmem_sh;
  __shared__ int abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int nkt = (p.Nk + 127) / 128;
  const int nqc = (p.nqp + BQ - 1) / BQ, nc = nqc * p.G;  // chunks per head and per tile
  WaitCtx ctx{&abort_flag, p.status};
  struct Tile {
    int j0, ul, b, kh, n;
  };
  auto tile_of = [&](int t) {
    Tile x;
    x.j0 = t % nkt * 128, x.ul = t / nkt;
    const int unit = p.u0 + x.ul;
    x.b = unit / p.Hkv, x.kh = unit % p.Hkv;
    x.n = key_count(p, x.b);
    return x;
  };

  if (threadIdx.x == 0) {
    abort_flag = 0;
    mbar_init(&bar_k, 1);
    for (int i = 0; i < NST; ++i) {
      mbar_init(&bar_full[i], 1);
      mbar_init(&bar_empty[i], 1);
    }
    mbar_init(&bar_s, 1);
    mbar_init(&bar_dp, 1);
    mbar_init(&bar_p, C::EWT);
    mbar_init(&bar_ds, C::EWT);
    mbar_init(&bar_kfree, 1);
    mbar_init(&bar_done, 1);
    mbar_init(&bar_acc, C::EWT);
    mbar_init(&bar_out, 1);
    fence_barrier_init();
  }
  if (warp == C::MMA_WARP) {
    tmem_alloc(&tmem_sh, C::TM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_sh, sbase = smem_u32(xsmem);

  if (warp == C::TMA_WARP) {
    if (lane == 0) {
      const int recs = p.nqp / 64;  // blocks of 64 records per head
      int t = 0, g = 0;             // tiles and chunks so far
      bool ok = true;
      for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x) {
        const Tile x = tile_of(tile);
        if (x.j0 >= x.n) continue;  // no key of this tile exists
        if (!(ok = mbar_wait(&bar_kfree, (t & 1) ^ 1, ctx))) break;
        mbar_arrive_expect_tx(&bar_k, 2 * C::K_BYTES);
        for (int y = 0; y < 128; y += 64) {  // the maps' boxes hold 64 rows
          load_rows<DP>(xsmem + y * 128, &maps.k, &bar_k, 128 * 128, x.j0 + y, x.kh, x.b);
          load_rows<DP>(xsmem + C::OFF_V + y * 128, &maps.v, &bar_k, 128 * 128, x.j0 + y, x.kh, x.b);
        }
        for (int c = 0; c < nc && ok; ++c, ++g) {
          const int st = g % NST, h = x.kh * p.G + c / nqc, q0 = c % nqc * BQ;
          // a last chunk of 128 queries may hold 64 padded rows only: no records for the others (`inside` below)
          const int rec = (p.nqp - q0 < BQ ? 64 : BQ) * 12;
          if (!(ok = mbar_wait(&bar_empty[st], ((g / NST) & 1) ^ 1, ctx))) break;
          // The last tile's dK and dV leave through its last chunk's slot, which chunk NST - 1 of this tile takes over.
          // Not later than this tile's last chunk, so that bar_out cannot run two phases ahead of the wait.
          if (!C::OWN && t > 0 && c == (NST < nc ? NST : nc) - 1 && !(ok = mbar_wait(&bar_out, (t - 1) & 1, ctx))) break;
          uint8_t* dst = xsmem + C::OFF_ST + st * C::STAGE;
          mbar_arrive_expect_tx(&bar_full[st], C::STAGE + rec);
          for (int y = 0; y < BQ; y += 64) {
            load_rows<DP>(dst + y * 128, &maps.q, &bar_full[st], BQ * 128, q0 + y, h, x.b);
            load_rows<DP>(dst + C::Q_BYTES + y * 128, &maps.dout, &bar_full[st], BQ * 128, q0 + y, h, x.b);
          }
          bulk_load(xsmem + C::OFF_REC + st * C::REC_BYTES, p.rec + ((long long)(x.b * p.H + h) * recs + q0 / 64) * 192,
                    rec, &bar_full[st]);
        }
        ++t;
      }
    }
  } else if (warp == C::MMA_WARP) {
    if (lane == 0) {
      int t = 0, g = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x) {
        const Tile x = tile_of(tile);
        if (x.j0 >= x.n) continue;
        const uint32_t slots = sbase + C::OFF_ST;
        if (!(ok = mbar_wait(&bar_k, t & 1, ctx) && mbar_wait(&bar_full[g % NST], (g / NST) & 1, ctx))) break;
        tc_fence_after();
        mma_scores<DP, BQ>(tmem + C::TM_S, sbase, slots + g % NST * C::STAGE);
        mma_commit(&bar_s);
        mma_scores<DP, BQ>(tmem + C::TM_DP, sbase + C::OFF_V, slots + g % NST * C::STAGE + C::Q_BYTES);
        mma_commit(&bar_dp);
        if (nc == 1) mma_commit(&bar_kfree);
        for (int c = 0; c < nc; ++c, ++g) {
          const int sn = (g + 1) % NST;
          const uint32_t q = slots + g % NST * C::STAGE, qn = slots + sn * C::STAGE;
          if (!(ok = mbar_wait(&bar_p, g & 1, ctx))) break;
          // the last tile's dK and dV have been read
          if (c == 0 && t > 0 && !(ok = mbar_wait(&bar_acc, (t - 1) & 1, ctx))) break;
          tc_fence_after();
          mma_pieces<DP, BQ, QT>(tmem + C::TM_DV, tmem + C::TM_S, q + C::Q_BYTES, c > 0);
          if (c + 1 < nc) {
            if (!(ok = mbar_wait(&bar_full[sn], ((g + 1) / NST) & 1, ctx))) break;
            tc_fence_after();
            mma_scores<DP, BQ>(tmem + C::TM_S, sbase, qn);
            mma_commit(&bar_s);
          }
          if (!(ok = mbar_wait(&bar_ds, g & 1, ctx))) break;
          tc_fence_after();
          mma_pieces<DP, BQ, QT>(tmem + C::TM_DK, tmem + C::TM_DP, q, c > 0);
          mma_commit(&bar_empty[g % NST]);
          if (c + 1 < nc) {
            mma_scores<DP, BQ>(tmem + C::TM_DP, sbase + C::OFF_V, qn + C::Q_BYTES);
            mma_commit(&bar_dp);
            if (c + 2 == nc) mma_commit(&bar_kfree);
          }
        }
        if (ok) mma_commit(&bar_done);
        ++t;
      }
    }
  } else {
    const int wg = warp / 4, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t sbuf = lanes + C::TM_S + wg * QT, dbuf = lanes + C::TM_DP + wg * QT;
    const AttnDrop drop = attn_drop(p.rng, DROP ? p.drop_thr : 0, p.drop_scale);
    const uint32_t thr2 = drop.pair();
    const uint64_t sc2 = f2(p.scale_log2, p.scale_log2), ds2 = f2(drop.scale, drop.scale);
    constexpr uint32_t no = kNoPairOffset * 0x10001u;
    const uint4 none = make_uint4(no, no, no, no);
    const uint32_t zeros[8] = {};
    const bool vk = vec_rows(p.dk), vv = vec_rows(p.dv), tk = p.out_tma & 2, tv = p.out_tma & 4;
    bool ok = true;
    int t = 0, gc = 0;  // tiles and chunks so far
    for (int tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
      const Tile x = tile_of(tile);
      const int b = x.b, kh = x.kh, j0 = x.j0, j = j0 + r;
      __nv_bfloat16* dK = reinterpret_cast<__nv_bfloat16*>(p.dk.p) + b * p.dk.s[0] + kh * p.dk.s[1];
      __nv_bfloat16* dV = reinterpret_cast<__nv_bfloat16*>(p.dv.p) + b * p.dv.s[0] + kh * p.dv.s[1];
      if (j0 >= x.n) {  // no key of this tile exists: zero gradients, and the scratch is not read here
        for (int y = threadIdx.x; y < 128 * p.D; y += C::EWT) {
          const int jj = j0 + y / p.D, d = y % p.D;
          if (jj < p.Nk) {
            dK[(long long)jj * p.dk.s[2] + d] = __float2bfloat16_rn(0.f);
            dV[(long long)jj * p.dv.s[2] + d] = __float2bfloat16_rn(0.f);
          }
        }
        continue;
      }
      const bool check_keys = p.kmask != nullptr || j0 + 128 > x.n, live = key_live(p, b, j, x.n);
      // ids and dS lie in granules of 8 queries: this key's first granule of a chunk, and 8 BQ granules per chunk
      const long long at = ((long long)(j / 64) * (p.nqp / 8) + wg * (QT / 8)) * 64 + j % 64;
      const uint4* idp = reinterpret_cast<const uint4*>(p.idsT) + at;
      uint4* const ds0 = reinterpret_cast<uint4*>(p.ds) + (long long)x.ul * p.G * (p.nkp / 8) * p.nqp + at;
      uint4 id[QT / 8];
      auto fetch = [&](int qc) {  // a chunk ahead
#pragma unroll
        for (int x = 0; x < QT / 8; ++x)
          id[x] = qc * BQ + wg * QT < p.Nq ? __ldg(idp + qc * (8 * BQ) + x * 64) : none;
      };
      if (BIAS) fetch(0);
      int qc = 0, g = 0;
      for (int c = 0; c < nc; ++c, ++gc) {
        const int st = gc % NST, i0 = qc * BQ + wg * QT, bh = b * p.H + kh * p.G + g;
        const bool inside = i0 < p.Nq;  // else padding: P = dS = 0
        uint4* ds = ds0 + (long long)g * (p.nkp / 8) * p.nqp + qc * (8 * BQ);
        if (BIAS && qc == 0) {  // the next head's bias
          named_sync(1, C::EWT);
          if (threadIdx.x <= kMaxBuckets)
            reinterpret_cast<float*>(xsmem + C::OFF_TAB)[threadIdx.x] = table_log2(p, kh * p.G + g, threadIdx.x);
          named_sync(1, C::EWT);
        }
        if (++qc == nqc) qc = 0, ++g;
        uint32_t keep = 0;
        if (DROP && inside) keep = keep_column<QT / 8>(drop, thr2, i0, j0 + (warp & 3) * 32, bh);
        const float* rec = reinterpret_cast<const float*>(xsmem + C::OFF_REC + st * C::REC_BYTES) + wg * QT / 64 * 192 +
                           wg * QT % 64;
        // bar_s follows bar_full, so the records are there too; the wait on bar_full makes their copy visible here
        if (ok) ok = warp_wait(&bar_full[st], (gc / NST) & 1, ctx) && warp_wait(&bar_s, gc & 1, ctx);
        if (!ok) continue;  // given up: only the barriers above are still met
        tc_fence_after();
        uint64_t pr[QT / 2];
#pragma unroll
        for (int k = 0; k < QT / 16; ++k) {
          if (!inside) {
            tmem_st8(sbuf + k * 8, zeros);
            continue;
          }
          uint32_t s[16], w[8];
          tmem_ld16_issue(sbuf + k * 16, s);
          tmem_wait16(s);
#pragma unroll
          for (int e = 0; e < 8; e += 2) {  // two pairs of queries
            const ulonglong2 r0 = *reinterpret_cast<const ulonglong2*>(rec + k * 16 + 2 * e);
            ulonglong2 r1 = make_ulonglong2(0, 0);
            if (BIAS) r1 = *reinterpret_cast<const ulonglong2*>(rec + 64 + k * 16 + 2 * e);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int q = e + u;
              uint64_t t = f2(__uint_as_float(s[2 * q]), __uint_as_float(s[2 * q + 1]));
              if (BIAS)
                t = add2(fma2(t, sc2, table_pair(C::OFF_TAB, reinterpret_cast<const uint32_t*>(id)[k * 8 + q])), u ? r0.y : r0.x);
              else
                t = fma2(t, sc2, u ? r0.y : r0.x);
              float x, y;
              unf2(t, x, y);
              t = f2(xex2(x), xex2(y));
              if (BIAS) t = mul2(t, u ? r1.y : r1.x);
              pr[k * 8 + q] = t;
              unf2(t, x, y);
              w[q] = pack_bf16(x, y);
              if (DROP) w[q] &= spread_pair(keep << (k * 8 + q));
            }
          }
          if (check_keys) {  // an absent key's row is 0 whatever K and V hold there
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = live ? w[e] : 0u;
          }
          tmem_st8(sbuf + k * 8, w);
        }
        if (BIAS && c + 1 < nc) fetch(qc);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&bar_p);
        if (!(ok = warp_wait(&bar_dp, gc & 1, ctx))) continue;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < QT / 16; ++k) {
          if (!inside) {
            tmem_st8(dbuf + k * 8, zeros);
            continue;
          }
          uint32_t dp[16], w[8];
          tmem_ld16_issue(dbuf + k * 16, dp);
          tmem_wait16(dp);
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const ulonglong2 r2 = *reinterpret_cast<const ulonglong2*>(rec + 128 + k * 16 + 2 * e);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int q = e + u;
              uint64_t da;
              if (DROP) {
                const uint32_t kb = keep << (k * 8 + q);
                da = f2(__uint_as_float(dp[2 * q] & spread_one<0>(kb)), __uint_as_float(dp[2 * q + 1] & spread_one<1>(kb)));
                da = fma2(da, ds2, u ? r2.y : r2.x);
              } else {
                da = add2(f2(__uint_as_float(dp[2 * q]), __uint_as_float(dp[2 * q + 1])), u ? r2.y : r2.x);
              }
              float x, y;
              unf2(mul2(pr[k * 8 + q], da), x, y);
              w[q] = pack_bf16(x, y);
            }
          }
          if (check_keys) {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = live ? w[e] : 0u;
          }
          tmem_st8(dbuf + k * 8, w);
          // granules without a query are neither written nor read
          if (i0 + k * 16 < p.Nq) ds[(2 * k) * 64] = make_uint4(w[0], w[1], w[2], w[3]);
          if (i0 + k * 16 + 8 < p.Nq) ds[(2 * k + 1) * 64] = make_uint4(w[4], w[5], w[6], w[7]);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&bar_ds);
      }
      if (ok) ok = warp_wait(&bar_done, t & 1, ctx);
      tc_fence_after();
      // dK and dV leave through a stage of their own (thread 0 saw it read before it went on to this tile) or the last
      // chunk's slot; DP = 192 has room for one of them at a time
      uint8_t* stage = xsmem + (C::OWN ? C::OFF_OUT : C::OFF_ST + (gc - 1) % NST * C::STAGE);
      constexpr bool BOTH = C::OWN || C::STAGE >= 2 * C::K_BYTES;
      const float fv = DROP ? p.drop_scale : 1.f;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const bool tma = which ? tv : tk;
        __nv_bfloat16* out = which ? dV + (long long)j * p.dv.s[2] : dK + (long long)j * p.dk.s[2];
        uint8_t* dst = stage + (BOTH ? which * C::K_BYTES : 0);
        if (ok) {
#pragma unroll 1
          for (int d = wg * 32; d < DP; d += 128) {
            float v[32];
            tmem_ld32(lanes + (which ? C::TM_DV : C::TM_DK) + d, v);
            if (tma) stage_row32(dst, r, d, v, which ? fv : p.scale);
            else if (j < p.Nk && d < p.D) store_row(out + d, v, which ? fv : p.scale, p.D - d, which ? vv : vk);
          }
        }
        if (which == 1) {
          tc_fence_before();
          mbar_arrive(&bar_acc);  // the accumulators may be overwritten
        }
        if (BOTH && which == 0) continue;
        fence_proxy_async_smem();
        named_sync(1, C::EWT);
        if (threadIdx.x == 0 && ok) {
          if (tk && (BOTH || which == 0)) store_tile<DP>(&maps.dk, stage, p.D, j0, kh, b);
          if (tv && which == 1) store_tile<DP>(&maps.dv, dst, p.D, j0, kh, b);
          bulk_wait_read0();
        }
        if (!BOTH && which == 0) named_sync(1, C::EWT);  // dK has left the stage
      }
      if (!C::OWN && threadIdx.x == 0) mbar_arrive(&bar_out);
      ++t;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::MMA_WARP) tmem_dealloc(tmem, C::TM_COLS);
}

// ---------------------------------------------------------------------------------------------------------------
// dQ = scale dS K from the dS scratch: one CTA per (128 queries, head of the launch's units), over 64-key chunks. The
// scratch's granules of 8 queries x 64 keys are the tensor core's unswizzled tiles with M contiguous (8 x 8 matrices of
// 128 bytes, 8 keys apart by 128 and 8 queries apart by 1024), so a chunk's A operand is one contiguous copy of 16 KB.
// Bound by reading the scratch (256x16x512x512x128: 548 us for 2.1 GB of dS, 0.5 of K and 0.5
// of dQ: 5.9 TB/s). Two of the epilogue's warps clear the rows of absent keys first (0 * NaN).
// ---------------------------------------------------------------------------------------------------------------
template <int DP>
struct DqCfg {
  static constexpr int NST = DP == 64 ? 4 : DP == 128 ? 3 : 2;
  static constexpr int A_BYTES = 16 * 1024, B_BYTES = DP / 64 * 64 * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int SMEM = NST * STAGE;
  static_assert(SMEM >= DP / 64 * 128 * 128, "the epilogue's tile");
  static constexpr int TM_COLS = DP == 64 ? 64 : DP == 128 ? 128 : 256;
  static constexpr int THREADS = 192, TMA_WARP = 4, MMA_WARP = 5;
};

template <int DP>
__global__ void __launch_bounds__(192, 2) xattn_bwd_dq_kernel(const __grid_constant__ XMaps maps, const XParams p) {
  using C = DqCfg<DP>;
  constexpr int NST = C::NST;
  __shared__ uint64_t bar_full[NST], bar_clean[NST], bar_empty[NST], bar_done;
  __shared__ uint32_t tmem_sh;
  __shared__ int abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int nqt = (p.Nq + 127) / 128, qt = blockIdx.x % nqt, ul = blockIdx.x / nqt;
  const int unit = p.u0 + ul / p.G, b = unit / p.Hkv, kh = unit % p.Hkv, h = kh * p.G + ul % p.G;
  const int n = key_count(p, b), nc = (n + 63) / 64;
  WaitCtx ctx{&abort_flag, p.status};
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < NST; ++i) {
      mbar_init(&bar_full[i], 1);
      mbar_init(&bar_clean[i], 64);
      mbar_init(&bar_empty[i], 1);
    }
    mbar_init(&bar_done, 1);
    fence_barrier_init();
  }
  if (warp == C::MMA_WARP) {
    tmem_alloc(&tmem_sh, C::TM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_sh, sbase = smem_u32(xsmem);

  if (warp == C::TMA_WARP) {
    if (lane == 0) {
      // the granules that hold queries (what the tile's other rows yield is not stored)
      const int rows = p.Nq - qt * 128, bytes = (rows < 128 ? (rows + 7) / 8 : 16) * 1024;
      const uint4* ds = reinterpret_cast<const uint4*>(p.ds) + (long long)ul * (p.nkp / 8) * p.nqp + (long long)qt * 16 * 64;
      for (int c = 0; c < nc; ++c) {
        const int st = c % NST;
        if (!mbar_wait(&bar_empty[st], ((c / NST) & 1) ^ 1, ctx)) break;
        uint8_t* dst = xsmem + st * C::STAGE;
        mbar_arrive_expect_tx(&bar_full[st], bytes + C::B_BYTES);
        bulk_load(dst, ds + (long long)c * (p.nqp / 8) * 64, bytes, &bar_full[st]);
        load_rows<DP>(dst + C::A_BYTES, &maps.k, &bar_full[st], 64 * 128, c * 64, kh, b);
      }
    }
  } else if (warp == C::MMA_WARP) {
    if (lane == 0) {
      constexpr uint32_t idesc = instr_desc(1, 1, 1, 128, DP);
      bool ok = true;
      for (int c = 0; c < nc; ++c) {
        const int st = c % NST;
        // every chunk is handed on by the clearing warps, whether it held an absent key or not
        if (!(ok = mbar_wait(&bar_clean[st], (c / NST) & 1, ctx))) break;
        tc_fence_after();
        const uint32_t a = sbase + st * C::STAGE, k = a + C::A_BYTES;
#pragma unroll
        for (int s = 0; s < 4; ++s)
          mma_ss<Kind::kF16>(tmem, smem_desc_plain(a + s * 2 * 128, 128, 1024),
                             smem_desc_sw128(k + s * 16 * 128, 64 * 128, 1024), idesc, c + s > 0);
        mma_commit(&bar_empty[st]);
      }
      if (ok) mma_commit(&bar_done);
    }
  } else {
    bool ok = true;
    if (warp < 2) {
      for (int c = 0; c < nc; ++c) {
        const int st = c % NST, j = c * 64 + threadIdx.x;
        const bool live = key_live(p, b, j, n);
        if (!(ok = warp_wait(&bar_full[st], (c / NST) & 1, ctx))) break;
        if (!live) {
          clear_row<DP>(xsmem + st * C::STAGE + C::A_BYTES, threadIdx.x);
          fence_proxy_async_smem();
        }
        mbar_arrive(&bar_clean[st]);
      }
    }
    if (ok) ok = warp_wait(&bar_done, 0, ctx);
    tc_fence_after();
    const int i = qt * 128 + warp * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    const bool vec = vec_rows(p.dq), tma = p.out_tma & 1;
    __nv_bfloat16* dQ = reinterpret_cast<__nv_bfloat16*>(p.dq.p) + b * p.dq.s[0] + h * p.dq.s[1];
    if (ok) {
#pragma unroll 1
      for (int d = 0; d < DP; d += 32) {
        float x[32];
        if (nc > 0) {
          tmem_ld32(lanes + d, x);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = 0.f;
        }
        if (tma) stage_row32(xsmem, warp * 32 + lane, d, x, p.scale);
        else if (i < p.Nq && d < p.D) store_row(dQ + (long long)i * p.dq.s[2] + d, x, p.scale, p.D - d, vec);
      }
    }
    if (tma) {
      fence_proxy_async_smem();
      named_sync(1, 128);
      if (threadIdx.x == 0 && ok) {
        store_tile<DP>(&maps.dq, xsmem, p.D, qt * 128, h, b);
        bulk_wait_read0();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::MMA_WARP) tmem_dealloc(tmem, C::TM_COLS);
}

}  // namespace xa
}  // namespace geoattn
