// Cross attention (queries and keys of different lengths), its bucketed bias and its dropout: what every kernel shares.
//
//   t_ij = log2(e) (scale q_i.k_j + table[h, ids[i, j]])      -inf where key j of batch b is absent (j >= lens[b] or
//                                                             key_mask[b, j] = 0) or the pair is excluded (ids >= T)
//   P_ij = 2^(t_ij - m_i) / l_i,  m_i = max_j t_ij,  l_i = sum_j 2^(t_ij - m_i)      0 for a row with nothing left
//   O_i  = sum_j A_ij v_j,  A_ij = keep_ij P_ij / (1 - p)
// and backward, with dA_ij = keep_ij (dO_i.v_j) / (1 - p) and delta_i = dO_i.O_i = sum_j P_ij dA_ij,
//   dS_ij = P_ij (dA_ij - delta_i);  dQ = scale dS K;  dK = scale dS^T Q;  dV = A^T dO;  dtable[h, t] = sum dS over
// the pairs of bucket t and the batch. Key head of query head h: h / G, G = H / Hkv; dK and dV sum over the G heads.
#pragma once
#include <cuda_bf16.h>

#include <cstdint>

#include "philox.cuh"

namespace geoattn {

constexpr int kMaxBuckets = 64;

struct XTensor {
  void* p;
  long long s[3];  // element strides of batch, head, row; the head dim is contiguous
};

struct XParams {
  int B, H, Hkv, G, Nq, Nk, D, T;
  XTensor q, k, v, o, dout, dq, dk, dv;
  const uint8_t* ids;       // [Nq][ids_ld] or null
  long long ids_ld;
  const uint16_t* idsQ;     // tiled offsets (ids_tile_kernel): rows = queries (nqp), columns = keys (nkp) (bf16 forward)
  const uint16_t* idsT;     // rows = keys (nkp), columns = queries (nqp) (backward)
  const void* table;        // [H][T], bf16 or fp32
  int table_bf16;
  const int* lens;          // [B] or null
  const uint8_t* kmask;     // [B][kmask_ld] or null
  long long kmask_ld;
  const long long* rng;     // (seed, offset) or null
  int drop_thr;             // 0: no dropout
  float drop_scale;
  float scale, scale_log2;  // scale, scale * log2(e)
  float2* stats;            // (m_i, 1 / l_i) [B*H][Nq]; (0, 0) for a row with nothing left. Kept apart: in m + log2(l)
                            // a bias near the type's lowest value would swallow log2(l)
  float* delta;             // [B*H][Nq] (fp32)
  float* rec;               // row records (bf16, xattn_records_kernel)
  void* ds;                 // dS of the launch's units, [unit * G + head][key / 64][query / 8][key % 64][8] (padded)
  int nqp, nkp;             // Nq, Nk rounded up to 64 and 128
  int u0;                   // first (batch, key head) unit of this launch
  int tiles;                // key tiles of the launch (key pass, tensor cores); query tiles (fp32 forward)
  int q0, rq;               // few-row kernels: first query and number of queries per head
  int out_tma;              // bit x: output x leaves through TMA stores (o; or dq, dk, dv)
  int pack;                 // forward, tensor cores: a tile holds the G * Nq rows of a key head's group
  int splits;               // > 1: key ranges per row, joined by xattn_combine_kernel
  float* part_o;            // [splits][B*H*Nq][D]
  float* part_ml;           // [splits][B*H*Nq][2]: running max (log2 units) and sum
  int* status;
};

constexpr int kNoPair = 255;
constexpr int kNoPairOffset = 4 * kMaxBuckets;  // byte offset behind the largest table: holds -inf

// Keys of batch b that exist: [0, n) before the key mask.
__device__ __forceinline__ int key_count(const XParams& p, int b) {
  if (!p.lens) return p.Nk;
  const int n = __ldg(p.lens + b);
  return n < 0 ? 0 : n > p.Nk ? p.Nk : n;
}
__device__ __forceinline__ bool key_live(const XParams& p, int b, int j, int n) {
  return j < n && (!p.kmask || __ldg(p.kmask + (long long)b * p.kmask_ld + j));
}
// table[h, t] in log2 units; -inf for ids that exclude their pair. A finite bias stays finite (a row whose pairs all
// have the type's lowest value is not an empty row).
__device__ __forceinline__ float table_log2(const XParams& p, int h, int t) {
  if (t >= p.T) return -INFINITY;
  const long long at = (long long)h * p.T + t;
  const float x = p.table_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.table)[at])
                               : reinterpret_cast<const float*>(p.table)[at];
  const float y = x * 1.4426950408889634f;
  return y == -INFINITY && x != -INFINITY ? -3.402823466e38f : y;
}

__device__ __forceinline__ float2 row_stats(float m, float l) {
  return l == 0.f ? make_float2(0.f, 0.f) : make_float2(m, 1.f / l);
}

__device__ __forceinline__ float xex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 values in one 64-bit register: one instruction works on both.
__device__ __forceinline__ uint64_t f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unf2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <class E>
__device__ __forceinline__ float to_f(E x) {
  return (float)x;
}
template <class E>
__device__ __forceinline__ E from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

}  // namespace geoattn
