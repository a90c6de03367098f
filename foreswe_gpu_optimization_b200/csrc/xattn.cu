// Host launchers of the cross attention, its bucketed bias and dropout, behind the C ABI in include/geoattn.h.
#include <cmath>
#include <cstdint>
#include <cstring>
#include <type_traits>

#include "../../include/geoattn.h"
#include "host_util.h"
#include "tma_host.h"
#include "xattn_aux.cuh"
#include "xattn_rows.cuh"
#include "xattn_simt.cuh"
#include "xattn_tc.cuh"

namespace geoattn {
namespace {

constexpr int kSMs = 148;  // B200

// Most dS^T scratch of one backward launch. Larger problems run in several launches over (batch, key head) units, so
// that the scratch stays bounded; below this size a launch already fills the GPU.
constexpr size_t kDsCap = (size_t)4 << 30;

struct XDims {
  int B, H, Hkv, G, Nq, Nk, D, DP, T, nqp, nkp;
  bool bf16;
  int fwd_rows, bwd_rows;  // few query rows: the kernels' rows (1, 2, 4 or 8), or 0
  int splits;           // forward key splits
  int bwd_splits;       // backward key splits (few query rows)
  int tail;             // fp32 forward: queries behind the last whole tile that the few-row kernel takes, or 0
  long long row_ctas;   // forward CTAs per key split (few query rows)
  int nqb;              // query padding of the dS^T scratch
  int units_per_launch; // backward
  int launches, chunks;
  size_t ds_unit;       // dS^T bytes of one (batch, key head) unit
};

// The few rows of heads that share a key head in one tile: K and V are read once per key head (128 x 64 / 8 heads, 1 query,
// 4096 keys of 128 with the bias: 380 against 2114 us).
bool packs_rows(const XDims& d) {
  return d.bf16 && d.G > 1 && (long long)d.G * d.Nq <= 128 && (d.T == 0 || d.G <= xa::kPackTables);
}

int forward_splits(const XDims& d) {
  // Enough key ranges to give every SM a tile when the rows alone do not.
  const long long tiles = packs_rows(d) ? (long long)d.B * d.Hkv : (long long)((d.Nq - d.tail + 127) / 128) * d.B * d.H;
  const int ktiles = (d.Nk + 63) / 64;
  if (tiles >= kSMs) return 1;
  long long want, most;
  if (d.bf16) {
    // Joining the ranges costs a launch of about 4 us, as much as 4 chunks of 64 keys: below 12 chunks one range is
    // faster (1 x 16 heads, 1 query, 512 keys: 13 against 17 us), and a range keeps at least 4. Lengths may differ, so
    // twice as many ranges as the GPU holds at once.
    want = (4 * kSMs + tiles - 1) / tiles;
    most = ktiles < 12 ? 1 : ktiles / 4;
  } else {
    // A chunk takes about 12 us on the FMA pipe: one wave of two CTAs per SM, at least two chunks each (8 x 8 heads,
    // 130 queries, 517 keys: 106 against 129 us).
    want = 2 * kSMs / tiles;
    most = ktiles / 2;
  }
  const long long n = want < most ? want : most;
  return n < 1 ? 1 : (int)n;
}

// Where the kernels for few query rows (xattn_rows.cuh) take a call: how many rows a CTA holds, or 0. Their time grows
// with the rows of a key head's group, that of the tiled kernels with its heads. Both sides measured:
//   fp32 forward, up to 32 queries per head (a tile holds 128): 64 x 16 heads, 4096 keys of 64, 8 queries: 702 against
//     3850 us; the queries behind the last whole tile where they are no more (8 x 8 heads, 130 queries, 517 keys of
//     48: 106 -> 78 us); backward, a group of up to 8 rows: 64 x 15 / 5 heads, 2 queries, 11785 keys of 64: 2.2 against
//     27.6 ms.
//   bf16 forward, one row and K and V of at most 32 MB: 1 x 16 heads, 512 keys of 192: 14.1 against 16.6 us; but 32 x
//     16, 4096 of 128: 234 against 166 us, and rows of heads that share a key head go into one tile: 128 x 16 / 8 heads,
//     512 keys of 128: 79 against 62 us.
//   bf16 backward, one query per head: a head dim of at most 64 (32 x 16 heads of one key head each, 2048 keys: 236
//     against 279 us; groups of 8: 507 against 852), a bias and shared key heads (groups of 4, 2048 keys of 128: 799
//     against 969 us), or fewer heads than SMs, which dQ's tiles cannot fill (1 x 16 heads, 16384 keys of 128: 157
//     against 232 us). Otherwise the tiles: 32 x 16 heads, 2048 keys of 128: 362 against 425 us.
int rows_of(long long rows) { return rows > 4 ? kRowMax : rows > 2 ? 4 : (int)rows; }
int forward_rows_of(const XDims& d) {
  const long long rows = (long long)d.G * (d.tail ? d.tail : d.Nq);
  if (d.tail) return rows_of(rows);
  if (d.bf16) return rows == 1 && (long long)d.B * d.Hkv * d.Nk * d.D <= 8 << 20 ? 1 : 0;
  return d.Nq <= 32 || rows <= kRowMax ? rows_of(rows) : 0;
}
int backward_rows_of(const XDims& d) {
  const long long rows = (long long)d.G * d.Nq;
  if (rows > kRowMax) return 0;
  if (d.bf16 && !(d.Nq == 1 && (d.DP == 64 || (d.T && d.G > 1) || (long long)d.B * d.H < kSMs))) return 0;
  return rows_of(rows);
}
// Key ranges of at least 512 keys, enough for four CTAs per SM.
int row_splits(const XDims& d, long long ctas) {
  const long long want = (4 * kSMs + ctas - 1) / ctas, most = d.Nk / 512;
  const long long n = want < most ? want : most;
  return n < 1 ? 1 : (int)n;
}

int check_xshape(const GeoXattnShape* s, XDims& d) {
  if (!s || s->batch <= 0 || s->heads <= 0 || s->kv_heads <= 0 || s->nq <= 0 || s->nk <= 0 || s->head_dim <= 0 ||
      s->heads % s->kv_heads || s->buckets < 0)
    return GEOATTN_ERR_INVALID;
  if (s->dtype != GEOATTN_DTYPE_BF16 && s->dtype != GEOATTN_DTYPE_FP32) return GEOATTN_ERR_INVALID;
  if (s->table_dtype != GEOATTN_DTYPE_BF16 && s->table_dtype != GEOATTN_DTYPE_FP32) return GEOATTN_ERR_INVALID;
  if (s->head_dim > 192 || s->buckets > kMaxBuckets) return GEOATTN_ERR_UNSUPPORTED;
  d.B = s->batch, d.H = s->heads, d.Hkv = s->kv_heads, d.G = d.H / d.Hkv;
  d.Nq = s->nq, d.Nk = s->nk, d.D = s->head_dim, d.T = s->buckets;
  d.DP = d.D <= 64 ? 64 : d.D <= 128 ? 128 : 192;
  d.bf16 = s->dtype == GEOATTN_DTYPE_BF16;
  // rows and keys fit an int after padding, and so do a launch's CTAs
  if (d.Nq > (1 << 30) || d.Nk > (1 << 30) || (long long)d.B * d.H > (1 << 30)) return GEOATTN_ERR_UNSUPPORTED;
  d.nqp = (d.Nq + 63) / 64 * 64;
  d.nkp = (d.Nk + 127) / 128 * 128;
  if (d.B > 65535 || d.H > 65535) return GEOATTN_ERR_UNSUPPORTED;  // grid of the row records
  if (d.T && (d.nqp / 64 > 65535 || d.nkp / 64 > 65535)) return GEOATTN_ERR_UNSUPPORTED;  // grid of the ids' tiles
  d.tail = !d.bf16 && d.Nq > 128 && d.Nq % 128 <= 32 ? d.Nq % 128 : 0;
  d.fwd_rows = forward_rows_of(d);
  d.bwd_rows = backward_rows_of(d);
  d.nqb = d.bwd_rows ? 8 : d.nqp;
  const long long row_units = (long long)d.B * d.Hkv;
  d.row_ctas = d.fwd_rows ? ((long long)d.G * (d.tail ? d.tail : d.Nq) + d.fwd_rows - 1) / d.fwd_rows * row_units : 0;
  d.splits = d.fwd_rows && !d.tail ? row_splits(d, d.row_ctas) : forward_splits(d);
  d.bwd_splits = d.bwd_rows ? row_splits(d, row_units) : 1;
  if (d.row_ctas * d.splits > (1ll << 30)) return GEOATTN_ERR_UNSUPPORTED;
  const long long qt = (d.Nq + 63) / 64, kt = (d.Nk + 31) / 32;
  if (qt * d.B * d.H * d.splits > (1ll << 30) || kt * d.B * d.Hkv > (1ll << 30)) return GEOATTN_ERR_UNSUPPORTED;
  d.ds_unit = d.bwd_rows && !d.T ? 0 : (size_t)d.G * d.nkp * d.nqb * (d.bf16 ? 2 : 4);
  const long long units = (long long)d.B * d.Hkv;
  long long per = d.ds_unit ? (long long)(kDsCap / d.ds_unit) : units;
  per = per < 1 ? 1 : per > units ? units : per;
  d.units_per_launch = (int)per;
  d.launches = (int)((units + per - 1) / per);
  const long long want = (16ll * kSMs + d.H - 1) / d.H, most = (long long)d.nkp * d.nqb / (d.bf16 ? 8 : 4) / 256;
  
  d.chunks = (int)(want < most ? want : most < 1 ? 1 : most);
  return GEOATTN_OK;
}

struct XFwdWs {
  int* status;
  float *part_o, *part_ml;
  uint16_t* ids;
};
size_t xfwd_ws(const XDims& d, uint8_t* base, XFwdWs* w) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    uint8_t* p = base ? base + off : nullptr;
    off += align_up(bytes);
    return p;
  };
  XFwdWs t{};
  t.status = reinterpret_cast<int*>(take(sizeof(int)));
  if (d.splits > 1) {
    const size_t rows = (size_t)d.splits * d.B * d.H * d.Nq;
    t.part_o = reinterpret_cast<float*>(take(rows * d.D * 4));
    t.part_ml = reinterpret_cast<float*>(take(rows * 2 * 4));
  }
  if (d.T && d.bf16 && !d.fwd_rows) t.ids = reinterpret_cast<uint16_t*>(take((size_t)d.nqp * d.nkp * 2));
  if (w) *w = t;
  return off;
}

struct XBwdWs {
  int* status;
  float *delta, *rec;
  void* ds;
  uint16_t* idsT;
  float* part;
  float* part_dq;
};
size_t xbwd_ws(const XDims& d, uint8_t* base, XBwdWs* w) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    uint8_t* p = base ? base + off : nullptr;
    off += align_up(bytes);
    return p;
  };
  XBwdWs t{};
  t.status = reinterpret_cast<int*>(take(sizeof(int)));
  if (d.bwd_splits > 1) t.part_dq = reinterpret_cast<float*>(take((size_t)d.bwd_splits * d.B * d.H * d.Nq * d.D * 4));
  if (!d.bwd_rows) {
    if (d.bf16) t.rec = reinterpret_cast<float*>(take((size_t)d.B * d.H * d.nqp * 3 * 4));
    else t.delta = reinterpret_cast<float*>(take((size_t)d.B * d.H * d.Nq * 4));
  }
  t.ds = take(d.ds_unit * d.units_per_launch);
  if (d.T) {
    t.idsT = reinterpret_cast<uint16_t*>(take((size_t)d.nkp * d.nqb * 2));
    t.part = reinterpret_cast<float*>(take((size_t)d.launches * d.H * d.chunks * d.T * 4));
  }
  if (w) *w = t;
  return off;
}

// Makes the current device's context current in this thread: the driver's tensor-map encoder wants one, and a thread
// whose first CUDA call this is (autograd's, a user's worker) may have none yet.
bool bind_context() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}

int status_of(cudaError_t e) { return e == cudaSuccess ? GEOATTN_OK : GEOATTN_ERR_LAUNCH; }

XTensor xt(const void* p, const long long* s) {
  XTensor t;
  t.p = const_cast<void*>(p);
  for (int i = 0; i < 3; ++i) t.s[i] = s[i];
  return t;
}

int check_inputs(const GeoXattnInputs& a, const XDims& d) {
  if (!dev_ptr(a.q.data) || !dev_ptr(a.k.data) || !dev_ptr(a.v.data)) return GEOATTN_ERR_INVALID;
  if (d.T && (!dev_ptr(a.ids) || !dev_ptr(a.table) || a.ids_ld < d.Nk)) return GEOATTN_ERR_INVALID;
  if (a.kv_lens && !dev_ptr(a.kv_lens)) return GEOATTN_ERR_INVALID;
  if (a.key_mask && (!dev_ptr(a.key_mask) || a.key_mask_ld < d.Nk)) return GEOATTN_ERR_INVALID;
  if (!(a.scale > 0.f) || std::isinf(a.scale)) return GEOATTN_ERR_INVALID;
  if (a.drop_threshold < 0 || a.drop_threshold > 65535 || (a.drop_threshold > 0 && !dev_ptr(a.rng)))
    return GEOATTN_ERR_INVALID;
  for (const GeoAttnTensor* t : {&a.q, &a.k, &a.v})
    if (t->stride[3] != 1) return GEOATTN_ERR_ALIGNMENT;
  return GEOATTN_OK;
}

XParams xparams(const GeoXattnInputs& a, const XDims& d) {
  XParams p;
  std::memset(&p, 0, sizeof(p));
  p.B = d.B, p.H = d.H, p.Hkv = d.Hkv, p.G = d.G, p.Nq = d.Nq, p.Nk = d.Nk, p.D = d.D, p.T = d.T;
  p.q = xt(a.q.data, a.q.stride), p.k = xt(a.k.data, a.k.stride), p.v = xt(a.v.data, a.v.stride);
  if (d.T) {
    p.ids = a.ids, p.ids_ld = a.ids_ld, p.table = a.table;
    p.table_bf16 = a.shape.table_dtype == GEOATTN_DTYPE_BF16;
  }
  p.lens = a.kv_lens, p.kmask = a.key_mask, p.kmask_ld = a.key_mask_ld;
  p.rng = a.rng, p.drop_thr = a.drop_threshold;
  p.drop_scale = (float)(65536.0 / (65536 - a.drop_threshold));
  p.scale = a.scale, p.scale_log2 = (float)((double)a.scale * 1.4426950408889634);
  p.nqp = d.nqp, p.nkp = d.nkp, p.splits = 1;
  p.q0 = 0, p.rq = d.Nq;
  return p;
}

template <class K>
int xlaunch(K kernel, long long grid, int threads, int smem, cudaStream_t st, const XParams& p) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return GEOATTN_ERR_LAUNCH;
  kernel<<<(unsigned)grid, threads, smem, st>>>(p);
  return status_of(cudaGetLastError());
}

template <int DP>
int simt_fwd(const XParams& p, cudaStream_t st) {
  return xlaunch(xattn_simt_fwd_kernel<DP>, (long long)p.tiles * p.B * p.H * p.splits,
                 SimtFwd<DP>::NT, SimtFwd<DP>::SMEM, st, p);
}
int forward_simt(XParams& p, const XDims& d, cudaStream_t st) {
  p.tiles = (d.Nq - d.tail + 127) / 128;
  return d.DP == 64 ? simt_fwd<64>(p, st) : d.DP == 128 ? simt_fwd<128>(p, st) : simt_fwd<192>(p, st);
}
template <int DP>
int simt_bwd(const XParams& p, int units, cudaStream_t st) {
  using C = SimtBwd<DP>;
  int rc = xlaunch(xattn_simt_bwd_keys_kernel<DP>, (long long)((p.Nk + C::TK - 1) / C::TK) * units, kSimtThreads,
                   C::SMEM, st, p);
  if (rc) return rc;
  return xlaunch(xattn_simt_bwd_dq_kernel<DP>, (long long)((p.Nq + 63) / 64) * units * p.G, kSimtThreads,
                 SimtDq<DP>::SMEM, st, p);
}
int backward_simt(const XParams& p, const XDims& d, int units, cudaStream_t st) {
  return d.DP == 64 ? simt_bwd<64>(p, units, st) : d.DP == 128 ? simt_bwd<128>(p, units, st) : simt_bwd<192>(p, units, st);
}

template <class F>
int with_rows(int dp, int rows, F f) {
  const auto nv = [&](auto v) {
    return rows == 1   ? f(v, std::integral_constant<int, 1>())
           : rows == 2 ? f(v, std::integral_constant<int, 2>())
           : rows == 4 ? f(v, std::integral_constant<int, 4>())
                       : f(v, std::integral_constant<int, 8>());
  };
  return dp == 64    ? nv(std::integral_constant<int, 1>())
         : dp == 128 ? nv(std::integral_constant<int, 2>())
                     : nv(std::integral_constant<int, 3>());
}
int forward_rows(const XParams& p, const XDims& d, cudaStream_t st) {
  return with_rows(d.DP, d.fwd_rows, [&](auto nv, auto r) {
    constexpr int NV = decltype(nv)::value, R = decltype(r)::value;
    const long long grid = d.row_ctas * d.splits;
    if (!d.bf16) return xlaunch(xattn_rows_fwd_kernel<float, NV, R>, grid, kRowThreads, 0, st, p);
    if constexpr (R == 1) return xlaunch(xattn_rows_fwd_kernel<__nv_bfloat16, NV, R>, grid, kRowThreads, 0, st, p);
    return (int)GEOATTN_ERR_UNSUPPORTED;  // forward_rows_of gives bf16 no other R
  });
}
template <class E>
int backward_rows(const XParams& p, const XDims& d, int units, cudaStream_t st) {
  return with_rows(d.DP, d.bwd_rows, [&](auto nv, auto r) {
    xattn_rows_bwd_kernel<E, decltype(nv)::value, decltype(r)::value>
        <<<(unsigned)((long long)units * d.bwd_splits), kRowThreads, 0, st>>>(p, units);
    return status_of(cudaGetLastError());
  });
}
// What the tensor-core kernels ask of their operands, asked of every bf16 call: which kernel runs is not the caller's
// concern.
bool tma_ok(const XTensor& t) {
  if (reinterpret_cast<uintptr_t>(t.p) & 15) return false;
  for (int i = 0; i < 3; ++i)
    if (t.s[i] <= 0 || ((t.s[i] * 2) & 15)) return false;
  return true;
}

// TMA map over a bf16 tensor [batch, heads, rows, D] (box: 64 columns x `rows` rows x `heads` heads).
int xmap(CUtensorMap* m, const XTensor& t, int D, int n, int heads, int batch, int box_rows, int box_heads) {
  if (!tma_ok(t)) return GEOATTN_ERR_ALIGNMENT;
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)n, (uint64_t)heads, (uint64_t)batch};
  const uint64_t str[3] = {(uint64_t)t.s[2] * 2, (uint64_t)t.s[1] * 2, (uint64_t)t.s[0] * 2};
  const uint32_t box[4] = {64, (uint32_t)box_rows, (uint32_t)box_heads, 1};
  return make_tmap(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, t.p, dims, str, box) ? GEOATTN_OK : GEOATTN_ERR_TMA;
}

template <class K>
int tc_launch(K kernel, long long grid, int threads, int smem, cudaStream_t st, const xa::XMaps& maps,
              const XParams& p) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return GEOATTN_ERR_LAUNCH;
  kernel<<<(unsigned)grid, threads, smem, st>>>(maps, p);
  return status_of(cudaGetLastError());
}

template <int DP>
int tc_fwd(const xa::XMaps& maps, const XParams& p, long long grid, cudaStream_t st) {
  using C = xa::FwdCfg<DP>;
  auto fwd = !p.ids ? (p.drop_thr ? xa::xattn_fwd_kernel<DP, 0, true> : xa::xattn_fwd_kernel<DP, 0, false>)
             : p.pack ? (p.drop_thr ? xa::xattn_fwd_kernel<DP, 2, true> : xa::xattn_fwd_kernel<DP, 2, false>)
                      : (p.drop_thr ? xa::xattn_fwd_kernel<DP, 1, true> : xa::xattn_fwd_kernel<DP, 1, false>);
  return tc_launch(fwd, grid, C::THREADS, C::SMEM, st, maps, p);
}

// Store maps of the outputs that TMA can write (box: 64 columns x 128 rows, or a packed tile's rows); the others leave
// by plain stores.
void out_map(CUtensorMap* m, int* flags, int bit, const XTensor& t, int D, int n, int heads, int batch, int rows = 128,
             int box_heads = 1) {
  if (xmap(m, t, D, n, heads, batch, rows, box_heads) == GEOATTN_OK) *flags |= bit;
}

int forward_tc(XParams& p, const XDims& d, uint16_t* ids, cudaStream_t st) {
  xa::XMaps maps;
  std::memset(&maps, 0, sizeof(maps));
  p.pack = packs_rows(d);
  int rc;
  if ((rc = p.pack ? xmap(&maps.q, p.q, d.D, d.Nq, d.H, d.B, d.Nq, d.G) : xmap(&maps.q, p.q, d.D, d.Nq, d.H, d.B, 128, 1)) ||
      (rc = xmap(&maps.k, p.k, d.D, d.Nk, d.Hkv, d.B, 64, 1)) || (rc = xmap(&maps.v, p.v, d.D, d.Nk, d.Hkv, d.B, 64, 1)))
    return rc;
  if (p.pack) out_map(&maps.o, &p.out_tma, 1, p.o, d.D, d.Nq, d.H, d.B, d.Nq, d.G);
  else out_map(&maps.o, &p.out_tma, 1, p.o, d.D, d.Nq, d.H, d.B);
  if (d.T) {
    ids_tile_kernel<false><<<dim3(d.nkp / 64, d.nqp / 64), 256, 0, st>>>(p.ids, p.ids_ld, d.Nq, d.Nk, d.nkp, d.T, ids);
    p.idsQ = ids;
    if ((rc = status_of(cudaGetLastError()))) return rc;
  }
  const long long grid = (long long)d.splits * d.B * (p.pack ? d.Hkv : (long long)((d.Nq + 127) / 128) * d.H);
  return d.DP == 64 ? tc_fwd<64>(maps, p, grid, st)
                    : d.DP == 128 ? tc_fwd<128>(maps, p, grid, st) : tc_fwd<192>(maps, p, grid, st);
}

int backward_maps(xa::XMaps& maps, XParams& p, const XDims& d) {
  int rc;
  if ((rc = xmap(&maps.q, p.q, d.D, d.Nq, d.H, d.B, 64, 1)) || (rc = xmap(&maps.dout, p.dout, d.D, d.Nq, d.H, d.B, 64, 1)) ||
      (rc = xmap(&maps.k, p.k, d.D, d.Nk, d.Hkv, d.B, 64, 1)) || (rc = xmap(&maps.v, p.v, d.D, d.Nk, d.Hkv, d.B, 64, 1)))
    return rc;
  out_map(&maps.dq, &p.out_tma, 1, p.dq, d.D, d.Nq, d.H, d.B);
  out_map(&maps.dk, &p.out_tma, 2, p.dk, d.D, d.Nk, d.Hkv, d.B);
  out_map(&maps.dv, &p.out_tma, 4, p.dv, d.D, d.Nk, d.Hkv, d.B);
  return GEOATTN_OK;
}

int records(const XParams& p, const XDims& d, cudaStream_t st) {
  const int heads_first = p.o.s[1] < p.o.s[2], hb = heads_first ? 16 : 1, ib = 256 / hb;
  const dim3 grid((d.nqp + ib - 1) / ib, (d.H + hb - 1) / hb, d.B);
  if (d.DP == 64) xa::xattn_records_kernel<8><<<grid, 256, 0, st>>>(p, heads_first);
  else if (d.DP == 128) xa::xattn_records_kernel<16><<<grid, 256, 0, st>>>(p, heads_first);
  else xa::xattn_records_kernel<32><<<grid, 256, 0, st>>>(p, heads_first);
  return status_of(cudaGetLastError());
}

template <int DP, int BQ>
int tc_bwd_keys(const xa::XMaps& maps, const XParams& p, int units, cudaStream_t st) {
  using C = xa::KeysCfg<DP, BQ>;
  const long long tiles = (long long)((p.Nk + 127) / 128) * units, grid = tiles < kSMs ? tiles : kSMs;
  XParams pk = p;
  pk.tiles = (int)tiles;
  auto keys = p.ids ? (p.drop_thr ? xa::xattn_bwd_keys_kernel<DP, BQ, true, true> : xa::xattn_bwd_keys_kernel<DP, BQ, true, false>)
                    : (p.drop_thr ? xa::xattn_bwd_keys_kernel<DP, BQ, false, true> : xa::xattn_bwd_keys_kernel<DP, BQ, false, false>);
  return tc_launch(keys, grid, C::THREADS, C::SMEM, st, maps, pk);
}

template <int DP>
int tc_bwd_dq(const xa::XMaps& maps, const XParams& p, int units, cudaStream_t st) {
  return tc_launch(xa::xattn_bwd_dq_kernel<DP>, (long long)((p.Nq + 127) / 128) * units * p.G, xa::DqCfg<DP>::THREADS,
                   xa::DqCfg<DP>::SMEM, st, maps, p);
}

int backward_tc(const xa::XMaps& maps, const XParams& p, const XDims& d, int units, cudaStream_t st) {
  const bool few = d.nqp <= 64;  // half of a chunk of 128 queries would be padding
  int rc = d.DP == 64    ? few ? tc_bwd_keys<64, 64>(maps, p, units, st) : tc_bwd_keys<64, 128>(maps, p, units, st)
           : d.DP == 128 ? few ? tc_bwd_keys<128, 64>(maps, p, units, st) : tc_bwd_keys<128, 128>(maps, p, units, st)
                         : tc_bwd_keys<192, 64>(maps, p, units, st);
  if (rc) return rc;
  return d.DP == 64 ? tc_bwd_dq<64>(maps, p, units, st)
                    : d.DP == 128 ? tc_bwd_dq<128>(maps, p, units, st) : tc_bwd_dq<192>(maps, p, units, st);
}

template <class S>
int table_grad(const XParams& p, const XDims& d, int units, float* part, cudaStream_t st) {
  if (cudaFuncSetAttribute(table_grad_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxBuckets * 1024) !=
      cudaSuccess)
    return GEOATTN_ERR_LAUNCH;
  table_grad_kernel<S><<<dim3(d.chunks, d.H), 256, d.T * 1024, st>>>(p, units, part);
  return status_of(cudaGetLastError());
}

}  // namespace
}  // namespace geoattn

using namespace geoattn;

extern "C" {

size_t geoattn_xattn_fwd_workspace_bytes(const GeoXattnShape* shape) {
  XDims d;
  return check_xshape(shape, d) ? 0 : xfwd_ws(d, nullptr, nullptr);
}

size_t geoattn_xattn_bwd_workspace_bytes(const GeoXattnShape* shape) {
  XDims d;
  return check_xshape(shape, d) ? 0 : xbwd_ws(d, nullptr, nullptr);
}

int geoattn_xattn_fwd(const GeoXattnFwdArgs* a, void* stream) {
  if (!a) return GEOATTN_ERR_INVALID;
  XDims d;
  if (int rc = check_xshape(&a->in.shape, d)) return rc;
  if (int rc = check_inputs(a->in, d)) return rc;
  if (!dev_ptr(a->o) || (a->stats && !dev_ptr(a->stats)) || !dev_ptr(a->workspace)) return GEOATTN_ERR_INVALID;
  if (a->o_stride[3] != 1 || (reinterpret_cast<uintptr_t>(a->workspace) & (kAlign - 1))) return GEOATTN_ERR_ALIGNMENT;
  if (!bind_context()) return GEOATTN_ERR_LAUNCH;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  XFwdWs ws;
  xfwd_ws(d, reinterpret_cast<uint8_t*>(a->workspace), &ws);
  XParams p = xparams(a->in, d);
  p.o = xt(a->o, a->o_stride), p.stats = reinterpret_cast<float2*>(a->stats);
  p.splits = d.splits, p.part_o = ws.part_o, p.part_ml = ws.part_ml, p.status = ws.status;
  if (d.bf16 && !(tma_ok(p.q) && tma_ok(p.k) && tma_ok(p.v))) return GEOATTN_ERR_ALIGNMENT;
  if (d.tail) p.q0 = d.Nq - d.tail, p.rq = d.tail;
  int rc = d.fwd_rows ? forward_rows(p, d, st)
           : d.bf16   ? forward_tc(p, d, ws.ids, st)
                      : forward_simt(p, d, st);
  if (!rc && d.tail) rc = forward_simt(p, d, st);
  if (rc || d.splits == 1) return rc;
  const long long rows = (long long)d.B * d.H * d.Nq;
  return d.bf16 ? xlaunch(xattn_combine_kernel<__nv_bfloat16>, (rows + 7) / 8, 256, 0, st, p)
                : xlaunch(xattn_combine_kernel<float>, (rows + 7) / 8, 256, 0, st, p);
}

int geoattn_xattn_bwd(const GeoXattnBwdArgs* a, void* stream) {
  if (!a) return GEOATTN_ERR_INVALID;
  XDims d;
  if (int rc = check_xshape(&a->in.shape, d)) return rc;
  if (int rc = check_inputs(a->in, d)) return rc;
  if (!dev_ptr(a->o.data) || !dev_ptr(a->dout.data) || !dev_ptr(a->stats) || !dev_ptr(a->dq) || !dev_ptr(a->dk) ||
      !dev_ptr(a->dv) || (d.T && !dev_ptr(a->dtable)) || !dev_ptr(a->workspace))
    return GEOATTN_ERR_INVALID;
  if (a->o.stride[3] != 1 || a->dout.stride[3] != 1 || a->dq_stride[3] != 1 || a->dk_stride[3] != 1 ||
      a->dv_stride[3] != 1 || (reinterpret_cast<uintptr_t>(a->workspace) & (kAlign - 1)))
    return GEOATTN_ERR_ALIGNMENT;
  if (!bind_context()) return GEOATTN_ERR_LAUNCH;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  XBwdWs ws;
  xbwd_ws(d, reinterpret_cast<uint8_t*>(a->workspace), &ws);
  XParams p = xparams(a->in, d);
  p.o = xt(a->o.data, a->o.stride), p.dout = xt(a->dout.data, a->dout.stride);
  p.dq = xt(a->dq, a->dq_stride), p.dk = xt(a->dk, a->dk_stride), p.dv = xt(a->dv, a->dv_stride);
  p.stats = reinterpret_cast<float2*>(const_cast<float*>(a->stats)), p.delta = ws.delta, p.rec = ws.rec, p.ds = ws.ds;
  p.idsT = ws.idsT, p.status = ws.status;
  p.nqp = d.nqb, p.splits = d.bwd_splits, p.part_o = ws.part_dq;
  if (d.bf16 && !(tma_ok(p.q) && tma_ok(p.k) && tma_ok(p.v) && tma_ok(p.dout))) return GEOATTN_ERR_ALIGNMENT;
  xa::XMaps maps;
  std::memset(&maps, 0, sizeof(maps));
  int rc = d.bf16 && !d.bwd_rows ? backward_maps(maps, p, d) : GEOATTN_OK;
  if (rc) return rc;
  rc = d.bwd_rows ? GEOATTN_OK
       : d.bf16   ? records(p, d, st)
                  : xlaunch(xattn_delta_kernel, ((long long)d.B * d.H * d.Nq + 31) / 32, 256, 0, st, p);
  if (rc) return rc;
  if (d.T) {
    ids_tile_kernel<true><<<dim3((d.nqb + 63) / 64, d.nkp / 64), 256, 0, st>>>(p.ids, p.ids_ld, d.Nq, d.Nk, d.nqb, d.T,
                                                                              ws.idsT);
    if ((rc = status_of(cudaGetLastError()))) return rc;
  }
  const int units = d.B * d.Hkv;
  for (int l = 0; l < d.launches; ++l) {
    p.u0 = l * d.units_per_launch;
    const int nu = units - p.u0 < d.units_per_launch ? units - p.u0 : d.units_per_launch;
    rc = d.bwd_rows ? d.bf16 ? backward_rows<__nv_bfloat16>(p, d, nu, st) : backward_rows<float>(p, d, nu, st)
         : d.bf16   ? backward_tc(maps, p, d, nu, st)
                    : backward_simt(p, d, nu, st);
    if (rc) return rc;
    if (d.T) {
      float* part = ws.part + (size_t)l * d.H * d.chunks * d.T;
      rc = d.bf16 ? table_grad<__nv_bfloat16>(p, d, nu, part, st) : table_grad<float>(p, d, nu, part, st);
      if (rc) return rc;
    }
  }
  if (d.bwd_splits > 1) {
    const long long grid = ((long long)d.B * d.H * d.Nq * d.D + 255) / 256;
    rc = d.bf16 ? xlaunch(xattn_rows_dq_sum_kernel<__nv_bfloat16>, grid, 256, 0, st, p)
                : xlaunch(xattn_rows_dq_sum_kernel<float>, grid, 256, 0, st, p);
    if (rc) return rc;
  }
  if (d.T) {
    table_grad_sum_kernel<<<d.H * d.T, 32, 0, st>>>(ws.part, d.launches, d.H, d.chunks, d.T, a->dtable,
                                                    a->in.shape.table_dtype == GEOATTN_DTYPE_BF16);
    rc = status_of(cudaGetLastError());
  }
  return rc;
}

int geoattn_distance_buckets(int nq, const double* lat_q, const double* lon_q, int nk, const double* lat_k,
                             const double* lon_k, const double* edges, int nedges, double max_km, unsigned char* ids,
                             void* stream) {
  if (nq <= 0 || nk <= 0 || nedges < 0) return GEOATTN_ERR_INVALID;
  if (nedges >= kMaxBuckets) return GEOATTN_ERR_UNSUPPORTED;
  if (!dev_ptr(lat_q) || !dev_ptr(lon_q) || !dev_ptr(lat_k) || !dev_ptr(lon_k) || (nedges && !dev_ptr(edges)) ||
      !dev_ptr(ids))
    return GEOATTN_ERR_INVALID;
  const long long blocks = ((long long)nq * nk + 255) / 256;
  if (blocks > (1ll << 31) - 1) return GEOATTN_ERR_UNSUPPORTED;
  distance_buckets_kernel<<<(unsigned)blocks, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      nq, lat_q, lon_q, nk, lat_k, lon_k, edges, nedges, max_km, ids);
  return status_of(cudaGetLastError());
}

int geoattn_dropout(int dtype, long long n, const void* x, const void* residual, void* y, const long long* rng,
                    int threshold, void* stream) {
  if (n <= 0 || threshold < 0 || threshold > 65536) return GEOATTN_ERR_INVALID;
  if (dtype != GEOATTN_DTYPE_BF16 && dtype != GEOATTN_DTYPE_FP32) return GEOATTN_ERR_INVALID;
  if (!dev_ptr(x) || !dev_ptr(y) || !dev_ptr(rng) || (residual && !dev_ptr(residual))) return GEOATTN_ERR_INVALID;
  const long long blocks = (n + 2047) / 2048;
  if (blocks > (1ll << 31) - 1) return GEOATTN_ERR_UNSUPPORTED;
  const float scale = threshold >= 65536 ? 0.f : (float)(65536.0 / (65536 - threshold));
  const int vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) |
                    reinterpret_cast<uintptr_t>(residual)) & 15) == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto kernel, auto* e) {
    using E = std::remove_pointer_t<decltype(e)>;
    kernel<<<(unsigned)blocks, 256, 0, st>>>(reinterpret_cast<const E*>(x), reinterpret_cast<const E*>(residual),
                                             reinterpret_cast<E*>(y), n, rng, threshold, scale, vec);
  };
  if (dtype == GEOATTN_DTYPE_BF16) {
    if (residual) go(dropout_kernel<__nv_bfloat16, true>, (__nv_bfloat16*)nullptr);
    else go(dropout_kernel<__nv_bfloat16, false>, (__nv_bfloat16*)nullptr);
  } else {
    if (residual) go(dropout_kernel<float, true>, (float*)nullptr);
    else go(dropout_kernel<float, false>, (float*)nullptr);
  }
  return status_of(cudaGetLastError());
}

int geoattn_rng_take(long long* state, long long* out, void* stream) {
  if (!dev_ptr(state) || !dev_ptr(out)) return GEOATTN_ERR_INVALID;
  rng_take_kernel<<<1, 1, 0, reinterpret_cast<cudaStream_t>(stream)>>>(state, out);
  return status_of(cudaGetLastError());
}

}  // extern "C"
