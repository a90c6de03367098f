// Counter-based random bits for dropout: Philox4x32 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC'11). One call maps a 128-bit counter and a 64-bit key to four 32-bit words, so any element's bits can
// be recomputed anywhere from its indexes and no mask is ever stored.
//
// 7 rounds: the fewest that the paper reports as passing its whole battery of tests; a round costs two 32x32->64
// products, two three-way xors and two key additions, and the attention kernels are bound by such integer work.
// 16 bits per element: an element is kept when its 16 bits are >= threshold = round(65536 p), so p is met to 2^-17 and
// the scale 65536 / (65536 - threshold) is exact for the probability that is really used.
#pragma once
#include <cstdint>

namespace geoattn {

struct PhiloxKey {
  uint32_t k0, k1;
};

__device__ __forceinline__ uint4 philox7(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, PhiloxKey key) {
  uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    const uint32_t n0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0, n2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Bit e of the result: element e of the call's eight is kept (word e / 2, low half first).
__device__ __forceinline__ uint32_t keep_bits8(uint4 w, uint32_t thr) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m |= ((x[i] & 0xFFFFu) >= thr ? 1u : 0u) << (2 * i);
    m |= ((x[i] >> 16) >= thr ? 1u : 0u) << (2 * i + 1);
  }
  return m;
}

// Two elements at once: bit 15 of the result is set where the low half of x is >= the low half of t (an unsigned
// 16-bit comparison), bit 31 for the high halves; the other bits are arbitrary. t holds the threshold twice.
__device__ __forceinline__ uint32_t keep_pair(uint32_t x, uint32_t t) {
  // the low 15 bits are compared by a subtraction that cannot borrow across the halves, the top bits by logic
  const uint32_t low = (x | 0x80008000u) - (t & 0x7FFF7FFFu);
  return (x & ~t) | (~(x ^ t) & low);
}
// 0xFFFF in each half whose bit 15 / 31 is set; all ones where bit 15 (HALF = 0) or bit 31 (HALF = 1) is.
// (prmt with bit 3 of a selector set replicates the chosen byte's sign.)
template <uint32_t SEL>
__device__ __forceinline__ uint32_t spread_signs(uint32_t d) {
  uint32_t r;
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(r) : "r"(d), "n"(SEL));
  return r;
}
__device__ __forceinline__ uint32_t spread_pair(uint32_t d) { return spread_signs<0xBB99>(d); }
template <int HALF>
__device__ __forceinline__ uint32_t spread_one(uint32_t d) {
  return spread_signs<HALF ? 0xBBBB : 0x9999>(d);
}

// Attention weights: element (b, h, i, j) is bit j % 8 of counter (j / 8, i, b * H + h, offset low) under the key
// (seed low, seed high ^ offset high). `rng` is (seed, offset) in device memory, so a captured graph sees new values.
struct AttnDrop {
  PhiloxKey key;
  uint32_t off, thr;
  float scale;  // 65536 / (65536 - thr)
  __device__ __forceinline__ uint32_t keep8(uint32_t i, uint32_t j8, uint32_t bh) const {
    return keep_bits8(philox7(j8, i, bh, off, key), thr);
  }
  __device__ __forceinline__ uint4 words(uint32_t i, uint32_t j8, uint32_t bh) const {
    return philox7(j8, i, bh, off, key);
  }
  __device__ __forceinline__ uint32_t pair() const { return thr * 0x10001u; }  // the threshold (< 65536) in both halves
};

__device__ __forceinline__ AttnDrop attn_drop(const long long* rng, int thr, float scale) {
  AttnDrop d{{0, 0}, 0, (uint32_t)thr, scale};
  if (thr > 0) {
    const unsigned long long seed = (unsigned long long)rng[0], off = (unsigned long long)rng[1];
    // the same in every lane; a warp-wide reduction puts the words into uniform registers, where the rounds' keys cost
    // the vector units nothing
    d.key = {__reduce_or_sync(0xffffffffu, (uint32_t)seed),
             __reduce_or_sync(0xffffffffu, (uint32_t)(seed >> 32) ^ (uint32_t)(off >> 32))};
    d.off = __reduce_or_sync(0xffffffffu, (uint32_t)off);
  }
  return d;
}

}  // namespace geoattn
