// Counter-based dropout masks.  Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011),
// the generator of gpt_randn, gives 128 bits per counter; they are read as EIGHT 16-bit numbers, so one block of ten rounds serves
// eight consecutive elements:
//   element i (row * d + column of the logical tensor): counter = (i >> 3, offset), key = seed,
//   u_i = 16 bits: word (i & 7) >> 1, its low half for even i, its high half for odd i;
//   kept iff u_i >= thr,  thr = p rounded to 1 / 65536;  kept values are multiplied by 65536 / (65536 - thr).
// With 32 bits per element the ten rounds (20 quarter-rate 32 x 32 -> 64 multiplies per 4 elements) cost as much issue time as the
// 10 bytes per element of a bf16 dropout + fp32 residual addition cost HBM time; with 16 bits they stay below it.
#pragma once
#include "common.h"

struct DropoutRng {
  uint64_t seed, offset;
  const uint64_t* offset_dev;   // device counter added to offset, or NULL
  uint32_t thr;                 // 0: keep everything; 65536: keep nothing
  float scale;
};

// host: the launch's description of a caller's gpt_dropout_t (NULL: keep everything)
static inline int gpt_dropout_rng(const gpt_dropout_t* d, DropoutRng* r, const char* who) {
  *r = DropoutRng{0, 0, nullptr, 0, 1.f};
  if (!d) return 0;
  GPT_REQUIRE(d->p >= 0.0 && d->p <= 1.0, "%s: dropout probability %g not in [0, 1]", who, d->p);
  GPT_REQUIRE((uintptr_t)d->offset_dev % 8 == 0, "%s: misaligned device counter", who);
  const double t = d->p * 65536.0;
  uint32_t thr = (uint32_t)t;                                   // nearest, ties to even
  const double f = t - (double)thr;
  if (f > 0.5 || (f == 0.5 && (thr & 1u))) ++thr;
  *r = DropoutRng{d->seed, d->offset, d->offset_dev, thr, thr >= 65536u ? 0.f : (float)(65536.0 / (65536.0 - (double)thr))};
  return 0;
}

// the counter of the launch: uniform over the grid
__device__ __forceinline__ uint64_t dropout_offset(const DropoutRng& r) { return r.offset + (r.offset_dev ? *r.offset_dev : 0ull); }

// the eight 16-bit numbers of block `blk` as four words
__device__ __forceinline__ void philox_words(uint64_t blk, uint64_t seed, uint64_t offset, uint32_t (&c)[4]) {
  c[0] = (uint32_t)blk; c[1] = (uint32_t)(blk >> 32); c[2] = (uint32_t)offset; c[3] = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c[0], p1 = (uint64_t)0xCD9E8D57u * c[2];
    const uint32_t n0 = (uint32_t)(p1 >> 32) ^ c[1] ^ k0, n2 = (uint32_t)(p0 >> 32) ^ c[3] ^ k1;
    c[0] = n0; c[1] = (uint32_t)p1; c[2] = n2; c[3] = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// bit j: element 8 blk + j is kept
__device__ __forceinline__ uint32_t dropout_keep8(const DropoutRng& r, uint64_t offset, uint64_t blk) {
  uint32_t c[4], keep = 0;
  philox_words(blk, r.seed, offset, c);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t u = (j & 1) ? c[j >> 1] >> 16 : c[j >> 1] & 0xffffu;
    keep |= (u >= r.thr ? 1u : 0u) << j;
  }
  return keep;
}
// the same for one element
__device__ __forceinline__ bool dropout_keep1(const DropoutRng& r, uint64_t offset, uint64_t i) {
  return (dropout_keep8(r, offset, i >> 3) >> (i & 7)) & 1u;
}

// ---- 8 consecutive elements of a row as floats, from / to fp32 or bf16 memory (16-byte aligned)
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const bf16_t* p, float (&v)[8]) {
  const u32x4 a = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(a[i] << 16);
    v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(bf16_t* p, const float (&v)[8]) {
  u32x4 a;
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<u32x4*>(p) = a;
}

static inline bool aligned16(const void* p) { return ((uintptr_t)p % 16) == 0; }
// rows of `ld` elements of es bytes all start 16-byte aligned
static inline bool rows_aligned16(const void* p, int64_t ld, size_t es) { return aligned16(p) && (ld * (int64_t)es) % 16 == 0; }
