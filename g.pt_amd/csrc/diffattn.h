// What the differential-attention kernels share: the launch's arguments, 16 x 16 matrix-core tiles of both types, masks.
#pragma once
#include "common.h"

namespace diffattn {

constexpr float LOG2E = 1.4426950408889634f;

struct Args {
  const void *q, *k, *v;
  int64_t ldq, bsq, ldk, bsk, ldv, bsv;
  const float* lam;
  const int32_t* lengths;
  void* out;
  int64_t ldo, bso;
  float* lse;                 // [2][B][H][Tq], base 2, of the scaled scores
  void* out2;                 // [B][Tq][H * 2 hd]
  float* part;                // split forward: [splits][B * H][Tq][4 hd + 4]
  int B, Tq, Tk, H, splits, split_keys;
  float scale, c2;            // c2 = scale * log2(e): exp(scale s - m) = exp2(c2 s - m')
  // backward
  const void* dout;
  int64_t lddo, bsdo;
  void *dq, *dk, *dv;
  int64_t lddq, bsdq, lddk, bsdk, lddv, bsdv;
  const float* delta;         // [2][B][H][Tq]: D_1, D_2
  float* dlam_part;           // [H][B * key tiles]
};

// Tq, Tk <= 32 (diffattn_short.hip); the backward needs dlam_part [H][B], no lse, out, out2 or delta
constexpr int SHORT = 32;
int short_attention(const Args& a, int dtype, int hd, bool backward, hipStream_t s);

__device__ __forceinline__ int valid_keys(const Args& a, int b) {
  if (!a.lengths) return a.Tk;
  const int n = a.lengths[b];
  return n < 0 ? 0 : n > a.Tk ? a.Tk : n;
}

// ---- 16 x 16 tiles: an operand fragment is 8 consecutive k-values of one row (row = lane & 15, k = 8 (lane >> 4) + j); the
// accumulator holds column lane & 15 and rows 4 (lane >> 4) + r.  bf16: one 16x16x32 instruction; fp32: eight 16x16x4 ones, the
// j-th on the j-th values (any order of k serves as long as both operands use it).
template <typename T>
struct Frag;
template <>
struct Frag<bf16_t> {
  bf16x8 v;
};
template <>
struct Frag<float> {
  float v[8];
};

__device__ __forceinline__ void frag_zero(Frag<bf16_t>& f) { f.v = bf16x8{0, 0, 0, 0, 0, 0, 0, 0}; }
__device__ __forceinline__ void frag_zero(Frag<float>& f) {
#pragma unroll
  for (int j = 0; j < 8; ++j) f.v[j] = 0.f;
}
// 8 consecutive elements at p (16-byte aligned), zeros where !ok
__device__ __forceinline__ Frag<bf16_t> frag_row(const bf16_t* p, bool ok) {
  Frag<bf16_t> f;
  frag_zero(f);
  if (ok) f.v = *reinterpret_cast<const bf16x8*>(p);
  return f;
}
__device__ __forceinline__ Frag<float> frag_row(const float* p, bool ok) {
  Frag<float> f;
  frag_zero(f);
  if (ok) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f.v[0] = a.x; f.v[1] = a.y; f.v[2] = a.z; f.v[3] = a.w; f.v[4] = b.x; f.v[5] = b.y; f.v[6] = b.z; f.v[7] = b.w;
  }
  return f;
}
// element `col` of the 8 rows that two accumulator tiles of 16 rows give a lane, in their order: row 16 (j >> 2) + 4 g + (j & 3),
// g = lane >> 4; rows >= n (counted from the tile's first) are zero
template <typename T>
__device__ __forceinline__ Frag<T> frag_column(const T* base, int64_t ld, int g, int n) {
  Frag<T> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int r = 16 * (j >> 2) + 4 * g + (j & 3);
    T t = 0;
    if (r < n) t = base[(int64_t)r * ld];
    if constexpr (sizeof(T) == 2) f.v[j] = (short)t;
    else f.v[j] = t;
  }
  return f;
}
// two accumulator tiles (rows 0..15 and 16..31 of the contraction) as an operand; bf16: rounded once
__device__ __forceinline__ void frag_from(Frag<bf16_t>& f, const f32x4& lo, const f32x4& hi) {
  const uint32_t w[4] = {pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3]), pack_bf16x2(hi[0], hi[1]), pack_bf16x2(hi[2], hi[3])};
  f.v = __builtin_bit_cast(bf16x8, u32x4{w[0], w[1], w[2], w[3]});
}
__device__ __forceinline__ void frag_from(Frag<float>& f, const f32x4& lo, const f32x4& hi) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f.v[j] = lo[j];
    f.v[4 + j] = hi[j];
  }
}
__device__ __forceinline__ f32x4 mma16(const Frag<bf16_t>& a, const Frag<bf16_t>& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(const Frag<float>& a, const Frag<float>& b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
  return c;
}

// 4 consecutive values to memory
__device__ __forceinline__ void store4(bf16_t* p, const f32x4& v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}
__device__ __forceinline__ void store4(float* p, const f32x4& v) { *reinterpret_cast<f32x4*>(p) = v; }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }   // v_exp_f32, 1 ulp; exp2(-inf) = 0

// max / sum over the four lanes that hold one accumulator column
__device__ __forceinline__ float col_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float col_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

}  // namespace diffattn
