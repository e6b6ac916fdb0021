// What the kernels for at most 32 tokens share: one wave per (sample, head), tiles of up to 32 rows in the wave's own LDS.  L: the
// tile's layout (Tile, or what has its ES, COLS, PITCH, CPR, REAL and at()).
#pragma once
#include "diffattn.h"

namespace diffattn {

// rows [0, n) of `src` (row stride ld elements, valid rows: `valid` <= n) to the tile at `dst`; zeros from row `valid` on
template <typename T, typename L>
__device__ __forceinline__ void load_tile(const T* src, int64_t ld, int n, int valid, char* dst, int lane) {
  const uint32_t bytes = valid > 0 ? (uint32_t)(((int64_t)(valid - 1) * ld + L::COLS) * L::ES) : 0u;
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)src, 0, bytes, 0x00020000);
  const int chunks = n * L::CPR;
#pragma unroll 4
  for (int c0 = 0; c0 < chunks; c0 += 64) {
    const int ci = c0 + lane, row = ci / L::CPR, pos = ci - row * L::CPR;
    uint32_t off = (uint32_t)(row * (uint32_t)(ld * L::ES)) + (uint32_t)((pos ^ L::f(row)) << 4);
    if (L::REAL != L::CPR && (pos ^ L::f(row)) >= L::REAL) off = 0xfffffff0u;           // a row's padding: outside the buffer
    if (ci < chunks) __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)(dst + c0 * 16), 16, off, 0, 0, 0);
  }
}

// S[row of A][row of B] over chunks [c0, c0 + n) of both tiles; ra / rb: this lane's row address base (row, or the zero chunk)
template <typename T, typename L>
__device__ __forceinline__ f32x16 rows_product(const char* ta, bool ina, const char* tb, bool inb, int r, int hh, int c0, int n, const char* zero) {
  f32x16 acc = zero16();
#pragma unroll
  for (int ks = 0; ks < n / 2; ++ks) {
    const int c = c0 + 2 * ks + hh;
    const u32x4 a = *reinterpret_cast<const u32x4*>(ina ? ta + L::at(r, c) : zero);
    const u32x4 b = *reinterpret_cast<const u32x4*>(inb ? tb + L::at(r, c) : zero);
    acc = mma_chunk<T>(a, b, acc);
  }
  return acc;
}

// acc^T[column 32 t + i of the tile][lane's column of X] = sum over the tile's rows (n valid) of tile[row][..] X[row][..].  ORDER of the
// rows in the operand: 0 = an accumulator's (operand_from), 1 = ascending (bf16: 16 s + 8 hh + j; fp32: 2 e + hh).  rest: X's second
// operand, if any
template <typename T, typename L, int ORDER, typename... Rest>
__device__ __forceinline__ f32x16 columns_product(const char* tile, int n, int t, const Operand& x, int lane, const char* zero, const Rest&... rest) {
  f32x16 acc = zero16();
  if constexpr (sizeof(T) == 2) {
    const int gq = lane >> 4, tq = (lane & 15) >> 2, tp = lane & 3, hh = gq >> 1;
    const int chunk = t * 4 + 2 * (gq & 1) + (tp >> 1), in = 8 * (tp & 1);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int r0 = 16 * s + (ORDER ? 8 : 4) * hh + tq, r1 = r0 + (ORDER ? 4 : 8);
      const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_ptr)(r0 < n ? tile + L::at(r0, chunk) + in : zero));
      const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_ptr)(r1 < n ? tile + L::at(r1, chunk) + in : zero));
      const bf16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, x.p[s], acc, 0, 0, 0);
      ((acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, rest.p[s], acc, 0, 0, 0)), ...);
    }
  } else {
    const int r = lane & 31, hh = lane >> 5, col = t * 32 + r;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int row = ORDER ? 2 * e + hh : row_of(e, hh);
      const float v = *reinterpret_cast<const float*>(row < n ? tile + L::at(row, col >> 2) + (col & 3) * 4 : zero);
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(v, x.f[e], acc, 0, 0, 0);
    }
  }
  return acc;
}

// acc^T (columns 32 t .. of row r on this lane) to the staging tile
template <typename T, typename L>
__device__ __forceinline__ void stage(char* tile, int r, int hh, int t, const f32x16& acc, float scale) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 v = {acc[4 * g] * scale, acc[4 * g + 1] * scale, acc[4 * g + 2] * scale, acc[4 * g + 3] * scale};
    if constexpr (sizeof(T) == 2) store4((bf16_t*)(tile + L::at(r, t * 4 + g) + 8 * hh), v);
    else store4((float*)(tile + L::at(r, t * 8 + 2 * g + hh)), v);
  }
}

__device__ __forceinline__ void lds_done() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

// n rows of the staging tile to memory, 16 bytes per lane, whole rows
template <typename T, typename L>
__device__ __forceinline__ void store_tile(T* dst, int64_t ld, int n, const char* tile, int lane) {
  const int chunks = n * L::REAL;
#pragma unroll 4
  for (int ci = lane; ci < chunks; ci += 64) {
    const int row = ci / L::REAL, c = ci - row * L::REAL;
    *reinterpret_cast<u32x4*>((char*)(dst + (int64_t)row * ld) + c * 16) = *reinterpret_cast<const u32x4*>(tile + L::at(row, c));
  }
}

// softmax over the keys of this lane's query: s -> probabilities
__device__ __forceinline__ void softmax32(f32x16& s, int len, int hh, float c2) {
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    if (row_of(e, hh) >= len) s[e] = -INFINITY;
    m = fmaxf(m, s[e]);
  }
  m = fmaxf(m, __shfl_xor(m, 32, 64));
  const float ref = len > 0 ? m * c2 : 0.f;               // no key: exp2(-inf) = 0 everywhere
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    s[e] = exp2_fast(s[e] * c2 - ref);
    sum += s[e];
  }
  sum += __shfl_xor(sum, 32, 64);
  const float inv = len > 0 ? 1.f / sum : 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) s[e] *= inv;
}

// A [query][key] matrix on its way through LDS: pitch in bytes (bf16: rows 18 banks apart, conflict-free for the 8-byte writes of 32
// rows and for the 4-row transposing reads)
template <typename T>
constexpr int P_PITCH = sizeof(T) == 2 ? 72 : 144;
template <typename T>
__host__ __device__ constexpr int matrix_bytes(int n) { return (n * P_PITCH<T> + 15) / 16 * 16; }

template <typename T>
__device__ __forceinline__ void put_matrix(char* m, const f32x16& x, int r, int hh) {
#pragma unroll
  for (int g = 0; g < 4; ++g) store4((T*)(m + r * P_PITCH<T>) + 8 * g + 4 * hh, f32x4{x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]});
}
// n rows of it as an operand that contracts over the rows (queries, ascending), keys on the lanes
template <typename T>
__device__ __forceinline__ void get_matrix(Operand& o, const char* m, int n, int lane, const char* zero) {
  if constexpr (sizeof(T) == 2) {
    const int gq = lane >> 4, tq = (lane & 15) >> 2, tp = lane & 3;
    const int col = (16 * (gq & 1) + 4 * tp) * 2;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int r0 = 16 * s + 8 * (gq >> 1) + tq, r1 = r0 + 4;
      const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_ptr)(r0 < n ? m + r0 * P_PITCH<T> + col : zero));
      const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_ptr)(r1 < n ? m + r1 * P_PITCH<T> + col : zero));
      o.p[s] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int q = 2 * e + (lane >> 5);
      o.f[e] = *reinterpret_cast<const float*>(q < n ? m + q * P_PITCH<T> + (lane & 31) * 4 : zero);
    }
  }
}

}  // namespace diffattn
