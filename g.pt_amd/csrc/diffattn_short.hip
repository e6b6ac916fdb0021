// Differential attention over Tq, Tk <= 32 tokens (the denoiser's own sequences: 18 and 26), forward and backward: one wave per
// (sample, head), everything between loads and stores in registers and the wave's own LDS.
//
// Each operand is read once.  What is used by rows only (the forward's K, the backward's V) goes straight to registers, the others to
// LDS by DMA (buffer loads: rows behind the sample's end lie outside the buffer's range and arrive as zeros), in rows of 2 hd
// elements; the outputs leave through the tiles of operands that are done with.  16-byte chunk c of row r is stored at chunk
// c ^ f(r), with f such that the lanes that LDS serves together hit different banks, by rows as well as in transposing reads.
// 32 x 32 tiles: S_i^T = K_i Q_i^T and dP^T = V dO^T with keys on the accumulator's rows and queries on its lanes: softmax and
// D_i = sum P_i dP are sums over a lane's registers and one exchange, in fp32 throughout.  The backward takes both transposed uses
// (dQ contracts over keys, dK and dV over queries) from one evaluation: dS_i^T is dQ's operand as it stands in the registers; dS_i
// and P go once through LDS for the other two.
// HBM-bound: the backward moves 11 row sets of Tq or Tk x 2 hd for some 2 MFLOP each.
#include "diffattn.h"

namespace diffattn {
namespace {

// rows [0, n) of `src` (row stride ld elements, valid rows: `valid` <= n) to the tile at `dst`; zeros from row `valid` on
template <typename T, int HD>
__device__ __forceinline__ void load_tile(const T* src, int64_t ld, int n, int valid, char* dst, int lane) {
  using L = Tile<T, HD>;
  const uint32_t bytes = valid > 0 ? (uint32_t)(((int64_t)(valid - 1) * ld + 2 * HD) * L::ES) : 0u;
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)src, 0, bytes, 0x00020000);
  const int chunks = n * L::CPR;
#pragma unroll 4
  for (int c0 = 0; c0 < chunks; c0 += 64) {
    const int ci = c0 + lane, row = ci / L::CPR, pos = ci - row * L::CPR;
    const uint32_t off = (uint32_t)(row * (uint32_t)(ld * L::ES)) + (uint32_t)((pos ^ L::f(row)) << 4);
    if (ci < chunks) __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)(dst + c0 * 16), 16, off, 0, 0, 0);
  }
}

// S[row of A][row of B] over chunks [c0, c0 + n) of both tiles; ra / rb: this lane's row address base (row, or the zero chunk)
template <typename T, int HD>
__device__ __forceinline__ f32x16 rows_product(const char* ta, bool ina, const char* tb, bool inb, int r, int hh, int c0, int n, const char* zero) {
  using L = Tile<T, HD>;
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
// rows in the operand: 0 = an accumulator's (operand_from), 1 = ascending (bf16: 16 s + 8 hh + j; fp32: 2 e + hh).  rest: X's second operand, if any
template <typename T, int HD, int ORDER, typename... Rest>
__device__ __forceinline__ f32x16 columns_product(const char* tile, int n, int t, const Operand& x, int lane, const char* zero, const Rest&... rest) {
  using L = Tile<T, HD>;
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
template <typename T, int HD>
__device__ __forceinline__ void stage(char* tile, int r, int hh, int t, const f32x16& acc, float scale) {
  using L = Tile<T, HD>;
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
template <typename T, int HD>
__device__ __forceinline__ void store_tile(T* dst, int64_t ld, int n, const char* tile, int lane) {
  using L = Tile<T, HD>;
  const int chunks = n * L::CPR;
#pragma unroll 4
  for (int ci = lane; ci < chunks; ci += 64) {
    const int row = ci / L::CPR, c = ci - row * L::CPR;
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

template <typename T, int HD>
__global__ __launch_bounds__(64, sizeof(T) == 2 ? 3 : 1) void short_fwd_kernel(Args a) {
  using L = Tile<T, HD>;
  constexpr int NT = 2 * HD / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x, r = lane & 31, hh = lane >> 5;
  const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H, len = valid_keys(a, b);
  char *tq = smem, *tv = tq + a.Tq * L::PITCH, *zero = tv + a.Tk * L::PITCH;
  if (lane < 4) reinterpret_cast<uint32_t*>(zero)[lane] = 0u;
  load_tile<T, HD>((const T*)a.q + (int64_t)b * a.bsq + h * 2 * HD, a.ldq, a.Tq, a.Tq, tq, lane);
  // K is only used by rows, once: straight to registers
  const bool kok = r < len, qok = r < a.Tq;
  u32x4 kf[L::CPR / 2];
  {
    const u32x4* kr = reinterpret_cast<const u32x4*>((const T*)a.k + (int64_t)b * a.bsk + (int64_t)(kok ? r : 0) * a.ldk + h * 2 * HD);
#pragma unroll
    for (int c = 0; c < L::CPR / 2; ++c) {
      kf[c] = u32x4{0u, 0u, 0u, 0u};
      if (kok) kf[c] = kr[2 * c + hh];
    }
  }
  load_tile<T, HD>((const T*)a.v + (int64_t)b * a.bsv + h * 2 * HD, a.ldv, a.Tk, len, tv, lane);
  const float lam = a.lam[h];
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  f32x16 s[2] = {zero16(), zero16()};
#pragma unroll
  for (int c = 0; c < L::CPR / 2; ++c) {
    const int m = c >= L::CM / 2;
    s[m] = mma_chunk<T>(kf[c], *reinterpret_cast<const u32x4*>(qok ? tq + L::at(r, 2 * c + hh) : zero), s[m]);
  }
#pragma unroll
  for (int m = 0; m < 2; ++m) softmax32(s[m], len, hh, a.c2);
  Operand p, rest;
#pragma unroll
  for (int e = 0; e < 16; ++e) s[0][e] -= lam * s[1][e];
  operand_from<T>(p, s[0]);                                 // the difference of the maps; bf16: in two operands, 16 bits
  if constexpr (sizeof(T) == 2) operand_rest(rest, s[0], p);
  lds_done();                                               // Q has been read: its tile takes the output
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    f32x16 o;
    if constexpr (sizeof(T) == 2) o = columns_product<T, HD, 0>(tv, a.Tk, t, p, lane, zero, rest);
    else o = columns_product<T, HD, 0>(tv, a.Tk, t, p, lane, zero);
    if (qok) stage<T, HD>(tq, r, hh, t, o, 1.f);
  }
  lds_done();
  store_tile<T, HD>((T*)a.out + (int64_t)b * a.bso + h * 2 * HD, a.ldo, a.Tq, tq, lane);
}

// A [query][key] matrix on its way through LDS: pitch in bytes (bf16: rows 18 banks apart, conflict-free for the 8-byte writes of 32
// rows and for the 4-row transposing reads)
template <typename T>
constexpr int P_PITCH = sizeof(T) == 2 ? 72 : 144;

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

template <typename T, int HD>
__global__ __launch_bounds__(64, sizeof(T) == 2 && HD < 128 ? 2 : 1) void short_bwd_kernel(Args a) {
  using L = Tile<T, HD>;
  constexpr int NT = 2 * HD / 32, HALF = NT / 2;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x, r = lane & 31, hh = lane >> 5;
  const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H, len = valid_keys(a, b);
  const int rows = a.Tq > a.Tk ? a.Tq : a.Tk;
  char *tq = smem, *tg = tq + rows * L::PITCH, *tk = tg + rows * L::PITCH, *tm = tk + rows * L::PITCH, *zero = tm + a.Tq * P_PITCH<T>;
  if (lane < 4) reinterpret_cast<uint32_t*>(zero)[lane] = 0u;
  load_tile<T, HD>((const T*)a.q + (int64_t)b * a.bsq + h * 2 * HD, a.ldq, a.Tq, a.Tq, tq, lane);
  load_tile<T, HD>((const T*)a.k + (int64_t)b * a.bsk + h * 2 * HD, a.ldk, a.Tk, len, tk, lane);
  load_tile<T, HD>((const T*)a.dout + (int64_t)b * a.bsdo + h * 2 * HD, a.lddo, a.Tq, a.Tq, tg, lane);
  // V is only used by rows, once: straight to registers, no LDS (5 instead of 4 waves per CU at 26 tokens, hd 96)
  const bool qok = r < a.Tq, kok = r < a.Tk, vok = r < len;
  u32x4 vf[L::CPR / 2];
  {
    const u32x4* vr = reinterpret_cast<const u32x4*>((const T*)a.v + (int64_t)b * a.bsv + (int64_t)(vok ? r : 0) * a.ldv + h * 2 * HD);
#pragma unroll
    for (int c = 0; c < L::CPR / 2; ++c) {
      vf[c] = u32x4{0u, 0u, 0u, 0u};
      if (vok) vf[c] = vr[2 * c + hh];
    }
  }
  const float lam = a.lam[h];
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  f32x16 s[2], dp = zero16();
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    s[m] = rows_product<T, HD>(tk, kok, tq, qok, r, hh, m * L::CM, L::CM, zero);
    softmax32(s[m], len, hh, a.c2);
  }
#pragma unroll
  for (int c = 0; c < L::CPR / 2; ++c) dp = mma_chunk<T>(vf[c], *reinterpret_cast<const u32x4*>(qok ? tg + L::at(r, 2 * c + hh) : zero), dp);
  float d[2] = {0.f, 0.f};
#pragma unroll
  for (int m = 0; m < 2; ++m) {
#pragma unroll
    for (int e = 0; e < 16; ++e) d[m] += row_of(e, hh) < len ? s[m][e] * dp[e] : 0.f;
    d[m] = col_sum(d[m]);
  }
  const float dl = wave_sum(qok && hh == 0 ? d[1] : 0.f);
  if (lane == 0) a.dlam_part[(int64_t)h * a.B + b] = dl;
  f32x16 p;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const bool in = qok && row_of(e, hh) < len;
    p[e] = in ? s[0][e] - lam * s[1][e] : 0.f;
    s[0][e] = in ? s[0][e] * (dp[e] - d[0]) : 0.f;
    s[1][e] = in ? -lam * (s[1][e] * (dp[e] - d[1])) : 0.f;
  }
  // dS_i^T is dQ's operand as it stands; P, dS_1 and dS_2 go through the one matrix buffer in turn
  Operand x, xp, xs[2];
  if (qok) put_matrix<T>(tm, p, r, hh);
  lds_done();
  get_matrix<T>(xp, tm, a.Tq, lane, zero);
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    lds_done();
    if (qok) put_matrix<T>(tm, s[m], r, hh);
    lds_done();
    get_matrix<T>(xs[m], tm, a.Tq, lane, zero);
  }
  // each output leaves through the tile of the operand that its products have just read (all tiles have max(Tq, Tk) rows)
  f32x16 acc[NT];
  auto put = [&](char* tile, T* dst, int64_t ld, int n, float scale) {
    lds_done();
#pragma unroll
    for (int t = 0; t < NT; ++t)
      if (r < n) stage<T, HD>(tile, r, hh, t, acc[t], scale);
    lds_done();
    store_tile<T, HD>(dst, ld, n, tile, lane);
  };
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    operand_from<T>(x, s[m]);
#pragma unroll
    for (int t = m * HALF; t < (m + 1) * HALF; ++t) acc[t] = columns_product<T, HD, 0>(tk, a.Tk, t, x, lane, zero);       // dQ_m^T = K_m^T dS_m^T
  }
  put(tk, (T*)a.dq + (int64_t)b * a.bsdq + h * 2 * HD, a.lddq, a.Tq, a.scale);
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = columns_product<T, HD, 1>(tq, a.Tq, t, xs[t / HALF], lane, zero);                 // dK_m^T = Q_m^T dS_m
  put(tq, (T*)a.dk + (int64_t)b * a.bsdk + h * 2 * HD, a.lddk, a.Tk, a.scale);
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = columns_product<T, HD, 1>(tg, a.Tq, t, xp, lane, zero);                           // dV^T = dO^T P
  put(tg, (T*)a.dv + (int64_t)b * a.bsdv + h * 2 * HD, a.lddv, a.Tk, 1.f);
}

template <typename T, int HD>
int go(const Args& a, bool backward, hipStream_t s) {
  using L = Tile<T, HD>;
  static GptPerDevice fwd_once, bwd_once;
  const dim3 grid((unsigned)(a.B * a.H));
  if (!backward) {
    const char* who = "gpt_diff_attention";
    if (int st = grant_lds(short_fwd_kernel<T, HD>, fwd_once, who)) return st;
    hipLaunchKernelGGL((short_fwd_kernel<T, HD>), grid, dim3(64), (a.Tq + a.Tk) * L::PITCH + 16, s, a);
    return gpt_launch_status(who);
  }
  const char* who = "gpt_diff_attention_bwd";
  if (int st = grant_lds(short_bwd_kernel<T, HD>, bwd_once, who)) return st;
  const int lds = 3 * (a.Tq > a.Tk ? a.Tq : a.Tk) * L::PITCH + a.Tq * P_PITCH<T> + 16;
  hipLaunchKernelGGL((short_bwd_kernel<T, HD>), grid, dim3(64), lds, s, a);
  return gpt_launch_status(who);
}

}  // namespace

int short_attention(const Args& a, int dtype, int hd, bool backward, hipStream_t s) {
#define GO(T)                                 \
  switch (hd) {                               \
    case 32: return go<T, 32>(a, backward, s);  \
    case 64: return go<T, 64>(a, backward, s);  \
    case 96: return go<T, 96>(a, backward, s);  \
    default: return go<T, 128>(a, backward, s); \
  }
  if (dtype == GPT_BF16) GO(bf16_t)
  GO(float)
#undef GO
}

}  // namespace diffattn
