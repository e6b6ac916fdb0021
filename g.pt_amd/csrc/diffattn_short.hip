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
// bf16: P and dS enter their products as two operands each (16 bits of mantissa; the values are exact products of them), so the
// results' own rounding is the only one to 8 bits.  HBM-bound, which is why that costs little: the backward reads 4 row sets of Tq or
// Tk x 2 hd and writes 3 for some 2 MFLOP each, the forward 3 and 1.  1024 samples x 26 tokens, 8 heads of 2 x 96, bf16: forward
// 74 us (64 at a copy's rate), backward 133 (111; 124 with one operand, whose dQ, dK, dV are off by 2.35e-3 rms instead of
// 1.66e-3); 64 samples forward 7.6.
#include "short_tiles.h"

namespace diffattn {
namespace {

template <typename T, int HD>
__global__ __launch_bounds__(64, sizeof(T) == 2 ? 3 : 1) void short_fwd_kernel(Args a) {
  using L = Tile<T, HD>;
  constexpr int NT = 2 * HD / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x, r = lane & 31, hh = lane >> 5;
  const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H, len = valid_keys(a, b);
  char *tq = smem, *tv = tq + a.Tq * L::PITCH, *zero = tv + a.Tk * L::PITCH;
  if (lane < 4) reinterpret_cast<uint32_t*>(zero)[lane] = 0u;
  load_tile<T, L>((const T*)a.q + (int64_t)b * a.bsq + h * 2 * HD, a.ldq, a.Tq, a.Tq, tq, lane);
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
  load_tile<T, L>((const T*)a.v + (int64_t)b * a.bsv + h * 2 * HD, a.ldv, a.Tk, len, tv, lane);
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
    if constexpr (sizeof(T) == 2) o = columns_product<T, L, 0>(tv, a.Tk, t, p, lane, zero, rest);
    else o = columns_product<T, L, 0>(tv, a.Tk, t, p, lane, zero);
    if (qok) stage<T, L>(tq, r, hh, t, o, 1.f);
  }
  lds_done();
  store_tile<T, L>((T*)a.out + (int64_t)b * a.bso + h * 2 * HD, a.ldo, a.Tq, tq, lane);
}

template <typename T, int HD>
__global__ __launch_bounds__(64, sizeof(T) == 2 && HD < 128 ? 2 : 1) void short_bwd_kernel(Args a) {
  using L = Tile<T, HD>;
  constexpr int NT = 2 * HD / 32, HALF = NT / 2, PARTS = sizeof(T) == 2 ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x, r = lane & 31, hh = lane >> 5;
  const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H, len = valid_keys(a, b);
  const int rows = a.Tq > a.Tk ? a.Tq : a.Tk;
  char *tq = smem, *tg = tq + rows * L::PITCH, *tk = tg + rows * L::PITCH, *tm = tk + rows * L::PITCH, *zero = tm + matrix_bytes<T>(a.Tq);
  if (lane < 4) reinterpret_cast<uint32_t*>(zero)[lane] = 0u;
  load_tile<T, L>((const T*)a.q + (int64_t)b * a.bsq + h * 2 * HD, a.ldq, a.Tq, a.Tq, tq, lane);
  load_tile<T, L>((const T*)a.k + (int64_t)b * a.bsk + h * 2 * HD, a.ldk, a.Tk, len, tk, lane);
  load_tile<T, L>((const T*)a.dout + (int64_t)b * a.bsdo + h * 2 * HD, a.lddo, a.Tq, a.Tq, tg, lane);
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
    s[m] = rows_product<T, L>(tk, kok, tq, qok, r, hh, m * L::CM, L::CM, zero);
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
  // dS_i^T is dQ's operand as it stands; P, dS_1 and dS_2 go through the one matrix buffer in turn, in bf16 each as two operands
  Operand x, low, xp[2], xs[2][2];
  auto turn = [&](Operand (&o)[2], f32x16 m) {
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      lds_done();
      if (qok) put_matrix<T>(tm, m, r, hh);
      lds_done();
      get_matrix<T>(o[part], tm, a.Tq, lane, zero);
      if constexpr (PARTS == 2)
#pragma unroll
        for (int e = 0; e < 16; ++e) m[e] -= bf16_to_f32(f32_to_bf16(m[e]));   // what put_matrix's rounding leaves
    }
  };
  turn(xp, p);
#pragma unroll
  for (int m = 0; m < 2; ++m) turn(xs[m], s[m]);
  auto product = [&](auto order, const char* tile, int n, int t, const Operand& hi, const Operand& lo) {
    if constexpr (PARTS == 2) return columns_product<T, L, order.value>(tile, n, t, hi, lane, zero, lo);
    else return columns_product<T, L, order.value>(tile, n, t, hi, lane, zero);
  };
  constexpr std::integral_constant<int, 0> by_key{};
  constexpr std::integral_constant<int, 1> by_query{};
  // each output leaves through the tile of the operand that its products have just read (all tiles have max(Tq, Tk) rows)
  f32x16 acc[NT];
  auto put = [&](char* tile, T* dst, int64_t ld, int n, float scale) {
    lds_done();
#pragma unroll
    for (int t = 0; t < NT; ++t)
      if (r < n) stage<T, L>(tile, r, hh, t, acc[t], scale);
    lds_done();
    store_tile<T, L>(dst, ld, n, tile, lane);
  };
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    operand_from<T>(x, s[m]);
    if constexpr (PARTS == 2) operand_rest(low, s[m], x);
#pragma unroll
    for (int t = m * HALF; t < (m + 1) * HALF; ++t) acc[t] = product(by_key, tk, a.Tk, t, x, low);                          // dQ_m^T = K_m^T dS_m^T
  }
  put(tk, (T*)a.dq + (int64_t)b * a.bsdq + h * 2 * HD, a.lddq, a.Tq, a.scale);
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = product(by_query, tq, a.Tq, t, xs[t / HALF][0], xs[t / HALF][PARTS - 1]);        // dK_m^T = Q_m^T dS_m
  put(tq, (T*)a.dk + (int64_t)b * a.bsdk + h * 2 * HD, a.lddk, a.Tk, a.scale);
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = product(by_query, tg, a.Tq, t, xp[0], xp[PARTS - 1]);                            // dV^T = dO^T P
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
  const int lds = 3 * (a.Tq > a.Tk ? a.Tq : a.Tk) * L::PITCH + matrix_bytes<T>(a.Tq) + 16;
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
