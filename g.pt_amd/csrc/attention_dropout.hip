// Multi-head attention over T <= 32 tokens with dropout on its probabilities, forward and backward: what attention.hip computes, for a
// training step with attn_pdrop > 0 (Gpt/models/transformer.py:34-51).
//
//   P = softmax(q k^T / sqrt(hd)),   P~ = keep * s * P,   y = P~ v
//   dP = keep * s * (dy v^T),   D = sum_j P dP,   dS = P (dP - D),   dq = dS k / sqrt(hd),   dk = dS^T q / sqrt(hd),   dv = P~^T dy
// The mask is a function of (seed, offset, element): element (((sample * H + head) * T + query) * 32 + key), so a row's 32 bits are four
// Philox blocks; nothing is stored, the backward draws it again.
//
// One wave per (sample, head), keys on the accumulator's rows and queries on its lanes: softmax and D are sums over a lane's registers
// and one exchange.  A lane draws two of its row's four blocks, its other half the other two.  What is used by rows only (the
// forward's q and k, the backward's v) goes straight to registers, the rest to LDS by DMA; dS and P~ go once through LDS for the
// products that contract over queries.  HBM-bound: the forward moves 4 row sets of T x hd, the backward 7;
// 512 samples x 26 tokens, 16 heads of 96, bf16: 42 and 84 us, 3.9 and 3.4 TB/s (a copy reaches 5.1; the kernels without dropout take
// 38 and 93); 128 samples 14 and 32 us.
#include "philox.h"
#include "short_tiles.h"

namespace {
using namespace diffattn;

// Rows of hd elements, padded to whole 128 bytes for the swizzle of Tile (the padding is neither read from memory nor stored)
template <typename T, int HD>
struct HeadTile {
  static constexpr int ES = sizeof(T), COLS = HD, REAL = HD * ES / 16, PITCH = (HD * ES + 127) / 128 * 128, CPR = PITCH / 16;
  static constexpr int MASK = PITCH % 256 == 0 ? 15 : 7;
  __device__ static __forceinline__ int f(int r) {
    const int b0 = (r >> 2) & 1, b1 = (r >> 3) & 1, pair = ((b0 ^ b1) << 1) | b1;
    if constexpr (PITCH % 256 == 0) return ((r & 3) << 2) | pair;
    return (((r >> 1) & 1) << 2) | pair;
  }
  __device__ static __forceinline__ int at(int r, int chunk) { return r * PITCH + ((chunk ^ f(r)) << 4); }
};

struct AttArgs {
  const void *qkv, *dy;   // [B, T, 3 H hd], [B, T, H hd]
  void* out;              // y [B, t_out, H hd] or dqkv [B, T, 3 H hd]
  int B, T, t_out, H;
  float scale;
  DropoutRng rng;
};

// the 32 keep bits of row `row` of the masks (bit = key), in both lanes (half 0 and 1) that hold it
__device__ __forceinline__ uint32_t row_keep(const DropoutRng& rng, uint64_t offset, uint64_t row, int hh) {
  const uint32_t own = dropout_keep8(rng, offset, row * 4 + 2 * hh) | dropout_keep8(rng, offset, row * 4 + 2 * hh + 1) << 8;
  const uint32_t other = (uint32_t)__shfl_xor((int)own, 32, 64);
  return hh ? other | own << 16 : own | other << 16;
}

// this lane's row of a [T][ld] matrix, the half's chunks of hd columns; zeros behind row n
template <typename T, typename L>
__device__ __forceinline__ void load_row(u32x4 (&x)[L::REAL / 2], const T* src, int64_t ld, int r, int hh, int n) {
  const u32x4* p = reinterpret_cast<const u32x4*>(src + (int64_t)(r < n ? r : 0) * ld);
#pragma unroll
  for (int c = 0; c < L::REAL / 2; ++c) {
    x[c] = u32x4{0u, 0u, 0u, 0u};
    if (r < n) x[c] = p[2 * c + hh];
  }
}

template <typename T, int HD>
__global__ __launch_bounds__(64, sizeof(T) == 2 ? 4 : 2) void att_fwd_kernel(AttArgs a) {
  using L = HeadTile<T, HD>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x, r = lane & 31, hh = lane >> 5;
  const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H, d = a.H * HD, ld = 3 * d;
  const T* q = (const T*)a.qkv + (int64_t)b * a.T * ld + h * HD;
  char *tv = smem, *zero = tv + a.T * L::PITCH;
  if (lane < 4) reinterpret_cast<uint32_t*>(zero)[lane] = 0u;
  load_tile<T, L>(q + 2 * d, ld, a.T, a.T, tv, lane);
  u32x4 qf[L::REAL / 2], kf[L::REAL / 2];
  load_row<T, L>(kf, q + d, ld, r, hh, a.T);
  load_row<T, L>(qf, q, ld, r, hh, a.T);
  const uint32_t keep = row_keep(a.rng, dropout_offset(a.rng), (uint64_t)blockIdx.x * a.T + r, hh);
  f32x16 s = zero16();
#pragma unroll
  for (int c = 0; c < L::REAL / 2; ++c) s = mma_chunk<T>(kf[c], qf[c], s);
  softmax32(s, a.T, hh, a.scale * LOG2E);
#pragma unroll
  for (int e = 0; e < 16; ++e) s[e] = (keep >> row_of(e, hh)) & 1u ? s[e] * a.rng.scale : 0.f;
  Operand p;
  operand_from<T>(p, s);                                    // bf16: rounded once, as attention.hip rounds P
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  f32x16 o[HD / 32];
#pragma unroll
  for (int t = 0; t < HD / 32; ++t) o[t] = columns_product<T, L, 0>(tv, a.T, t, p, lane, zero);
  lds_done();                                               // V has been read: its tile takes the output
#pragma unroll
  for (int t = 0; t < HD / 32; ++t)
    if (r < a.t_out) stage<T, L>(tv, r, hh, t, o[t], 1.f);
  lds_done();
  store_tile<T, L>((T*)a.out + (int64_t)b * a.t_out * d + h * HD, d, a.t_out, tv, lane);
}

template <typename T, int HD>
__global__ __launch_bounds__(64, sizeof(T) == 2 ? 3 : 1) void att_bwd_kernel(AttArgs a) {
  using L = HeadTile<T, HD>;
  constexpr int NT = HD / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x, r = lane & 31, hh = lane >> 5;
  const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H, d = a.H * HD, ld = 3 * d;
  const T* q = (const T*)a.qkv + (int64_t)b * a.T * ld + h * HD;
  T* dq = (T*)a.out + (int64_t)b * a.T * ld + h * HD;
  char *tq = smem, *tk = tq + a.T * L::PITCH, *tg = tk + a.T * L::PITCH, *tm = tg + a.T * L::PITCH, *zero = tm + matrix_bytes<T>(a.T);
  if (lane < 4) reinterpret_cast<uint32_t*>(zero)[lane] = 0u;
  load_tile<T, L>(q, ld, a.T, a.T, tq, lane);
  load_tile<T, L>(q + d, ld, a.T, a.T, tk, lane);
  load_tile<T, L>((const T*)a.dy + (int64_t)b * a.T * d + h * HD, d, a.T, a.T, tg, lane);
  u32x4 vf[L::REAL / 2];
  load_row<T, L>(vf, q + 2 * d, ld, r, hh, a.T);
  const uint32_t keep = row_keep(a.rng, dropout_offset(a.rng), (uint64_t)blockIdx.x * a.T + r, hh);
  const bool ok = r < a.T;
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  f32x16 s = rows_product<T, L>(tk, ok, tq, ok, r, hh, 0, L::REAL, zero), dp = zero16();
#pragma unroll
  for (int c = 0; c < L::REAL / 2; ++c) dp = mma_chunk<T>(vf[c], *reinterpret_cast<const u32x4*>(ok ? tg + L::at(r, 2 * c + hh) : zero), dp);
  softmax32(s, a.T, hh, a.scale * LOG2E);
  float dd = 0.f;
  f32x16 p;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const bool in = (keep >> row_of(e, hh)) & 1u;
    p[e] = in && ok ? s[e] * a.rng.scale : 0.f;
    dp[e] = in ? dp[e] * a.rng.scale : 0.f;
    dd += row_of(e, hh) < a.T ? s[e] * dp[e] : 0.f;
  }
  dd = col_sum(dd);
#pragma unroll
  for (int e = 0; e < 16; ++e) s[e] = ok && row_of(e, hh) < a.T ? s[e] * (dp[e] - dd) : 0.f;
  // dS^T is dQ's operand as it stands; P~ and dS go through the one matrix buffer in turn
  Operand x, xp, xs;
  if (ok) put_matrix<T>(tm, p, r, hh);
  lds_done();
  get_matrix<T>(xp, tm, a.T, lane, zero);
  lds_done();
  if (ok) put_matrix<T>(tm, s, r, hh);
  lds_done();
  get_matrix<T>(xs, tm, a.T, lane, zero);
  operand_from<T>(x, s);
  // each output leaves through the tile of the operand that its products have just read
  f32x16 acc[NT];
  auto put = [&](char* tile, T* dst, float scale) {
    lds_done();
#pragma unroll
    for (int t = 0; t < NT; ++t)
      if (ok) stage<T, L>(tile, r, hh, t, acc[t], scale);
    lds_done();
    store_tile<T, L>(dst, ld, a.T, tile, lane);
  };
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = columns_product<T, L, 0>(tk, a.T, t, x, lane, zero);      // dQ^T = K^T dS^T
  put(tk, dq, a.scale);
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = columns_product<T, L, 1>(tq, a.T, t, xs, lane, zero);     // dK^T = Q^T dS
  put(tq, dq + d, a.scale);
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = columns_product<T, L, 1>(tg, a.T, t, xp, lane, zero);     // dV^T = dO^T P~
  put(tg, dq + 2 * d, 1.f);
}

template <typename T, int HD>
int go(const AttArgs& a, bool backward, const char* who, hipStream_t s) {
  using L = HeadTile<T, HD>;
  static GptPerDevice fwd_once, bwd_once;
  const dim3 grid((unsigned)(a.B * a.H));
  if (!backward) {
    if (int st = grant_lds(att_fwd_kernel<T, HD>, fwd_once, who)) return st;
    hipLaunchKernelGGL((att_fwd_kernel<T, HD>), grid, dim3(64), a.T * L::PITCH + 16, s, a);
  } else {
    if (int st = grant_lds(att_bwd_kernel<T, HD>, bwd_once, who)) return st;
    hipLaunchKernelGGL((att_bwd_kernel<T, HD>), grid, dim3(64), 3 * a.T * L::PITCH + matrix_bytes<T>(a.T) + 16, s, a);
  }
  return gpt_launch_status(who);
}

int attention(int dtype, const void* qkv, const void* dy, void* out, int B, int T, int t_out, int n_head, int hd, const gpt_dropout_t* drop,
              bool backward, const char* who, void* stream) {
  GPT_REQUIRE(dtype == GPT_F32 || dtype == GPT_BF16, "%s: bad dtype %d", who, dtype);
  GPT_REQUIRE(qkv && out && drop && (dy || !backward), "%s: null operand", who);
  GPT_REQUIRE(B > 0 && T > 0 && T <= 32 && n_head > 0, "%s: need B > 0, 0 < T <= 32, n_head > 0 (B=%d T=%d H=%d)", who, B, T, n_head);
  GPT_REQUIRE(hd == 32 || hd == 64 || hd == 96 || hd == 128, "%s: unsupported head dim %d (32, 64, 96, 128)", who, hd);
  GPT_REQUIRE(t_out > 0 && t_out <= T, "%s: stored rows %d out of range (T=%d)", who, t_out, T);
  GPT_REQUIRE((int64_t)B * n_head < (1 << 26) && (int64_t)n_head * hd < (1 << 22), "%s: too large (B=%d H=%d)", who, B, n_head);
  GPT_REQUIRE((uintptr_t)qkv % 16 == 0 && (uintptr_t)dy % 16 == 0 && (uintptr_t)out % 16 == 0, "%s: operands must be 16-byte aligned", who);
  AttArgs a = {qkv, dy, out, B, T, t_out, n_head, 1.f / sqrtf((float)hd), {}};
  if (int st = gpt_dropout_rng(drop, &a.rng, who)) return st;
  hipStream_t s = (hipStream_t)stream;
#define GO(TT)                                            \
  switch (hd) {                                           \
    case 32: return go<TT, 32>(a, backward, who, s);      \
    case 64: return go<TT, 64>(a, backward, who, s);      \
    case 96: return go<TT, 96>(a, backward, who, s);      \
    default: return go<TT, 128>(a, backward, who, s);     \
  }
  if (dtype == GPT_BF16) GO(bf16_t)
  GO(float)
#undef GO
}

}  // namespace

extern "C" int gpt_attention_dropout(int dtype, const void* qkv, void* y, int B, int T, int t_out, int n_head, int hd, const gpt_dropout_t* drop,
                                     void* stream) {
  return attention(dtype, qkv, nullptr, y, B, T, t_out, n_head, hd, drop, false, "gpt_attention_dropout", stream);
}

extern "C" int gpt_attention_dropout_bwd(int dtype, const void* qkv, const void* dy, void* dqkv, int B, int T, int n_head, int hd,
                                         const gpt_dropout_t* drop, void* stream) {
  return attention(dtype, qkv, dy, dqkv, B, T, T, n_head, hd, drop, true, "gpt_attention_dropout_bwd", stream);
}
