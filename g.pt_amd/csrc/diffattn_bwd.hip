// Differential attention, backward (diffattn_short.hip takes Tq, Tk <= 32).  With dP = dO V^T, D_i = rowsum(P_i dP):
//   dS_1 = P_1 (dP - D_1),  dS_2 = -lam P_2 (dP - D_2)
//   dQ_i = c dS_i K_i,  dK_i = c dS_i^T Q_i,  dV = (P_1 - lam P_2)^T dO,  dlam = -sum P_2 dP
// The maps are recomputed from the kept log-sum-exps; D_i = dO . O_i comes from the kept outputs.  Two sweeps, over key tiles for dQ
// and over query tiles for dK / dV, so that every sum is taken by one wave in a fixed order; dlam is summed from the fp32 P_2 and dP
// of the second sweep (from the rounded outputs it would carry their rounding error).
// A wave holds 32 rows of its side for BOTH maps - operands and accumulators, up to 450 registers, one wave per SIMD - because dP
// serves both: a wave per map would compute it twice (a third more matrix work in dQ, a half in dK / dV).  The other side comes in
// tiles of 32 rows by LDS-DMA, shared by the workgroup's waves; every tile is used twice, by rows for the scores and transposed for
// the gradient products.
#include "diffattn.h"

namespace diffattn {
int make_args(const gpt_diff_attention_t* p, const char* who, Args* a);

namespace {

// per (sample, head, query) the two log-sum-exps and D_1 = dO . (out + lam out2), D_2 = dO . out2: 16 lanes each
template <typename T, int HD>
__global__ __launch_bounds__(256) void stats_kernel(Args a, f32x4* stats) {
  constexpr int CH = 2 * HD * sizeof(T) / 16, PER = 16 / sizeof(T);
  const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), rows = (int64_t)a.B * a.Tq * a.H;
  if (row >= rows) return;                                               // whole groups of 16 lanes
  const int lane = threadIdx.x & 15;
  const int h = (int)(row % a.H), qi = (int)(row / a.H % a.Tq), b = (int)(row / a.H / a.Tq);
  const T* g = (const T*)a.dout + (int64_t)b * a.bsdo + (int64_t)qi * a.lddo + h * 2 * HD;
  const T* o = (const T*)a.out + (int64_t)b * a.bso + (int64_t)qi * a.ldo + h * 2 * HD;
  const T* o2 = (const T*)a.out2 + row * (2 * HD);
  float d = 0.f, d2 = 0.f;
#pragma unroll
  for (int c = 0; c < (CH + 15) / 16; ++c) {
    const int ch = c * 16 + lane;
    if (ch >= CH) break;
    const u32x4 x = reinterpret_cast<const u32x4*>(g)[ch], y = reinterpret_cast<const u32x4*>(o)[ch], z = reinterpret_cast<const u32x4*>(o2)[ch];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      float xv, yv, zv;
      if constexpr (sizeof(T) == 2) {
        const int sh = (j & 1) ? 0 : 16;
        xv = __uint_as_float((x[j >> 1] << sh) & 0xffff0000u);
        yv = __uint_as_float((y[j >> 1] << sh) & 0xffff0000u);
        zv = __uint_as_float((z[j >> 1] << sh) & 0xffff0000u);
      } else {
        xv = __uint_as_float(x[j]); yv = __uint_as_float(y[j]); zv = __uint_as_float(z[j]);
      }
      d += xv * yv;
      d2 += xv * zv;
    }
  }
#pragma unroll
  for (int s = 1; s < 16; s <<= 1) {
    d += __shfl_xor(d, s, 64);
    d2 += __shfl_xor(d2, s, 64);
  }
  if (lane == 0) {
    const int64_t i = ((int64_t)b * a.H + h) * a.Tq + qi, n = (int64_t)a.B * a.H * a.Tq;
    stats[i] = f32x4{a.lse[i], a.lse[n + i], d + a.lam[h] * d2, d2};
  }
}

// stages of the tile ring: three where a workgroup has a CU's LDS to itself (the tile after next is in flight while one is used)
template <typename T, int NW>
constexpr int STAGES = sizeof(T) == 2 && NW == 4 ? 3 : 2;
// LDS-DMA instructions a wave issues per tile of 32 rows
template <typename T, int HD, int NW>
constexpr int DMA_OPS = 32 * Tile<T, HD>::CPR / (NW * 64);

// dQ: NW waves of 32 queries; K | V tiles of 32 keys
template <typename T, int HD, int NW>
__global__ __launch_bounds__(NW * 64) void dq_kernel(Args a) {
  using L = Tile<T, HD>;
  constexpr int NT = NW * 64, NS = STAGES<T, NW>, TILE = 32 * L::PITCH, CT = HD / 32, CC = 32 * L::ES / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];            // [NS][K | V]
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, hh = lane >> 5;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int blocks = (a.Tq + 32 * NW - 1) / (32 * NW);
  int pair, block;
  xcd_block(blockIdx.x, gridDim.x, blocks, &pair, &block);
  const int b = pair / a.H, h = pair - b * a.H, len = valid_keys(a, b);
  const T* kb = (const T*)a.k + (int64_t)b * a.bsk + h * 2 * HD;
  const T* vb = (const T*)a.v + (int64_t)b * a.bsv + h * 2 * HD;
  const int qi = (block * NW + wid) * 32 + r;
  const bool qok = qi < a.Tq;
  u32x4 qf[L::CPR / 2], gf[L::CPR / 2];
  {
    const u32x4* qr = reinterpret_cast<const u32x4*>((const T*)a.q + (int64_t)b * a.bsq + (int64_t)(qok ? qi : 0) * a.ldq + h * 2 * HD);
    const u32x4* gr = reinterpret_cast<const u32x4*>((const T*)a.dout + (int64_t)b * a.bsdo + (int64_t)(qok ? qi : 0) * a.lddo + h * 2 * HD);
#pragma unroll
    for (int s = 0; s < L::CPR / 2; ++s) {
      qf[s] = qr[2 * s + hh];
      gf[s] = gr[2 * s + hh];
    }
  }
  const f32x4 st = a.stats[(int64_t)pair * a.Tq + (qok ? qi : 0)];
  const float lam = a.lam[h];
  f32x16 acc[2][CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) acc[0][t] = acc[1][t] = zero16();
  const int rb = row_base<T, HD>(lane);
  const ColBase<T, HD> cb(lane);
  const int n = (len + 31) / 32;
  auto fetch = [&](int it) {
    char* dst = smem + (it % NS) * 2 * TILE;
    dma_tile<T, HD, 32, NT>(kb + (int64_t)it * 32 * a.ldk, a.ldk, len - it * 32, dst, tid, wid);
    dma_tile<T, HD, 32, NT>(vb + (int64_t)it * 32 * a.ldv, a.ldv, len - it * 32, dst + TILE, tid, wid);
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i)
    if (i < n) fetch(i);
  for (int it = 0; it < n; ++it) {
    if (NS == 3 && it + 1 < n) tile_barrier<2 * DMA_OPS<T, HD, NW>>();       // tile `it` is here, the next one may be in flight
    else tile_barrier<0>();
    if (it + NS - 1 < n) fetch(it + NS - 1);                                 // into the buffer that was read before the barrier
    const char *tk = smem + (it % NS) * 2 * TILE, *tv = tk + TILE;
    f32x16 s[2] = {zero16(), zero16()}, dp = zero16();
#pragma unroll
    for (int c = 0; c < L::CPR / 2; ++c) {
      const int m = c >= L::CM / 2;
      s[m] = mma_chunk<T>(*reinterpret_cast<const u32x4*>(tk + L::add(rb, 2 * c)), qf[c], s[m]);
      dp = mma_chunk<T>(*reinterpret_cast<const u32x4*>(tv + L::add(rb, 2 * c)), gf[c], dp);
    }
    Operand x[2];
    const bool whole = it * 32 + 32 <= len;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float p = exp2_fast(s[m][e] * a.c2 - st[m]), v = p * (dp[e] - st[2 + m]);
        s[m][e] = whole || it * 32 + row_of(e, hh) < len ? (m ? -lam * v : v) : 0.f;
      }
      operand_from<T>(x[m], s[m]);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int t = 0; t < CT; ++t) acc[m][t] = columns_product<T, HD>(tk, cb, 0, m * L::CM + t * CC, x[m], acc[m][t]);
  }
  if (!qok) return;
  T* dq = (T*)a.dq + (int64_t)b * a.bsdq + (int64_t)qi * a.lddq + h * 2 * HD + 4 * hh;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x16& c = acc[m][t];
        store4(dq + m * HD + t * 32 + 8 * g, f32x4{c[4 * g], c[4 * g + 1], c[4 * g + 2], c[4 * g + 3]} * a.scale);
      }
}

// dK and / or dV: NW waves of 32 keys; Q | dO | statistics tiles of 32 queries.  fp32 at hd 96 and 128 runs the two one after the other: the
// operands and accumulators of both do not fit a wave's 512 registers.
enum { WANT_DK = 1, WANT_DV = 2 };

template <typename T, int HD, int NW, int WANT>
__global__ __launch_bounds__(NW * 64) void dkv_kernel(Args a) {
  using L = Tile<T, HD>;
  constexpr bool DK = (WANT & WANT_DK) != 0, DV = (WANT & WANT_DV) != 0;
  constexpr int NT = NW * 64, NS = STAGES<T, NW>, TILE = 32 * L::PITCH, STAGE = 2 * TILE + 512, CT = HD / 32, CC = 32 * L::ES / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];            // [NS][Q | dO | stats]
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, hh = lane >> 5;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int blocks = (a.Tk + 32 * NW - 1) / (32 * NW);
  int pair, block;
  xcd_block(blockIdx.x, gridDim.x, blocks, &pair, &block);
  const int b = pair / a.H, h = pair - b * a.H, len = valid_keys(a, b);
  const T* qb = (const T*)a.q + (int64_t)b * a.bsq + h * 2 * HD;
  const T* gb = (const T*)a.dout + (int64_t)b * a.bsdo + h * 2 * HD;
  const f32x4* sb = a.stats + (int64_t)pair * a.Tq;
  const int key = (block * NW + wid) * 32 + r;
  const bool ok = key < len;
  u32x4 kf[L::CPR / 2], vf[DK ? L::CPR / 2 : 1];
  {
    const u32x4* kr = reinterpret_cast<const u32x4*>((const T*)a.k + (int64_t)b * a.bsk + (int64_t)(ok ? key : 0) * a.ldk + h * 2 * HD);
    const u32x4* vr = reinterpret_cast<const u32x4*>((const T*)a.v + (int64_t)b * a.bsv + (int64_t)(ok ? key : 0) * a.ldv + h * 2 * HD);
#pragma unroll
    for (int s = 0; s < L::CPR / 2; ++s) {
      kf[s] = kr[2 * s + hh];
      if constexpr (DK) vf[s] = vr[2 * s + hh];
    }
  }
  const float lam = a.lam[h];
  f32x16 dk[2][DK ? CT : 1], dv[DV ? 2 * CT : 1];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    if constexpr (DK) dk[0][t] = dk[1][t] = zero16();
    if constexpr (DV) dv[t] = dv[CT + t] = zero16();
  }
  double dlam = 0.0;
  const int rb = row_base<T, HD>(lane);
  const ColBase<T, HD> cb(lane);
  const int n = block * NW * 32 < len ? (a.Tq + 31) / 32 : 0;               // a block without a valid key: zeros
  auto fetch = [&](int it) {
    char* dst = smem + (it % NS) * STAGE;
    dma_tile<T, HD, 32, NT>(qb + (int64_t)it * 32 * a.ldq, a.ldq, a.Tq - it * 32, dst, tid, wid);
    dma_tile<T, HD, 32, NT>(gb + (int64_t)it * 32 * a.lddo, a.lddo, a.Tq - it * 32, dst + TILE, tid, wid);
    dma_bytes(sb + it * 32, (a.Tq - it * 32) * 16, dst + 2 * TILE, lane);    // every wave the same 512 bytes: one count for all
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i)
    if (i < n) fetch(i);
  for (int it = 0; it < n; ++it) {
    if (NS == 3 && it + 1 < n) tile_barrier<2 * DMA_OPS<T, HD, NW> + 1>();
    else tile_barrier<0>();
    if (it + NS - 1 < n) fetch(it + NS - 1);
    const char *tq = smem + (it % NS) * STAGE, *tg = tq + TILE;
    const f32x4* ts = reinterpret_cast<const f32x4*>(tg + TILE);
    f32x16 s[2] = {zero16(), zero16()}, dp = zero16();
#pragma unroll
    for (int c = 0; c < L::CPR / 2; ++c) {
      const int m = c >= L::CM / 2;
      s[m] = mma_chunk<T>(*reinterpret_cast<const u32x4*>(tq + L::add(rb, 2 * c)), kf[c], s[m]);
      if constexpr (DK) dp = mma_chunk<T>(*reinterpret_cast<const u32x4*>(tg + L::add(rb, 2 * c)), vf[c], dp);
    }
    // queries behind Tq arrive as zeros in Q, dO and the statistics: their dP, D and gradient products are 0
    f32x16 p;
    float part = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const f32x4 st = ts[row_of(e, hh)];
      const float p0 = exp2_fast(s[0][e] * a.c2 - st[0]), p1 = exp2_fast(s[1][e] * a.c2 - st[1]);
      if constexpr (DV) p[e] = p0 - lam * p1;
      if constexpr (DK) {
        part += p1 * dp[e];
        s[0][e] = p0 * (dp[e] - st[2]);
        s[1][e] = -lam * (p1 * (dp[e] - st[3]));
      }
    }
    dlam += part;
    Operand x;
    if constexpr (DV) {
      operand_from<T>(x, p);
#pragma unroll
      for (int t = 0; t < 2 * CT; ++t) dv[t] = columns_product<T, HD>(tg, cb, 0, t * CC, x, dv[t]);
    }
    if constexpr (DK) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        operand_from<T>(x, s[m]);
#pragma unroll
        for (int t = 0; t < CT; ++t) dk[m][t] = columns_product<T, HD>(tq, cb, 0, m * L::CM + t * CC, x, dk[m][t]);
      }
    }
  }
  if constexpr (DK) {
    float sum = ok ? (float)dlam : 0.f;
    sum = wave_sum(sum);
    if (lane == 0) a.dlam_part[((int64_t)h * a.B + b) * (blocks * NW) + block * NW + wid] = sum;
  }
  if (key >= a.Tk) return;
  // a masked key's lane has computed with another row's operands: it stores zeros
  auto put = [&](T* row, const f32x16& c, float f) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      store4(row + 8 * g, ok ? f32x4{c[4 * g], c[4 * g + 1], c[4 * g + 2], c[4 * g + 3]} * f : f32x4{0.f, 0.f, 0.f, 0.f});
  };
  if constexpr (DK) {
    T* row = (T*)a.dk + (int64_t)b * a.bsdk + (int64_t)key * a.lddk + h * 2 * HD + 4 * hh;
#pragma unroll
    for (int t = 0; t < 2 * CT; ++t) put(row + t * 32, dk[t / CT][t % CT], a.scale);
  }
  if constexpr (DV) {
    T* row = (T*)a.dv + (int64_t)b * a.bsdv + (int64_t)key * a.lddv + h * 2 * HD + 4 * hh;
#pragma unroll
    for (int t = 0; t < 2 * CT; ++t) put(row + t * 32, dv[t], 1.f);
  }
}

// dlam[h] = -(sum of the head's partial sums): one workgroup per head, each thread every 256th in index order, then a fixed tree
__global__ __launch_bounds__(256) void dlam_kernel(const float* __restrict__ part, int64_t n, float* __restrict__ dlam) {
  __shared__ float red[4];
  const float* p = part + (int64_t)blockIdx.x * n;
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 256) s += p[i];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) dlam[blockIdx.x] = -((red[0] + red[1]) + (red[2] + red[3]));
}

// partial sums of dlam per (head, sample): one per 32 keys of the workgroups' blocks
int64_t key_tiles(int Tk) { return ((int64_t)Tk + 127) / 128 * 4; }

// waves of 32 rows per workgroup: four share the tiles where that still gives every CU a workgroup
int waves_for(int64_t pairs, int T) { return T > 32 && pairs * ((T + 127) / 128) >= 192 ? 4 : 1; }

template <typename T, int HD, int NW>
int launch_dq(const Args& a, hipStream_t s) {
  const char* who = "gpt_diff_attention_bwd";
  static GptPerDevice once;
  const int64_t grid = ((int64_t)a.Tq + 32 * NW - 1) / (32 * NW) * a.H * a.B;
  GPT_REQUIRE(grid * NW * 64 < (1ll << 32) && grid < (1ll << 31), "%s: too many workgroups (%lld)", who, (long long)grid);
  if (int st = grant_lds(dq_kernel<T, HD, NW>, once, who)) return st;
  hipLaunchKernelGGL((dq_kernel<T, HD, NW>), dim3((unsigned)grid), dim3(NW * 64), (STAGES<T, NW> * 64 * Tile<T, HD>::PITCH), s, a);
  return gpt_launch_status(who);
}

template <typename T, int HD, int NW, int WANT>
int launch_dkv(const Args& a, hipStream_t s) {
  const char* who = "gpt_diff_attention_bwd";
  static GptPerDevice once;
  const int64_t grid = ((int64_t)a.Tk + 32 * NW - 1) / (32 * NW) * a.H * a.B;
  GPT_REQUIRE(grid * NW * 64 < (1ll << 32) && grid < (1ll << 31), "%s: too many workgroups (%lld)", who, (long long)grid);
  if (int st = grant_lds(dkv_kernel<T, HD, NW, WANT>, once, who)) return st;
  hipLaunchKernelGGL((dkv_kernel<T, HD, NW, WANT>), dim3((unsigned)grid), dim3(NW * 64), (STAGES<T, NW> * (64 * Tile<T, HD>::PITCH + 512)), s, a);
  return gpt_launch_status(who);
}

template <typename T, int HD, int NW>
int launch_dkv_all(const Args& a, hipStream_t s) {
  if constexpr (sizeof(T) == 4 && HD >= 96) {
    if (int st = launch_dkv<T, HD, NW, WANT_DK>(a, s)) return st;
    return launch_dkv<T, HD, NW, WANT_DV>(a, s);
  } else {
    return launch_dkv<T, HD, NW, WANT_DK | WANT_DV>(a, s);
  }
}

template <typename T, int HD>
int launch(const Args& a, f32x4* stats, float* dlam, hipStream_t s) {
  const char* who = "gpt_diff_attention_bwd";
  const int64_t rows = (int64_t)a.B * a.Tq * a.H, nd = (rows + 15) / 16, pairs = (int64_t)a.B * a.H;
  GPT_REQUIRE(nd < (1ll << 24), "%s: too many rows (%lld)", who, (long long)rows);
  hipLaunchKernelGGL((stats_kernel<T, HD>), dim3((unsigned)nd), dim3(256), 0, s, a, stats);
  if (int st = gpt_launch_status(who)) return st;
  const int nk = waves_for(pairs, a.Tk);
  if (int st = nk == 4 ? launch_dkv_all<T, HD, 4>(a, s) : launch_dkv_all<T, HD, 1>(a, s)) return st;
  if (int st = waves_for(pairs, a.Tq) == 4 ? launch_dq<T, HD, 4>(a, s) : launch_dq<T, HD, 1>(a, s)) return st;
  const int64_t tiles = ((int64_t)a.Tk + 32 * nk - 1) / (32 * nk) * nk;
  hipLaunchKernelGGL(dlam_kernel, dim3(a.H), dim3(256), 0, s, a.dlam_part, (int64_t)a.B * tiles, dlam);
  return gpt_launch_status(who);
}

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

}  // namespace
}  // namespace diffattn

using namespace diffattn;

static int64_t bwd_workspace(int B, int Tq, int Tk, int n_head) {
  if (Tq <= SHORT && Tk <= SHORT) return round16((int64_t)n_head * B * 4);
  return (int64_t)16 * B * n_head * Tq + round16((int64_t)n_head * B * key_tiles(Tk) * 4);
}

extern "C" int gpt_diff_attention_bwd_workspace(int dtype, int B, int Tq, int Tk, int n_head, int hd, int64_t* host_bytes) {
  GPT_REQUIRE(host_bytes && (dtype == GPT_F32 || dtype == GPT_BF16) && B > 0 && Tq > 0 && Tk > 0 && n_head > 0 && hd > 0,
              "gpt_diff_attention_bwd_workspace: bad arguments");
  *host_bytes = bwd_workspace(B, Tq, Tk, n_head);
  return 0;
}

extern "C" int gpt_diff_attention_bwd(const gpt_diff_attention_t* f, const gpt_diff_attention_bwd_t* p, void* stream) {
  const char* who = "gpt_diff_attention_bwd";
  Args a;
  if (int st = make_args(f, who, &a)) return st;
  GPT_REQUIRE(p && p->dout && p->dq && p->dk && p->dv && p->dlam, "%s: null operand", who);
  const bool is_short = f->Tq <= SHORT && f->Tk <= SHORT;
  GPT_REQUIRE(is_short || (f->lse && f->out2), "%s: needs the forward's lse and out2", who);
  const int64_t w = (int64_t)f->n_head * 2 * f->hd, es = f->dtype == GPT_BF16 ? 2 : 4;
  auto rows_ok = [&](const void* ptr, int64_t ld, int64_t bs, int T, bool written) {
    return (uintptr_t)ptr % 16 == 0 && (ld * es) % 16 == 0 && (bs * es) % 16 == 0 && bs >= 0 && (T == 1 || ld >= w) && ld < (1 << 25) &&
           (!written || f->B == 1 || bs >= w);
  };
  GPT_REQUIRE(rows_ok(p->dout, p->lddo, p->bsdo, f->Tq, false) && rows_ok(p->dq, p->lddq, p->bsdq, f->Tq, true) &&
                  rows_ok(p->dk, p->lddk, p->bsdk, f->Tk, true) && rows_ok(p->dv, p->lddv, p->bsdv, f->Tk, true),
              "%s: gradient rows must be 16-byte aligned, a row's width or more apart", who);
  const int64_t need = bwd_workspace(f->B, f->Tq, f->Tk, f->n_head);
  GPT_REQUIRE(p->ws && (uintptr_t)p->ws % 16 == 0 && p->ws_bytes >= need, "%s: needs %lld bytes of scratch", who, (long long)need);
  a.dout = p->dout; a.lddo = p->lddo; a.bsdo = p->bsdo;
  a.dq = p->dq; a.lddq = p->lddq; a.bsdq = p->bsdq;
  a.dk = p->dk; a.lddk = p->lddk; a.bsdk = p->bsdk;
  a.dv = p->dv; a.lddv = p->lddv; a.bsdv = p->bsdv;
  hipStream_t s = (hipStream_t)stream;
  if (is_short) {
    a.dlam_part = (float*)p->ws;
    if (int st = short_attention(a, f->dtype, f->hd, true, s)) return st;
    hipLaunchKernelGGL(dlam_kernel, dim3(a.H), dim3(256), 0, s, a.dlam_part, (int64_t)a.B, p->dlam);
    return gpt_launch_status(who);
  }
  f32x4* stats = (f32x4*)p->ws;
  a.stats = stats;
  a.dlam_part = (float*)((char*)p->ws + (int64_t)16 * f->B * f->n_head * f->Tq);
#define GO(T)                                          \
  switch (f->hd) {                                     \
    case 32: return launch<T, 32>(a, stats, p->dlam, s);  \
    case 64: return launch<T, 64>(a, stats, p->dlam, s);  \
    case 96: return launch<T, 96>(a, stats, p->dlam, s);  \
    default: return launch<T, 128>(a, stats, p->dlam, s); \
  }
  if (f->dtype == GPT_BF16) GO(bf16_t)
  GO(float)
#undef GO
}
