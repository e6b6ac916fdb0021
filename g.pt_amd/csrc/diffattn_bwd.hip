// Differential attention, backward.  With dP = dO V^T, D_i = rowsum(P_i dP):
//   dS_1 = P_1 (dP - D_1),  dS_2 = -lam P_2 (dP - D_2)
//   dQ_i = c dS_i K_i,  dK_i = c dS_i^T Q_i,  dV = (P_1 - lam P_2)^T dO,  dlam = -sum P_2 dP
// The maps are recomputed from the kept log-sum-exps.  D_i = dO . O_i comes from the kept outputs.  Two sweeps, over key tiles for dQ
// and over query tiles for dK / dV, so that every sum is taken by one wave in a fixed order; dlam is summed from the fp32 P_2 and dP
// of the second sweep (from the rounded outputs it would carry their rounding error).
#include "diffattn.h"

namespace diffattn {
int make_args(const gpt_diff_attention_t* p, const char* who, Args* a);

namespace {

// D_1, D_2 per (sample, query, head): one wave each; O_1 = out + lam O_2
template <typename T, int HD>
__global__ __launch_bounds__(256) void delta_kernel(Args a, float* delta) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), rows = (int64_t)a.B * a.Tq * a.H;
  if (row >= rows) return;
  const int lane = threadIdx.x & 63;
  const int h = (int)(row % a.H), qi = (int)(row / a.H % a.Tq), b = (int)(row / a.H / a.Tq);
  const T* g = (const T*)a.dout + (int64_t)b * a.bsdo + (int64_t)qi * a.lddo + h * 2 * HD;
  const T* o = (const T*)a.out + (int64_t)b * a.bso + (int64_t)qi * a.ldo + h * 2 * HD;
  const T* o2 = (const T*)a.out2 + ((int64_t)b * a.Tq + qi) * (a.H * 2 * HD) + h * 2 * HD;
  float d = 0.f, d2 = 0.f;
  for (int c = lane; c < 2 * HD; c += 64) {
    const float x = elem<T>::load(g + c);
    d += x * elem<T>::load(o + c);
    d2 += x * elem<T>::load(o2 + c);
  }
  d = wave_sum(d);
  d2 = wave_sum(d2);
  if (lane == 0) {
    const int64_t i = ((int64_t)b * a.H + h) * a.Tq + qi;
    delta[i] = d + a.lam[h] * d2;
    delta[(int64_t)a.B * a.H * a.Tq + i] = d2;
  }
}

// dQ: one wave, 16 queries, both maps
template <typename T, int HD>
__global__ __launch_bounds__(256) void dq_kernel(Args a) {
  constexpr int KC = HD / 32, CT = HD / 16;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int tiles = (a.Tq + 15) / 16, groups = (tiles + 3) / 4;
  int id = blockIdx.x;
  const int tile = (id % groups) * 4 + (threadIdx.x >> 6);
  id /= groups;
  const int h = id % a.H, b = id / a.H;
  if (tile >= tiles) return;
  const int len = valid_keys(a, b), qi = tile * 16 + col;
  const bool qok = qi < a.Tq;
  const T* kb = (const T*)a.k + (int64_t)b * a.bsk + h * 2 * HD;
  const T* vb = (const T*)a.v + (int64_t)b * a.bsv + h * 2 * HD;
  const T* qr = (const T*)a.q + (int64_t)b * a.bsq + (int64_t)(qok ? qi : 0) * a.ldq + h * 2 * HD;
  const T* gr = (const T*)a.dout + (int64_t)b * a.bsdo + (int64_t)(qok ? qi : 0) * a.lddo + h * 2 * HD;
  Frag<T> qf[2][KC], gf[2 * KC];
#pragma unroll
  for (int c = 0; c < 2 * KC; ++c) {
    qf[c / KC][c % KC] = frag_row(qr + c * 32 + g * 8, qok);
    gf[c] = frag_row(gr + c * 32 + g * 8, qok);
  }
  const int64_t n = (int64_t)a.B * a.H * a.Tq, si = ((int64_t)b * a.H + h) * a.Tq + (qok ? qi : 0);
  const float lse[2] = {a.lse[si], a.lse[n + si]}, dl[2] = {a.delta[si], a.delta[n + si]}, sign[2] = {1.f, -a.lam[h]};
  f32x4 acc[2][CT];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int kt = 0; kt < len; kt += 32) {
    f32x4 dp[2], ds[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int key = kt + 16 * u + col;
      const bool ok = key < len;
      const T* kr = kb + (int64_t)(ok ? key : 0) * a.ldk + g * 8;
      const T* vr = vb + (int64_t)(ok ? key : 0) * a.ldv + g * 8;
      dp[u] = ds[0][u] = ds[1][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2 * KC; ++c) {
        dp[u] = mma16(frag_row(vr + c * 32, ok), gf[c], dp[u]);
        ds[c / KC][u] = mma16(frag_row(kr + c * 32, ok), qf[c / KC][c % KC], ds[c / KC][u]);
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool in = kt + 16 * u + 4 * g + r < len;
          ds[m][u][r] = in ? sign[m] * exp2_fast(ds[m][u][r] * a.c2 - lse[m]) * (dp[u][r] - dl[m]) : 0.f;
        }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      Frag<T> df;
      frag_from(df, ds[m][0], ds[m][1]);
#pragma unroll
      for (int t = 0; t < CT; ++t)
        acc[m][t] = mma16(frag_column<T>(kb + (int64_t)kt * a.ldk + m * HD + t * 16 + col, a.ldk, g, len - kt), df, acc[m][t]);
    }
  }
  if (!qok) return;
  T* dq = (T*)a.dq + (int64_t)b * a.bsdq + (int64_t)qi * a.lddq + h * 2 * HD;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < CT; ++t) store4(dq + m * HD + t * 16 + 4 * g, acc[m][t] * a.scale);
}

// dK, dV and the tile's share of sum P_2 dP: one wave, 16 keys, both maps
template <typename T, int HD>
__global__ __launch_bounds__(256) void dkv_kernel(Args a) {
  constexpr int KC = HD / 32, CT = HD / 16;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int tiles = (a.Tk + 15) / 16, groups = (tiles + 3) / 4;
  int id = blockIdx.x;
  const int tile = (id % groups) * 4 + (threadIdx.x >> 6);
  id /= groups;
  const int h = id % a.H, b = id / a.H;
  if (tile >= tiles) return;
  const int len = valid_keys(a, b), key = tile * 16 + col;
  const bool ok = key < len;
  const T* kr = (const T*)a.k + (int64_t)b * a.bsk + (int64_t)(ok ? key : 0) * a.ldk + h * 2 * HD;
  const T* vr = (const T*)a.v + (int64_t)b * a.bsv + (int64_t)(ok ? key : 0) * a.ldv + h * 2 * HD;
  const T* qb = (const T*)a.q + (int64_t)b * a.bsq + h * 2 * HD;
  const T* gb = (const T*)a.dout + (int64_t)b * a.bsdo + h * 2 * HD;
  Frag<T> kf[2][KC], vf[2 * KC];
#pragma unroll
  for (int c = 0; c < 2 * KC; ++c) {
    kf[c / KC][c % KC] = frag_row(kr + c * 32 + g * 8, ok);
    vf[c] = frag_row(vr + c * 32 + g * 8, ok);
  }
  const int64_t n = (int64_t)a.B * a.H * a.Tq, s0 = ((int64_t)b * a.H + h) * a.Tq;
  const float lam = a.lam[h], sign[2] = {1.f, -lam};
  f32x4 dv[2 * CT], dk[2][CT];
  float dlam = 0.f;
#pragma unroll
  for (int t = 0; t < CT; ++t) dv[t] = dv[CT + t] = dk[0][t] = dk[1][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int last = tile * 16 < len ? a.Tq : 0;             // a tile without a valid key: zeros
  for (int qt = 0; qt < last; qt += 32) {
    f32x4 dp[2], p[2], ds[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int qi = qt + 16 * u + col;
      const bool in = qi < a.Tq;
      const T* qr = qb + (int64_t)(in ? qi : 0) * a.ldq + g * 8;
      const T* gr = gb + (int64_t)(in ? qi : 0) * a.lddo + g * 8;
      dp[u] = ds[0][u] = ds[1][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2 * KC; ++c) {
        dp[u] = mma16(frag_row(gr + c * 32, in), vf[c], dp[u]);
        ds[c / KC][u] = mma16(frag_row(qr + c * 32, in), kf[c / KC][c % KC], ds[c / KC][u]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = qt + 16 * u + 4 * g + r;
        const bool valid = ok && row < a.Tq;
        const int64_t i = s0 + (row < a.Tq ? row : 0);
        float pm[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          pm[m] = valid ? exp2_fast(ds[m][u][r] * a.c2 - a.lse[m * n + i]) : 0.f;
          ds[m][u][r] = valid ? sign[m] * pm[m] * (dp[u][r] - a.delta[m * n + i]) : 0.f;
        }
        p[u][r] = pm[0] - lam * pm[1];
        dlam += valid ? pm[1] * dp[u][r] : 0.f;
      }
    }
    Frag<T> pf, df[2];
    frag_from(pf, p[0], p[1]);
    frag_from(df[0], ds[0][0], ds[0][1]);
    frag_from(df[1], ds[1][0], ds[1][1]);
#pragma unroll
    for (int t = 0; t < 2 * CT; ++t) {
      dv[t] = mma16(frag_column<T>(gb + (int64_t)qt * a.lddo + t * 16 + col, a.lddo, g, a.Tq - qt), pf, dv[t]);
      dk[t / CT][t % CT] = mma16(frag_column<T>(qb + (int64_t)qt * a.ldq + t * 16 + col, a.ldq, g, a.Tq - qt), df[t / CT], dk[t / CT][t % CT]);
    }
  }
  dlam = wave_sum(dlam);
  if (lane == 0) a.dlam_part[((int64_t)h * a.B + b) * tiles + tile] = dlam;
  if (key >= a.Tk) return;
  T* dkr = (T*)a.dk + (int64_t)b * a.bsdk + (int64_t)key * a.lddk + h * 2 * HD;
  T* dvr = (T*)a.dv + (int64_t)b * a.bsdv + (int64_t)key * a.lddv + h * 2 * HD;
#pragma unroll
  for (int t = 0; t < 2 * CT; ++t) {
    store4(dkr + t * 16 + 4 * g, dk[t / CT][t % CT] * a.scale);
    store4(dvr + t * 16 + 4 * g, dv[t]);
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

int64_t key_tiles(int Tk) { return (Tk + 15) / 16; }

template <typename T, int HD>
int launch(const Args& a, float* delta, float* dlam, hipStream_t s) {
  const char* who = "gpt_diff_attention_bwd";
  const int64_t rows = (int64_t)a.B * a.Tq * a.H, nd = (rows + 3) / 4;
  const int64_t nq = (((int64_t)a.Tq + 15) / 16 + 3) / 4 * a.H * a.B, nk = (key_tiles(a.Tk) + 3) / 4 * a.H * a.B;
  GPT_REQUIRE(nd < (1ll << 24) && nq < (1ll << 24) && nk < (1ll << 24), "%s: too many workgroups", who);
  hipLaunchKernelGGL((delta_kernel<T, HD>), dim3((unsigned)nd), dim3(256), 0, s, a, delta);
  if (int st = gpt_launch_status(who)) return st;
  hipLaunchKernelGGL((dkv_kernel<T, HD>), dim3((unsigned)nk), dim3(256), 0, s, a);
  if (int st = gpt_launch_status(who)) return st;
  hipLaunchKernelGGL((dq_kernel<T, HD>), dim3((unsigned)nq), dim3(256), 0, s, a);
  if (int st = gpt_launch_status(who)) return st;
  hipLaunchKernelGGL(dlam_kernel, dim3(a.H), dim3(256), 0, s, a.dlam_part, (int64_t)a.B * key_tiles(a.Tk), dlam);
  return gpt_launch_status(who);
}

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

}  // namespace
}  // namespace diffattn

using namespace diffattn;

static int64_t bwd_workspace(int B, int Tq, int Tk, int n_head) {
  if (Tq <= SHORT && Tk <= SHORT) return round16((int64_t)n_head * B * 4);
  return round16((int64_t)2 * B * n_head * Tq * 4) + round16((int64_t)n_head * B * key_tiles(Tk) * 4);
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
  float* delta = (float*)p->ws;
  a.delta = delta;
  a.dlam_part = (float*)((char*)p->ws + round16((int64_t)2 * f->B * f->n_head * f->Tq * 4));
#define GO(T)                                          \
  switch (f->hd) {                                     \
    case 32: return launch<T, 32>(a, delta, p->dlam, s);  \
    case 64: return launch<T, 64>(a, delta, p->dlam, s);  \
    case 96: return launch<T, 96>(a, delta, p->dlam, s);  \
    default: return launch<T, 128>(a, delta, p->dlam, s); \
  }
  if (f->dtype == GPT_BF16) GO(bf16_t)
  GO(float)
#undef GO
}
