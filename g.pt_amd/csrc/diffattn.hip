// Differential attention, forward:  out = (softmax(c Q1 K1^T) - lam softmax(c Q2 K2^T)) V   per (sample, head).
// Stands beside attention.hip (one softmax map, T <= 32).
//
// One sweep over the keys with the running maximum and sum of both softmaxes.  The products are computed transposed,
//   S^T = K Q^T,   O^T = V^T P^T,
// so that a lane holds one query's scores (reductions over keys stay in its registers but for two exchanges) and the exponentiated
// accumulator of S^T is the operand of the second product as it stands.
#include "diffattn.h"

namespace diffattn {
namespace {

// One wave: 16 queries, both maps; operands straight from global memory.
template <typename T, int HD>
__global__ __launch_bounds__(256) void fwd_kernel(Args a) {
  constexpr int KC = HD / 32, CT = 2 * HD / 16;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int tiles = (a.Tq + 15) / 16, groups = (tiles + 3) / 4;
  int id = blockIdx.x;
  const int tile = (id % groups) * 4 + (threadIdx.x >> 6);
  id /= groups;
  const int h = id % a.H;
  id /= a.H;
  const int b = id % a.B, split = id / a.B;
  if (tile >= tiles) return;
  const int len = valid_keys(a, b);
  const int k0 = split * a.split_keys, k1 = min(len, k0 + a.split_keys);
  const T* kb = (const T*)a.k + (int64_t)b * a.bsk + h * 2 * HD;
  const T* vb = (const T*)a.v + (int64_t)b * a.bsv + h * 2 * HD;
  const int qi = tile * 16 + col;
  const bool qok = qi < a.Tq;
  const T* qr = (const T*)a.q + (int64_t)b * a.bsq + (int64_t)(qok ? qi : 0) * a.ldq + h * 2 * HD;
  Frag<T> qf[2][KC];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int c = 0; c < KC; ++c) qf[m][c] = frag_row(qr + m * HD + c * 32 + g * 8, qok);
  f32x4 o[2][CT];
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < CT; ++t) o[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int kt = k0; kt < k1; kt += 32) {
    Frag<T> pf[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      f32x4 s[2];
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int key = kt + 16 * u + col;
        const T* kr = kb + (int64_t)(key < k1 ? key : k0) * a.ldk + m * HD + g * 8;
#pragma unroll
        for (int c = 0; c < KC; ++c) s[u] = mma16(frag_row(kr + c * 32, key < k1), qf[m][c], s[u]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (kt + 16 * u + 4 * g + r >= k1) s[u][r] = -INFINITY;
          mx = fmaxf(mx, s[u][r]);
        }
      }
      mx = fmaxf(top[m], col_max(mx));                    // finite, or NaN: the tile has a valid key
      const float ref = mx * a.c2, alpha = exp2_fast(top[m] * a.c2 - ref);
      top[m] = mx;
      float part = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[u][r] = exp2_fast(s[u][r] * a.c2 - ref);
          part += s[u][r];
        }
      sum[m] = sum[m] * alpha + part;
#pragma unroll
      for (int t = 0; t < CT; ++t) o[m][t] *= alpha;
      frag_from(pf[m], s[0], s[1]);
    }
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      const Frag<T> vf = frag_column<T>(vb + (int64_t)kt * a.ldv + t * 16 + col, a.ldv, g, k1 - kt);
#pragma unroll
      for (int m = 0; m < 2; ++m) o[m][t] = mma16(vf, pf[m], o[m][t]);
    }
  }
#pragma unroll
  for (int m = 0; m < 2; ++m) sum[m] = col_sum(sum[m]);
  if (!qok) return;
  if (a.splits > 1) {
    float* p = a.part + (((int64_t)split * a.B * a.H + (int64_t)b * a.H + h) * a.Tq + qi) * (4 * HD + 4);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int t = 0; t < CT; ++t) store4(p + m * 2 * HD + t * 16 + 4 * g, o[m][t]);
    if (g == 0) store4(p + 4 * HD, f32x4{top[0], sum[0], top[1], sum[1]});
    return;
  }
  const float lam = a.lam[h];
  const float inv0 = sum[0] > 0.f ? 1.f / sum[0] : sum[0], inv1 = sum[1] > 0.f ? 1.f / sum[1] : sum[1];   // no key: 0; NaN stays
  T* orow = (T*)a.out + (int64_t)b * a.bso + (int64_t)qi * a.ldo + h * 2 * HD;
  T* o2 = a.out2 ? (T*)a.out2 + ((int64_t)b * a.Tq + qi) * (a.H * 2 * HD) + h * 2 * HD : nullptr;
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    const f32x4 second = o[1][t] * inv1;
    store4(orow + t * 16 + 4 * g, o[0][t] * inv0 - second * lam);
    if (o2) store4(o2 + t * 16 + 4 * g, second);
  }
  if (a.lse && g == 0) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
      a.lse[(((int64_t)m * a.B + b) * a.H + h) * a.Tq + qi] = sum[m] == 0.f ? INFINITY : top[m] * a.c2 + __builtin_amdgcn_logf(sum[m]);
  }
}

// joins the splits of one (sample, head, query): one wave; lane owns 4 columns of 4 hd
template <typename T, int HD>
__global__ __launch_bounds__(256) void combine_kernel(Args a) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), rows = (int64_t)a.B * a.H * a.Tq;
  if (row >= rows) return;
  const int lane = threadIdx.x & 63;
  constexpr int W = 4 * HD + 4;
  const float* p = a.part + row * W;
  const int64_t step = rows * W;
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    const f32x4 t = *reinterpret_cast<const f32x4*>(p + s * step + 4 * HD);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      if (t[2 * m + 1] == 0.f) continue;                   // a split without a valid key
      const float mx = fmaxf(top[m], t[2 * m]);
      sum[m] = sum[m] * exp2_fast((top[m] - mx) * a.c2) + t[2 * m + 1] * exp2_fast((t[2 * m] - mx) * a.c2);
      top[m] = mx;
    }
  }
  const int qi = (int)(row % a.Tq), h = (int)(row / a.Tq % a.H), b = (int)(row / a.Tq / a.H);
  if (lane * 4 < 2 * HD) {
    f32x4 o[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
    for (int s = 0; s < a.splits; ++s) {
      const f32x4 t = *reinterpret_cast<const f32x4*>(p + s * step + 4 * HD);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (t[2 * m + 1] == 0.f) continue;
        o[m] += *reinterpret_cast<const f32x4*>(p + s * step + m * 2 * HD + lane * 4) * exp2_fast((t[2 * m] - top[m]) * a.c2);
      }
    }
    const f32x4 first = sum[0] == 0.f ? o[0] : o[0] / sum[0], second = sum[1] == 0.f ? o[1] : o[1] / sum[1];
    store4((T*)a.out + (int64_t)b * a.bso + (int64_t)qi * a.ldo + h * 2 * HD + lane * 4, first - second * a.lam[h]);
    if (a.out2) store4((T*)a.out2 + ((int64_t)b * a.Tq + qi) * (a.H * 2 * HD) + h * 2 * HD + lane * 4, second);
  }
  if (a.lse && lane < 2) {
    const float s = lane ? sum[1] : sum[0], t = lane ? top[1] : top[0];
    a.lse[(((int64_t)lane * a.B + b) * a.H + h) * a.Tq + qi] = s == 0.f ? INFINITY : t * a.c2 + __builtin_amdgcn_logf(s);
  }
}

// spans of keys per (sample, head, query tile): as many as fill the chip's 256 CUs with two workgroups each, none shorter than 256 keys
int splits_for(int B, int Tq, int Tk, int H) {
  const int64_t wgs = (int64_t)B * H * ((Tq + 63) / 64);
  if (wgs >= 256) return 1;
  const int64_t want = (512 + wgs - 1) / wgs, most = (Tk + 255) / 256;
  return (int)(want < most ? want : most);
}

template <typename T, int HD>
int launch(const Args& a, hipStream_t s) {
  const int64_t groups = ((int64_t)(a.Tq + 15) / 16 + 3) / 4, grid = groups * a.H * a.B * a.splits;
  GPT_REQUIRE(grid < (1ll << 24), "gpt_diff_attention: too many workgroups (%lld)", (long long)grid);
  hipLaunchKernelGGL((fwd_kernel<T, HD>), dim3((unsigned)grid), dim3(256), 0, s, a);
  if (int st = gpt_launch_status("gpt_diff_attention")) return st;
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.B * a.H * a.Tq;
    hipLaunchKernelGGL((combine_kernel<T, HD>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
    return gpt_launch_status("gpt_diff_attention");
  }
  return 0;
}

}  // namespace

// the checks both directions share; fills what the descriptor says
int make_args(const gpt_diff_attention_t* p, const char* who, Args* a) {
  GPT_REQUIRE(p, "%s: null descriptor", who);
  GPT_REQUIRE(p->dtype == GPT_F32 || p->dtype == GPT_BF16, "%s: bad dtype %d", who, p->dtype);
  GPT_REQUIRE(p->B > 0 && p->Tq > 0 && p->Tk > 0 && p->n_head > 0, "%s: need B, Tq, Tk, n_head > 0 (%d, %d, %d, %d)", who, p->B, p->Tq, p->Tk,
              p->n_head);
  GPT_REQUIRE(p->hd == 32 || p->hd == 64 || p->hd == 96 || p->hd == 128, "%s: unsupported head dim %d (32, 64, 96, 128)", who, p->hd);
  GPT_REQUIRE(p->n_head <= 4096 && (int64_t)p->B * p->n_head <= (1 << 24) && p->Tq <= (1 << 24) && p->Tk <= (1 << 24),
              "%s: size out of range (B=%d heads=%d Tq=%d Tk=%d)", who, p->B, p->n_head, p->Tq, p->Tk);
  GPT_REQUIRE(p->q && p->k && p->v && p->lam && p->out, "%s: null operand", who);
  GPT_REQUIRE(p->scale > 0.f && p->scale < INFINITY, "%s: scale must be positive and finite (%g)", who, p->scale);
  const int64_t w = (int64_t)p->n_head * 2 * p->hd, es = p->dtype == GPT_BF16 ? 2 : 4;
  auto rows_ok = [&](const void* ptr, int64_t ld, int64_t bs, int T) {
    return (uintptr_t)ptr % 16 == 0 && (ld * es) % 16 == 0 && (bs * es) % 16 == 0 && bs >= 0 && (T == 1 || ld >= w) && ld < (1 << 25);
  };
  GPT_REQUIRE(rows_ok(p->q, p->ldq, p->bsq, p->Tq) && rows_ok(p->k, p->ldk, p->bsk, p->Tk) && rows_ok(p->v, p->ldv, p->bsv, p->Tk),
              "%s: q, k, v rows must be 16-byte aligned, a row's width or more apart (ld %lld %lld %lld)", who, (long long)p->ldq,
              (long long)p->ldk, (long long)p->ldv);
  GPT_REQUIRE(rows_ok(p->out, p->ldo, p->bso, p->Tq) && (p->B == 1 || p->bso >= w), "%s: bad strides of out (%lld, %lld)", who,
              (long long)p->ldo, (long long)p->bso);
  GPT_REQUIRE((uintptr_t)p->out2 % 16 == 0 && (uintptr_t)p->lse % 4 == 0 && (uintptr_t)p->lam % 4 == 0 && (uintptr_t)p->lengths % 4 == 0,
              "%s: misaligned operand", who);
  *a = Args{};
  a->q = p->q; a->k = p->k; a->v = p->v;
  a->ldq = p->ldq; a->bsq = p->bsq; a->ldk = p->ldk; a->bsk = p->bsk; a->ldv = p->ldv; a->bsv = p->bsv;
  a->lam = p->lam; a->lengths = p->lengths;
  a->out = p->out; a->ldo = p->ldo; a->bso = p->bso; a->lse = p->lse; a->out2 = p->out2;
  a->B = p->B; a->Tq = p->Tq; a->Tk = p->Tk; a->H = p->n_head;
  a->scale = p->scale; a->c2 = p->scale * LOG2E;
  a->splits = 1; a->split_keys = p->Tk;
  return 0;
}

}  // namespace diffattn

using namespace diffattn;

static int64_t fwd_workspace(int B, int Tq, int Tk, int n_head, int hd) {
  if (Tq <= SHORT && Tk <= SHORT) return 0;
  const int n = splits_for(B, Tq, Tk, n_head);
  return n > 1 ? (int64_t)n * B * n_head * Tq * (4 * hd + 4) * (int64_t)sizeof(float) : 0;
}

extern "C" int gpt_diff_attention_workspace(int dtype, int B, int Tq, int Tk, int n_head, int hd, int64_t* host_bytes) {
  GPT_REQUIRE(host_bytes && (dtype == GPT_F32 || dtype == GPT_BF16) && B > 0 && Tq > 0 && Tk > 0 && n_head > 0 && hd > 0,
              "gpt_diff_attention_workspace: bad arguments");
  *host_bytes = fwd_workspace(B, Tq, Tk, n_head, hd);
  return 0;
}

extern "C" int gpt_diff_attention(const gpt_diff_attention_t* p, void* stream) {
  const char* who = "gpt_diff_attention";
  Args a;
  if (int st = make_args(p, who, &a)) return st;
  if (p->Tq <= SHORT && p->Tk <= SHORT) return short_attention(a, p->dtype, p->hd, false, (hipStream_t)stream);
  const int64_t need = fwd_workspace(p->B, p->Tq, p->Tk, p->n_head, p->hd);
  if (need > 0) {
    GPT_REQUIRE(p->ws && (uintptr_t)p->ws % 16 == 0 && p->ws_bytes >= need, "%s: needs %lld bytes of scratch", who, (long long)need);
    const int n = splits_for(p->B, p->Tq, p->Tk, p->n_head);
    a.part = (float*)p->ws;
    a.splits = n;
    a.split_keys = ((p->Tk + n - 1) / n + 31) / 32 * 32;
  }
  hipStream_t s = (hipStream_t)stream;
#define GO(T)                           \
  switch (p->hd) {                      \
    case 32: return launch<T, 32>(a, s);  \
    case 64: return launch<T, 64>(a, s);  \
    case 96: return launch<T, 96>(a, s);  \
    default: return launch<T, 128>(a, s); \
  }
  if (p->dtype == GPT_BF16) GO(bf16_t)
  GO(float)
#undef GO
}
