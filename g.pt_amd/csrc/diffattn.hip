// Differential attention, forward:  out = (softmax(c Q1 K1^T) - lam softmax(c Q2 K2^T)) V   per (sample, head).
// Stands beside attention.hip (one softmax map, T <= 32); diffattn_short.hip takes Tq, Tk <= 32.
//
// One sweep over the keys with the running maximum and sum of each softmax.  The products are computed transposed,
//   S^T = K Q^T,   O^T = V^T P^T,
// so that a lane holds one query's scores (reductions over keys stay in its registers but for one exchange) and the exponentiated
// accumulator of S^T is the operand of the second product as it stands.
// A wave takes 32 queries and ONE map: its accumulator is 32 x 2 hd (128 registers at hd 128) where both maps' would leave one wave
// per SIMD; the two waves of a query group join their halves through LDS at the end.  K | V tiles of 64 or 32 keys come by
// LDS-DMA, double-buffered, one barrier per tile, and serve all waves of the workgroup.
// bf16: P enters the second product as two operands, its rounding to bf16 and what that left (16 bits of mantissa), so that the output's
// own rounding is the only one to 8 bits.  One operand alone leaves the output 2.55e-3 rms off at 4096 keys where rounding the exact
// result leaves 1.66e-3 (the maps' difference cancels values, not their noise).  The second costs nothing where memory is the bound (one
// query group) and, where the matrix unit is, half of its work again: 2 x 4096 tokens, 8 heads, hd 128, 563 us (1.22 PFLOP/s of its 687
// GFLOP) instead of 407, 16 samples of up to 515 tokens, hd 64, with what is kept for the backward, 53 instead of 44.
// The accumulator is rescaled only when a row's maximum has grown by more than a factor of 2^8 over the reference its sums are held
// against: P stays below 2^8.
#include "diffattn.h"

namespace diffattn {
namespace {

#define PIN() __builtin_amdgcn_sched_barrier(0)

constexpr float SLACK = 8.f;     // log2 of the growth that is let pass
constexpr int MAX_SPLITS = 512;

// Keys per tile.  With one query group (Tq <= 32) the kernel streams K and V: tiles of 32 keys leave a CU room for two workgroups, one
// loading while the other computes.  1 query x 16384 keys, hd 128, 32 (sample, head): 100.7 us (5.3 TB/s), tiles of 64 keys 124.3.
template <typename T, int NW>
constexpr int KEYS = sizeof(T) == 2 && NW > 1 ? 64 : 32;

// column c of a row of Args::rest's plane (plane = the map whose output's rounding it is)
template <int HD>
__device__ __forceinline__ bf16_t* rest_row(const Args& a, int plane, int b, int qi, int c) {
  return a.rest ? a.rest + (((int64_t)plane * a.B + b) * a.Tq + qi) * (a.H * 2 * HD) + c : nullptr;
}

// 16 columns of a row from the two lanes that hold them (this one columns 4 hh .. of the first 8 in x, of the next 8 in y), and what the
// rounding leaves to `rest`.  bf16: the lanes exchange a half each, so that both store 16 bytes (16 samples of up to 515
// tokens, hd 64, forward with all that it keeps: 62 us by 8 bytes, 52 by 16)
template <bool KEPT>
__device__ __forceinline__ void store_columns(bf16_t* p, bf16_t* rest, const f32x4& x, const f32x4& y, int hh) {
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float u = i < 2 ? x[2 * i] : y[2 * i - 4], v = i < 2 ? x[2 * i + 1] : y[2 * i - 3];
    hi[i] = pack_bf16x2(u, v);
    lo[i] = pack_bf16x2(u - __uint_as_float(hi[i] << 16), v - __uint_as_float(hi[i] & 0xffff0000u));
  }
  auto store = [&](bf16_t* dst, const uint32_t (&w)[4]) {
    const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    *reinterpret_cast<u32x4*>(dst + 8 * hh) = u32x4{a[0], b[0], a[1], b[1]};
  };
  store(p, hi);
  if constexpr (KEPT) store(rest, lo);
}
template <bool>
__device__ __forceinline__ void store_columns(float* p, bf16_t*, const f32x4& x, const f32x4& y, int hh) {
  store4(p + 4 * hh, x);
  store4(p + 8 + 4 * hh, y);
}

template <typename T, int HD, int NW>
__global__ __launch_bounds__(NW * 128) void fwd_kernel(Args a) {
  using L = Tile<T, HD>;
  constexpr int NT = NW * 128, KT = KEYS<T, NW>, NU = KT / 32, TILE = KT * L::PITCH, CT = 2 * HD / 32;
  // From hd 64 on the order is written out (PIN): operands read from LDS three fragments ahead, the products of a tile's first 32 keys
  // beside the exponentials of the other 32.  2 x 4096 tokens, 8 heads: hd 128 617 -> 584 us, hd 96 490 -> 471, hd 64 370 -> 351; hd 32
  // 216 -> 218: left to the compiler
  constexpr bool STEPPED = sizeof(T) == 2 && NW > 1 && HD >= 64;
  constexpr int LEAD = 3, R = LEAD + 1;
  constexpr bool WHOLE = sizeof(T) == 2;                                  // P in two bf16 operands
  extern __shared__ __attribute__((aligned(16))) char smem[];            // [2][K | V]
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, hh = lane >> 5;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6), m = wid & 1, grp = wid >> 1;
  const int blocks = (a.Tq + 32 * NW - 1) / (32 * NW);
  int pair, rest;
  xcd_block(blockIdx.x, gridDim.x, blocks * a.splits, &pair, &rest);
  const int split = rest / blocks, block = rest - split * blocks, b = pair / a.H, h = pair - b * a.H;
  const int k0 = split * a.split_keys, k1 = min(valid_keys(a, b), k0 + a.split_keys);
  const T* kb = (const T*)a.k + (int64_t)b * a.bsk + h * 2 * HD;
  const T* vb = (const T*)a.v + (int64_t)b * a.bsv + h * 2 * HD;
  const int qi = block * 32 * NW + grp * 32 + r;
  const bool qok = qi < a.Tq;
  u32x4 qf[L::CM / 2];
  {
    const T* qr = (const T*)a.q + (int64_t)b * a.bsq + (int64_t)(qok ? qi : 0) * a.ldq + h * 2 * HD;
#pragma unroll
    for (int s = 0; s < L::CM / 2; ++s) {
      qf[s] = reinterpret_cast<const u32x4*>(qr)[m * L::CM + 2 * s + hh];
      if (!qok) qf[s] = u32x4{0u, 0u, 0u, 0u};
    }
  }
  f32x16 o[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) o[t] = zero16();
  float top = -INFINITY, sum = 0.f;                                       // raw scores; of exp2(c2 (s - top))
  const int rb = row_base<T, HD>(lane);
  const ColBase<T, HD> cb(lane);
  const int n = k1 > k0 ? (k1 - k0 + KT - 1) / KT : 0;
  auto fetch = [&](int it) {
    const int key = k0 + it * KT;
    char* dst = smem + (it & 1) * 2 * TILE;
    dma_tile<T, HD, KT, NT>(kb + (int64_t)key * a.ldk, a.ldk, k1 - key, dst, tid, wid);
    dma_tile<T, HD, KT, NT>(vb + (int64_t)key * a.ldv, a.ldv, k1 - key, dst + TILE, tid, wid);
  };
  if (n > 0) fetch(0);
  for (int it = 0; it < n; ++it) {
    tile_barrier<0>();                                                     // tile `it` is here, the other buffer has been read
    if (it + 1 < n) fetch(it + 1);
    if (block * 32 * NW + grp * 32 >= a.Tq) continue;                       // a wave without a query only loads
    const char *tk = smem + (it & 1) * 2 * TILE, *tv = tk + TILE;
    f32x16 s[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) s[u] = zero16();
    if constexpr (STEPPED) {
      int rk = rb + (it & 1) * 2 * TILE;                                     // opaque: the variants of it are formed as they are used
      asm volatile("" : "+v"(rk));
      constexpr int N = 2 * (L::CM / 2);
      u32x4 ring[R];
      auto rows = [&](int i) { return *reinterpret_cast<const u32x4*>(smem + (i & 1) * 32 * L::PITCH + L::add(rk, m * L::CM + (i & ~1))); };
#pragma unroll
      for (int i = 0; i < LEAD; ++i) ring[i] = rows(i);
      PIN();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i + LEAD < N) ring[(i + LEAD) % R] = rows(i + LEAD);
        s[i & 1] = mma_chunk<T>(ring[i % R], qf[i / 2], s[i & 1]);
        PIN();
      }
    } else
#pragma unroll
    for (int c = 0; c < L::CM / 2; ++c)
#pragma unroll
      for (int u = 0; u < NU; ++u)
        s[u] = mma_chunk<T>(*reinterpret_cast<const u32x4*>(tk + u * 32 * L::PITCH + L::add(rb, m * L::CM + 2 * c)), qf[c], s[u]);
    if (k0 + (it + 1) * KT > k1) {
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (k0 + it * KT + u * 32 + row_of(e, hh) >= k1) s[u][e] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[u][e]);
    mx = col_max(mx);
    if (__any((mx - top) * a.c2 > SLACK)) {
      const float now = fmaxf(top, mx), alpha = now == -INFINITY ? 1.f : exp2_fast((top - now) * a.c2);
      top = now;
      sum *= alpha;
#pragma unroll
      for (int t = 0; t < CT; ++t) o[t] *= alpha;
    }
    const float ref = top == -INFINITY ? 0.f : top * a.c2;                   // nothing but -inf so far: exp2(-inf) = 0
    float part = 0.f;                                                       // the tile's sum first: chains of 32 and of n additions, not 32 n
    Operand p[NU], low[WHOLE ? NU : 1];
    if constexpr (STEPPED) {
      int lo = cb.lo + (it & 1) * 2 * TILE + TILE, hi = cb.hi + (it & 1) * 2 * TILE + TILE;
      asm volatile("" : "+v"(lo), "+v"(hi));
      bf16x8 ring[R];
      auto cols = [&](int u, int i) { return columns_frag<HD>(smem + (2 * u + (i & 1)) * 16 * L::PITCH, lo, hi, 4 * (i >> 1)); };
      auto weigh = [&](int u, int e) {
        s[u][e] = exp2_fast(s[u][e] * a.c2 - ref);
        part += s[u][e];
      };
#pragma unroll
      for (int i = 0; i < LEAD; ++i) ring[i] = cols(0, i);
#pragma unroll
      for (int e = 0; e < 16; ++e) weigh(0, e);
      operand_from<T>(p[0], s[0]);
      operand_rest(low[0], s[0], p[0]);
      PIN();
      constexpr int N = 2 * CT;
#pragma unroll
      for (int e = 0; e < 16; ++e) {                                         // the first half's products beside the second half's weights
#pragma unroll
        for (int i = e * N / 16; i < (e + 1) * N / 16; ++i) {
          ring[(i + LEAD) % R] = i + LEAD < N ? cols(0, i + LEAD) : cols(1, i + LEAD - N);
          o[i >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[i % R], p[0].p[i & 1], o[i >> 1], 0, 0, 0);
          o[i >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[i % R], low[0].p[i & 1], o[i >> 1], 0, 0, 0);
        }
        weigh(1, e);
        if (e & 1) PIN();
      }
      operand_from<T>(p[1], s[1]);
      operand_rest(low[1], s[1], p[1]);
      sum += part;
#pragma unroll
      for (int i = N; i < 2 * N; ++i) {
        if (i + LEAD < 2 * N) ring[(i + LEAD) % R] = cols(1, i + LEAD - N);
        o[(i - N) >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[i % R], p[1].p[i & 1], o[(i - N) >> 1], 0, 0, 0);
        o[(i - N) >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[i % R], low[1].p[i & 1], o[(i - N) >> 1], 0, 0, 0);
        PIN();
      }
      continue;
    }
#pragma unroll
    for (int u = 0; u < NU; ++u) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[u][e] = exp2_fast(s[u][e] * a.c2 - ref);
        part += s[u][e];
      }
      operand_from<T>(p[u], s[u]);
      if constexpr (WHOLE) operand_rest(low[u], s[u], p[u]);
    }
    sum += part;
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        if constexpr (WHOLE) o[t] = columns_product<T, HD>(tv, cb, u * 32, t * (32 * L::ES / 16), p[u], o[t], low[u]);
        else o[t] = columns_product<T, HD>(tv, cb, u * 32, t * (32 * L::ES / 16), p[u], o[t]);
      }
  }
  sum = col_sum(sum);
  if (a.splits > 1) {
    if (!qok) return;
    float* p = a.part + (((int64_t)split * a.B * a.H + pair) * a.Tq + qi) * (4 * HD + 4);
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        store4(p + m * 2 * HD + t * 32 + 8 * g + 4 * hh, f32x4{o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3]});
    if (hh == 0) {
      p[4 * HD + 2 * m] = top;
      p[4 * HD + 2 * m + 1] = sum;
    }
    return;
  }
  // the second map's wave hands its normalised half over: [t][g] planes of 64 x 16 bytes, the same lane reads what a lane wrote
  const float inv = n > 0 ? 1.f / sum : 0.f;                                 // no key: 0; nothing but scores of -inf: 0 / 0
  f32x4* ex = reinterpret_cast<f32x4*>(smem) + grp * (CT * 4 * 64) + lane;
  tile_barrier<0>();
  if (m == 1) {
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g) ex[(t * 4 + g) * 64] = f32x4{o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3]} * inv;
  }
  tile_barrier<0>();
  if (!qok) return;
  if (a.lse && hh == 0) a.lse[((int64_t)m * a.B * a.H + pair) * a.Tq + qi] = n > 0 ? top * a.c2 + __builtin_amdgcn_logf(sum) : INFINITY;
  auto finish = [&](auto kept) {                                               // the rows of map m, with what their rounding leaves or without
    const bool second = m == 1;
    const float lam = second ? 0.f : a.lam[h];
    T* orow = second ? (T*)a.out2 + ((int64_t)b * a.Tq + qi) * (a.H * 2 * HD) + h * 2 * HD
                     : (T*)a.out + (int64_t)b * a.bso + (int64_t)qi * a.ldo + h * 2 * HD;
    bf16_t* rrow = kept.value ? rest_row<HD>(a, m, b, qi, h * 2 * HD) : nullptr;
#pragma unroll
    for (int i = 0; i < 2 * CT; ++i) {
      f32x4 x[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int t = i / 2, g = 2 * (i & 1) + k;
        x[k] = f32x4{o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3]} * inv;
        if (!second) x[k] -= ex[(t * 4 + g) * 64] * lam;
      }
      store_columns<kept.value>(orow + i * 16, rrow + i * 16, x[0], x[1], hh);
      PIN();                                                                   // (all of `ex` read at once would spill)
    }
  };
  if (m == 1 && !a.out2) return;
  if (sizeof(T) == 2 && a.rest) finish(std::integral_constant<bool, sizeof(T) == 2>{});
  else finish(std::integral_constant<bool, false>{});
}

// joins few splits: one wave per (sample, head, query); lane owns 4 columns of 2 hd
template <typename T, int HD>
__global__ __launch_bounds__(256) void join_few_kernel(Args a) {
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
      if (t[2 * m + 1] == 0.f) continue;                   // a split without a key, or of scores of -inf
      const float mx = fmaxf(top[m], t[2 * m]);
      sum[m] = sum[m] * exp2_fast((top[m] - mx) * a.c2) + t[2 * m + 1] * exp2_fast((t[2 * m] - mx) * a.c2);
      top[m] = mx;
    }
  }
  const int qi = (int)(row % a.Tq), h = (int)(row / a.Tq % a.H), b = (int)(row / a.Tq / a.H);
  const bool keys = valid_keys(a, b) > 0;
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
    const f32x4 first = keys ? o[0] / sum[0] : o[0], second = keys ? o[1] / sum[1] : o[1];
    const int c = h * 2 * HD + lane * 4;
    store4((T*)a.out + (int64_t)b * a.bso + (int64_t)qi * a.ldo + c, rest_row<HD>(a, 0, b, qi, c), first - second * a.lam[h]);
    if (a.out2) store4((T*)a.out2 + ((int64_t)b * a.Tq + qi) * (a.H * 2 * HD) + c, rest_row<HD>(a, 1, b, qi, c), second);
  }
  if (a.lse && lane < 2) {
    const float s = lane ? sum[1] : sum[0], t = lane ? top[1] : top[0];
    a.lse[(((int64_t)lane * a.B + b) * a.H + h) * a.Tq + qi] = keys ? t * a.c2 + __builtin_amdgcn_logf(s) : INFINITY;
  }
}

// joins many splits: one workgroup per (sample, head, query); each thread owns 4 columns of one map, the splits dealt out to the
// thread groups and their shares added in group order through LDS
template <typename T, int HD>
__global__ __launch_bounds__(256) void join_many_kernel(Args a) {
  constexpr int W = 4 * HD + 4, COLS = HD, GROUPS = 256 / COLS;                // COLS threads: 4 columns each of both maps' 2 hd
  __shared__ float weight[MAX_SPLITS][2];                                      // of a split's sums in the whole
  __shared__ float total[2][2];                                                // top, sum of each map
  __shared__ f32x4 share[256];
  const int64_t row = blockIdx.x, rows = (int64_t)a.B * a.H * a.Tq;
  const float* p = a.part + row * W;
  const int64_t step = rows * W;
  const int tid = threadIdx.x;
  if (tid < 128) {                                                             // wave m: map m
    const int lane = tid & 63, m = tid >> 6;
    float top = -INFINITY, sum = 0.f;
    for (int s = lane; s < a.splits; s += 64) {
      const float t = p[s * step + 4 * HD + 2 * m], v = p[s * step + 4 * HD + 2 * m + 1];
      if (v == 0.f) continue;                                                  // a split without a key, or of scores of -inf
      const float mx = fmaxf(top, t);
      sum = sum * exp2_fast((top - mx) * a.c2) + v * exp2_fast((t - mx) * a.c2);
      top = mx;
    }
    const float all = wave_max(top);
    sum = wave_sum(sum == 0.f ? 0.f : sum * exp2_fast((top - all) * a.c2));
    for (int s = lane; s < a.splits; s += 64) {
      const float v = p[s * step + 4 * HD + 2 * m + 1];
      weight[s][m] = v == 0.f ? 0.f : exp2_fast((p[s * step + 4 * HD + 2 * m] - all) * a.c2) / sum;
    }
    if (lane == 0) {
      total[m][0] = all;
      total[m][1] = sum;
    }
  }
  __syncthreads();
  const int c = tid % COLS, grp = tid / COLS, m = c / (HD / 2);
  if (grp < GROUPS) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s = grp; s < a.splits; s += GROUPS) {
      const float w = weight[s][m];
      if (w != 0.f) acc += *reinterpret_cast<const f32x4*>(p + s * step + c * 4) * w;   // (a weight of 0: sums that hold nothing, or nothing left of them)
    }
    share[tid] = acc;
  }
  __syncthreads();
  const int qi = (int)(row % a.Tq), h = (int)(row / a.Tq % a.H), b = (int)(row / a.Tq / a.H);
  const bool keys = valid_keys(a, b) > 0;
  if (tid < HD / 2) {
    f32x4 first = share[tid], second = share[tid + HD / 2];
#pragma unroll
    for (int q = 1; q < GROUPS; ++q) {
      first += share[q * COLS + tid];
      second += share[q * COLS + tid + HD / 2];
    }
    if (keys && total[0][1] == 0.f) first *= NAN;                               // 0 / 0 (no split has a weight)
    if (keys && total[1][1] == 0.f) second *= NAN;
    const int col = h * 2 * HD + tid * 4;
    store4((T*)a.out + (int64_t)b * a.bso + (int64_t)qi * a.ldo + col, rest_row<HD>(a, 0, b, qi, col), first - second * a.lam[h]);
    if (a.out2) store4((T*)a.out2 + ((int64_t)b * a.Tq + qi) * (a.H * 2 * HD) + col, rest_row<HD>(a, 1, b, qi, col), second);
  }
  if (a.lse && tid < 2) {
    const float s = total[tid][1];
    a.lse[(((int64_t)tid * a.B + b) * a.H + h) * a.Tq + qi] = keys ? total[tid][0] * a.c2 + __builtin_amdgcn_logf(s) : INFINITY;
  }
}

// query groups of 32 per workgroup: four share a K | V tile where that still leaves every CU a workgroup
int groups_for(int64_t pairs, int Tq) { return Tq <= 32 ? 1 : pairs * ((Tq + 127) / 128) >= 256 ? 4 : 2; }

// spans of keys per (sample, head, query block): as many as give 256 CUs a workgroup each (two of the small ones), none shorter than
// 256 keys (fp32, where a key costs eight times as much: 128)
int splits_for(int dtype, int B, int Tq, int Tk, int H) {
  const int64_t pairs = (int64_t)B * H;
  const int nw = groups_for(pairs, Tq);
  const int64_t wgs = pairs * ((Tq + 32 * nw - 1) / (32 * nw));
  if (wgs >= 192) return 1;
  const int64_t want = (nw == 1 ? MAX_SPLITS : 256) / wgs, least = dtype == GPT_BF16 ? 256 : 128, most = (Tk + least - 1) / least;
  return (int)(want < most ? want : most);
}

template <typename T, int HD, int NW>
int launch_nw(const Args& a, hipStream_t s) {
  const char* who = "gpt_diff_attention";
  static GptPerDevice once;
  if (int st = grant_lds(fwd_kernel<T, HD, NW>, once, who)) return st;
  const int64_t grid = (int64_t)a.B * a.H * a.splits * ((a.Tq + 32 * NW - 1) / (32 * NW));
  GPT_REQUIRE(grid * NW * 128 < (1ll << 32) && grid < (1ll << 31), "%s: too many workgroups (%lld)", who, (long long)grid);
  constexpr int LDS = 4 * KEYS<T, NW> * Tile<T, HD>::PITCH;
  static_assert(NW * 2 * HD / 32 * 4 * 64 * 16 <= LDS, "the hand-over of the second map's halves has to fit the tiles' LDS");
  hipLaunchKernelGGL((fwd_kernel<T, HD, NW>), dim3((unsigned)grid), dim3(NW * 128), LDS, s, a);
  return gpt_launch_status(who);
}

template <typename T, int HD>
int launch(const Args& a, hipStream_t s) {
  const int nw = groups_for((int64_t)a.B * a.H, a.Tq);
  if (int st = nw == 4 ? launch_nw<T, HD, 4>(a, s) : nw == 2 ? launch_nw<T, HD, 2>(a, s) : launch_nw<T, HD, 1>(a, s)) return st;
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.B * a.H * a.Tq;
    // few splits come with many rows, where a wave each is enough: 2 splits x 4112 rows (hd 96, fp32) 7.0 us, a workgroup each 11.2;
    // 64 splits x 32 rows (hd 128) go through a wave one after another, 12.6 us, a workgroup 4.9
    if (a.splits < 8)
      hipLaunchKernelGGL((join_few_kernel<T, HD>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((join_many_kernel<T, HD>), dim3((unsigned)rows), dim3(256), 0, s, a);
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
  a->ldq = row_step(p->ldq, p->Tq, w); a->bsq = p->bsq;
  a->ldk = row_step(p->ldk, p->Tk, w); a->bsk = p->bsk;
  a->ldv = row_step(p->ldv, p->Tk, w); a->bsv = p->bsv;
  a->lam = p->lam; a->lengths = p->lengths;
  a->out = p->out; a->ldo = p->ldo; a->bso = p->bso; a->lse = p->lse; a->out2 = p->out2;
  a->B = p->B; a->Tq = p->Tq; a->Tk = p->Tk; a->H = p->n_head;
  a->scale = p->scale; a->c2 = p->scale * LOG2E;
  a->splits = 1; a->split_keys = p->Tk;
  return 0;
}

int check_rest(const gpt_diff_attention_t* p, void* rest, const char* who, Args* a) {
  GPT_REQUIRE(!rest || (p->dtype == GPT_BF16 && p->out2), "%s: rest belongs to a bf16 call that keeps out2", who);
  GPT_REQUIRE((uintptr_t)rest % 16 == 0, "%s: misaligned operand", who);
  a->rest = (bf16_t*)rest;
  return 0;
}

}  // namespace diffattn

using namespace diffattn;

static int64_t fwd_workspace(int dtype, int B, int Tq, int Tk, int n_head, int hd) {
  if (Tq <= SHORT && Tk <= SHORT) return 0;
  const int n = splits_for(dtype, B, Tq, Tk, n_head);
  return n > 1 ? (int64_t)n * B * n_head * Tq * (4 * hd + 4) * (int64_t)sizeof(float) : 0;
}

extern "C" int gpt_diff_attention_workspace(int dtype, int B, int Tq, int Tk, int n_head, int hd, int64_t* host_bytes) {
  GPT_REQUIRE(host_bytes && (dtype == GPT_F32 || dtype == GPT_BF16) && B > 0 && Tq > 0 && Tk > 0 && n_head > 0 && hd > 0,
              "gpt_diff_attention_workspace: bad arguments");
  *host_bytes = fwd_workspace(dtype, B, Tq, Tk, n_head, hd);
  return 0;
}

extern "C" int gpt_diff_attention(const gpt_diff_attention_t* p, void* stream) { return gpt_diff_attention_keep(p, nullptr, stream); }

extern "C" int gpt_diff_attention_keep(const gpt_diff_attention_t* p, void* rest, void* stream) {
  const char* who = "gpt_diff_attention";
  Args a;
  if (int st = make_args(p, who, &a)) return st;
  if (int st = check_rest(p, rest, who, &a)) return st;
  if (p->Tq <= SHORT && p->Tk <= SHORT) return short_attention(a, p->dtype, p->hd, false, (hipStream_t)stream);
  const int64_t need = fwd_workspace(p->dtype, p->B, p->Tq, p->Tk, p->n_head, p->hd);
  if (need > 0) {
    GPT_REQUIRE(p->ws && (uintptr_t)p->ws % 16 == 0 && p->ws_bytes >= need, "%s: needs %lld bytes of scratch", who, (long long)need);
    const int n = splits_for(p->dtype, p->B, p->Tq, p->Tk, p->n_head);
    a.part = (float*)p->ws;
    a.splits = n;
    a.split_keys = ((p->Tk + n - 1) / n + 63) / 64 * 64;
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
