// Differential attention, backward (diffattn_short.hip takes Tq, Tk <= 32).  With dP = dO V^T, D_i = rowsum(P_i dP):
//   dS_1 = P_1 (dP - D_1),  dS_2 = -lam P_2 (dP - D_2)
//   dQ_i = c dS_i K_i,  dK_i = c dS_i^T Q_i,  dV = (P_1 - lam P_2)^T dO,  dlam = -sum P_2 dP
// The maps are recomputed from the kept log-sum-exps; D_i = dO . O_i comes from the kept outputs. Two sweeps, over key tiles for dQ
// and over query tiles for dK / dV, so that every sum is taken by one wave in a fixed order (or by one per span, joined in the spans'
// order).  dlam, which is what nearly cancelling terms leave: in bf16 from the fp32 P_2 and dP of the second sweep (D_2 is good to 16 bits); in
// fp32 the sum of the rows' D_2, whose maps the forward has divided by their own sums (a row of recomputed P_2 adds to 1 within the
// rounding of its log-sum-exp: 40 draws of 4 x 257 tokens 6.3e-7 of dlam off rms, from D_2 4.8e-7, the plain formula in fp32 5.5e-7).
// A wave holds 16 rows of its side for BOTH maps - operands and accumulators, some 230 registers at hd 128, two waves per SIMD: dP
// serves both maps, so a wave per map would compute it twice (a third more matrix work in dQ, a half in dK / dV), and 32 rows per wave
// would leave one wave per SIMD with nothing beside it while it waits for LDS or exponentials (T = 4096, 16 (sample, head), hd 128, with
// one bf16 operand: dK / dV 1069 us, dQ 735; with 16 rows 640 and 470).  The other side comes in tiles of 32 rows by LDS-DMA, shared
// by the workgroup's waves; every tile is used twice, by rows for the scores and transposed for the gradient products.
// bf16: P and dS enter the gradient products as two operands each (16 bits of mantissa), so that the gradients' own rounding is the
// only one to 8 bits: one operand leaves dQ, dK, dV 2.35e-3 rms off where rounding the exact result leaves 1.66e-3.  It costs half of
// dK / dV's matrix work again and a third of dQ's: 757 and 538 us (1.09 and 1.02 PFLOP/s of their 824 and 550 GFLOP) instead of 640 and
// 471; 16 samples of up to 515 tokens, hd 64, 53 and 44 instead of 47 and 39.
#include "diffattn.h"

namespace diffattn {
int make_args(const gpt_diff_attention_t* p, const char* who, Args* a);
int check_rest(const gpt_diff_attention_t* p, void* rest, const char* who, Args* a);

namespace {

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
__device__ __forceinline__ void frag_negate(Frag<bf16_t>& f) {
  u32x4 w = __builtin_bit_cast(u32x4, f.v);
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] ^= 0x80008000u;
  f.v = __builtin_bit_cast(bf16x8, w);
}
__device__ __forceinline__ void frag_negate(Frag<float>& f) {
#pragma unroll
  for (int j = 0; j < 8; ++j) f.v[j] = -f.v[j];
}
// block c of 32 elements of the row at p (16-byte aligned), zeros where !ok: lane group g takes 8 consecutive ones in bf16, two
// 16-byte chunks four apart in fp32 (as row16 reads them)
__device__ __forceinline__ Frag<bf16_t> frag_row(const bf16_t* p, int c, int g, bool ok) {
  Frag<bf16_t> f;
  frag_zero(f);
  if (ok) f.v = *reinterpret_cast<const bf16x8*>(p + c * 32 + g * 8);
  return f;
}
__device__ __forceinline__ Frag<float> frag_row(const float* p, int c, int g, bool ok) {
  Frag<float> f;
  frag_zero(f);
  if (ok) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p + c * 32 + g * 4), b = *reinterpret_cast<const f32x4*>(p + c * 32 + 16 + g * 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) { f.v[j] = a[j]; f.v[4 + j] = b[j]; }
  }
  return f;
}
// two accumulator tiles (rows 0..15 and 16..31 of the contraction) as an operand; bf16: as two, `low` what the rounding to the first
// leaves (16 bits of mantissa together; fp32 has no second)
__device__ __forceinline__ void frag_pair(Frag<bf16_t>& f, Frag<bf16_t>& low, const f32x4& lo, const f32x4& hi) {
#pragma clang fp contract(off)                                           // (an fma with the product that x is would keep both its factors)
  u32x4 w, v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float x = j < 2 ? lo[2 * j] : hi[2 * j - 4], y = j < 2 ? lo[2 * j + 1] : hi[2 * j - 3];
    w[j] = pack_bf16x2(x, y);
    v[j] = pack_bf16x2(x - __uint_as_float(w[j] << 16), y - __uint_as_float(w[j] & 0xffff0000u));
  }
  f.v = __builtin_bit_cast(bf16x8, w);
  low.v = __builtin_bit_cast(bf16x8, v);
}
__device__ __forceinline__ void frag_pair(Frag<float>& f, Frag<float>&, const f32x4& lo, const f32x4& hi) {
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


// this lane's row of 16 in a tile: chunk 4 ks + (lane >> 4) in bf16, chunks 8 ks + (lane >> 4) and four further in fp32
template <typename T, int HD>
__device__ __forceinline__ int row16_base(int lane) {
  return Tile<T, HD>::at(lane & 15, lane >> 4);
}
template <typename T, int HD>
__device__ __forceinline__ Frag<T> row16(const char* tile, int rb, int row0, int ks) {
  using L = Tile<T, HD>;
  Frag<T> f;
  const char* p = tile + row0 * L::PITCH;                                  // constant but for smem: the instruction's offset
  if constexpr (sizeof(T) == 2) {
    f.v = *reinterpret_cast<const bf16x8*>(p + L::add(rb, 4 * ks));
  } else {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p + L::add(rb, 8 * ks)), b = *reinterpret_cast<const f32x4*>(p + L::add(rb, 8 * ks + 4));
#pragma unroll
    for (int j = 0; j < 4; ++j) { f.v[j] = a[j]; f.v[4 + j] = b[j]; }
  }
  return f;
}

// columns 16 t .. of a tile of 32 rows as an operand whose contraction index is the rows, in the order in which two accumulator tiles
// hold them (frag_from): slot j of lane group g = row 16 (j >> 2) + 4 g + (j & 3)
template <typename T, int HD>
__device__ __forceinline__ int col16_base(int lane) {
  using L = Tile<T, HD>;
  const int g = lane >> 4;
  if constexpr (sizeof(T) == 2) return L::at(4 * g + ((lane & 15) >> 2), (lane & 3) >> 1) + 8 * (lane & 1);
  return L::at(4 * g, (lane & 15) >> 2) + (lane & 3) * 4;
}
template <typename T, int HD>
__device__ __forceinline__ Frag<T> col16(const char* tile, int cb, int t) {
  using L = Tile<T, HD>;
  Frag<T> f;
  if constexpr (sizeof(T) == 2) {
    const char* p = tile + L::add(cb, 2 * t);
    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_ptr)p);
    const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_ptr)(p + 16 * L::PITCH));
    f.v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)                                            // f(row) = ((j & 3) << 2) ^ f(4 g): fp32 rows are multiples of 256 bytes
      f.v[j] = *reinterpret_cast<const float*>(tile + L::add(cb ^ ((j & 3) << 6), 4 * t) + (16 * (j >> 2) + (j & 3)) * L::PITCH);
  }
  return f;
}

// per (sample, head, query) the two log-sum-exps and D_1 = dO . (out + lam out2), D_2 = dO . out2: 16 lanes each.  In bf16 with what
// their roundings left added back: dS = P (dP - D) is small where a row has few keys or one that outweighs the others, and D from the rounded
// outputs is off by 2^-9 of dP there (a row of one key has dS = 0; 16 samples of up to 515 tokens: dQ 1.71e-3 rms off, 1.66e-3 with it)
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
    u32x4 ry = {0u, 0u, 0u, 0u}, rz = ry;
    if (sizeof(T) == 2 && a.rest) {
      const bf16_t* r = a.rest + row * (2 * HD);
      ry = reinterpret_cast<const u32x4*>(r)[ch];
      rz = reinterpret_cast<const u32x4*>(r + rows * (2 * HD))[ch];
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      float xv, yv, zv;
      if constexpr (sizeof(T) == 2) {
        const int sh = (j & 1) ? 0 : 16;
        xv = __uint_as_float((x[j >> 1] << sh) & 0xffff0000u);
        yv = __uint_as_float((y[j >> 1] << sh) & 0xffff0000u) + __uint_as_float((ry[j >> 1] << sh) & 0xffff0000u);
        zv = __uint_as_float((z[j >> 1] << sh) & 0xffff0000u) + __uint_as_float((rz[j >> 1] << sh) & 0xffff0000u);
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

// stages of the tile ring: the tile in use, the next one in flight and, where the halves of a workgroup run a part apart, the one before
template <typename T, int NW>
constexpr int STAGES = sizeof(T) == 2 && NW == 8 ? 3 : 2;
// Operands read from LDS ahead of the matrix instruction that takes them: left to itself the compiler reads each one right before its
// use and waits out the LDS latency there (dK / dV at T = 4096, hd 128: 850 us).  PIN() keeps the written order.
template <typename T>
constexpr int AHEAD = sizeof(T) == 2 ? 3 : 1;
// x, opaque to the compiler: what is formed from it is formed where it is used and holds no register over the loop
template <typename V>
__device__ __forceinline__ V opaque(V x) {
  asm volatile("" : "+v"(x));
  return x;
}
#define PIN() __builtin_amdgcn_sched_barrier(0)

// dQ: NW waves of 16 queries; K | V tiles of 32 keys.  S_i^T = K_i Q_i^T and dP^T = V dO^T: keys on the accumulator's rows.
template <typename T, int HD, int NW>
__global__ __launch_bounds__(NW * 64) void dq_kernel(Args a) {
  using L = Tile<T, HD>;
  constexpr int NT = NW * 64, NS = STAGES<T, NW>, TILE = 32 * L::PITCH, STAGE = 2 * TILE, KC = HD / 32, CT = HD / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];            // [NS][K | V]
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int blocks = (a.Tq + 16 * NW - 1) / (16 * NW);
  int pair, block;
  xcd_block(blockIdx.x, gridDim.x, blocks * a.k_splits, &pair, &block);
  const int split = block / blocks;
  block -= split * blocks;
  const int b = pair / a.H, h = pair - b * a.H, len = valid_keys(a, b);
  const T* kb = (const T*)a.k + (int64_t)b * a.bsk + h * 2 * HD;
  const T* vb = (const T*)a.v + (int64_t)b * a.bsv + h * 2 * HD;
  const int qi = (block * NW + wid) * 16 + col;
  const bool qok = qi < a.Tq;
  Frag<T> qf[2 * KC], gf[2 * KC];
  {
    const T* qr = (const T*)a.q + (int64_t)b * a.bsq + (int64_t)(qok ? qi : 0) * a.ldq + h * 2 * HD;
    const T* gr = (const T*)a.dout + (int64_t)b * a.bsdo + (int64_t)(qok ? qi : 0) * a.lddo + h * 2 * HD;
#pragma unroll
    for (int c = 0; c < 2 * KC; ++c) {
      qf[c] = frag_row(qr, c, g, qok);
      gf[c] = frag_row(gr, c, g, qok);
    }
  }
  const f32x4 st = a.stats[(int64_t)pair * a.Tq + (qok ? qi : 0)];
  const float lam = a.lam[h];
  f32x4 acc[2 * CT];
#pragma unroll
  for (int t = 0; t < 2 * CT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int rb = row16_base<T, HD>(lane), cb = col16_base<T, HD>(lane);
  const int first = split * a.k_tiles, n = min((len + 31) / 32 - first, a.k_tiles);   // tiles of this span
  auto fetch = [&](int it, int at) {
    char* dst = smem + at;
    it += first;
    dma_tile<T, HD, 32, NT>(kb + (int64_t)it * 32 * a.ldk, a.ldk, len - it * 32, dst, tid, wid);
    dma_tile<T, HD, 32, NT>(vb + (int64_t)it * 32 * a.ldv, a.ldv, len - it * 32, dst + TILE, tid, wid);
  };
  // The step's three parts: scores and dP (matrix), dS (vector), products with K (matrix).  All waves meet at one barrier per tile, and
  // the two waves of a SIMD would do the same part at the same time: the workgroup's second half runs a part behind, its products with
  // K taken from the tile before while the first half computes scores.
  constexpr int NA = 4 * KC, R = AHEAD<T> + 1;
  const bool late = NS == 3 && wid >= NW / 2;
  f32x4 dp[2], s[2][2];
  Frag<T> ring[R], x[2], low[2];
  auto scores = [&](int at, int it) {
    // the lane's place in this stage, opaque to the compiler: it would keep every variant of it in a register over the loop
    int rk = rb + at;
    asm volatile("" : "+v"(rk));
    auto rows = [&](int u, int i) { return row16<T, HD>(smem + (i & 1 ? 0 : TILE), rk, 16 * u, i / 2); };
#pragma unroll
    for (int i = 0; i < AHEAD<T>; ++i) ring[i] = rows(0, i);
    PIN();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      dp[u] = s[0][u] = s[1][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        const int n = u * NA + i + AHEAD<T>;
        if (n < 2 * NA) ring[n % R] = rows(n / NA, n % NA);
        const Frag<T>& f = ring[(u * NA + i) % R];
        if (i & 1) s[i / 2 / KC][u] = mma16(f, qf[i / 2], s[i / 2 / KC][u]);
        else dp[u] = mma16(f, gf[i / 2], dp[u]);
        PIN();
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[m][u][r] = exp2_fast(s[m][u][r] * a.c2 - st[m]) * (dp[u][r] - st[2 + m]);
    it += first;
    if (it * 32 + 32 > len) {
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (it * 32 + 16 * u + 4 * g + r >= len) s[m][u][r] = 0.f;
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) frag_pair(x[m], low[m], s[m][0], s[m][1]);
  };
  auto products = [&](int at) {
    int ck = cb + at;
    asm volatile("" : "+v"(ck));
#pragma unroll
    for (int t = 0; t < AHEAD<T>; ++t) ring[t] = col16<T, HD>(smem, ck, t);
    PIN();
#pragma unroll
    for (int t = 0; t < 2 * CT; ++t) {
      if (t + AHEAD<T> < 2 * CT) ring[(t + AHEAD<T>) % R] = col16<T, HD>(smem, ck, t + AHEAD<T>);
      acc[t] = mma16(ring[t % R], x[t / CT], acc[t]);
      if constexpr (sizeof(T) == 2) acc[t] = mma16(ring[t % R], low[t / CT], acc[t]);
      PIN();
    }
  };
  int before = 0, now = 0;                                                  // stages of the previous tile and of this one
  if (n > 0) fetch(0, 0);
  for (int it = 0; it < n; ++it) {
    tile_barrier<0>();
    const int next = now + STAGE == NS * STAGE ? 0 : now + STAGE;
    if (it + 1 < n) fetch(it + 1, next);                                     // the buffer of two tiles (NS == 2: one tile) ago
    if (late && it > 0) products(before);
    scores(now, it);
    if (!late) products(now);
    before = now;
    now = next;
  }
  if (late && n > 0) products(before);
  if constexpr (sizeof(T) == 4) {
    const float sum = wave_sum(qok && g == 0 ? st[3] : 0.f);
    if (lane == 0 && split == 0) a.dlam_part[((int64_t)h * a.B + b) * (blocks * NW) + block * NW + wid] = sum;
  }
  if (!qok) return;
  auto store = [&](auto* dq) {
#pragma unroll
    for (int t = 0; t < 2 * CT; ++t) store4(dq + t * 16, acc[t] * (t < CT ? a.scale : -lam * a.scale));   // -lam of dS_2: here, once
  };
  if (a.k_splits > 1) store(a.dq_part + (((int64_t)split * a.B * a.H + pair) * a.Tq + qi) * (2 * HD) + 4 * g);
  else store((T*)a.dq + (int64_t)b * a.bsdq + (int64_t)qi * a.lddq + h * 2 * HD + 4 * g);
}

// dK, dV and the tile's share of sum P_2 dP: NW waves of 16 keys; Q | dO | statistics tiles of 32 queries.  S_i = Q_i K_i^T and
// dP = dO V^T: queries on the accumulator's rows.  Queries behind Tq arrive as zeros in all three: their dP, D and products are 0.
template <typename T, int HD, int NW>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 2 && HD == 64 ? 3 : 1) void dkv_kernel(Args a) {
  using L = Tile<T, HD>;
  constexpr int NT = NW * 64, NS = STAGES<T, NW>, TILE = 32 * L::PITCH, STAGE = 2 * TILE + 512, KC = HD / 32, CT = HD / 16;
  constexpr bool NEGATE = sizeof(T) == 2;
  extern __shared__ __attribute__((aligned(16))) char smem[];            // [NS][Q | dO | stats]
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int blocks = (a.Tk + 16 * NW - 1) / (16 * NW);
  int pair, block;
  xcd_block(blockIdx.x, gridDim.x, blocks * a.q_splits, &pair, &block);
  const int split = block / blocks;
  block -= split * blocks;
  const int b = pair / a.H, h = pair - b * a.H, len = valid_keys(a, b);
  const T* qb = (const T*)a.q + (int64_t)b * a.bsq + h * 2 * HD;
  const T* gb = (const T*)a.dout + (int64_t)b * a.bsdo + h * 2 * HD;
  const f32x4* sb = a.stats + (int64_t)pair * a.Tq;
  const int key = (block * NW + wid) * 16 + col;
  const bool ok = key < len;
  Frag<T> kf[2 * KC], vf[2 * KC];
  {
    const T* kr = (const T*)a.k + (int64_t)b * a.bsk + (int64_t)(ok ? key : 0) * a.ldk + h * 2 * HD;
    const T* vr = (const T*)a.v + (int64_t)b * a.bsv + (int64_t)(ok ? key : 0) * a.ldv + h * 2 * HD;
#pragma unroll
    for (int c = 0; c < 2 * KC; ++c) {
      kf[c] = frag_row(kr, c, g, ok);
      vf[c] = frag_row(vr, c, g, ok);
      if (NEGATE && wid & 1) frag_negate(vf[c]);
    }
  }
  // The matrix unit's sums lean down by some 2^-32 of their terms' size: next to nothing, but dlam's terms nearly cancel (at 4 x 4096 x
  // 4096 of them the lean is 1e-6 of it).  Where it is summed here every other wave takes -V and so has the lean of -dP.
  const float sign = NEGATE && wid & 1 ? -1.f : 1.f;
  const float lam = a.lam[h];
  f32x4 dk[2 * CT], dv[2 * CT];
#pragma unroll
  for (int t = 0; t < 2 * CT; ++t) dk[t] = dv[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  double dlam = 0.0;
  const int rb = row16_base<T, HD>(lane), cb = col16_base<T, HD>(lane);
  const int first = split * a.q_tiles;
  const int n = block * NW * 16 < len ? min((a.Tq + 31) / 32 - first, a.q_tiles) : 0;   // a block without a valid key: zeros
  auto fetch = [&](int it, int at) {
    char* dst = smem + at;
    it += first;
    dma_tile<T, HD, 32, NT>(qb + (int64_t)it * 32 * a.ldq, a.ldq, a.Tq - it * 32, dst, tid, wid);
    dma_tile<T, HD, 32, NT>(gb + (int64_t)it * 32 * a.lddo, a.lddo, a.Tq - it * 32, dst + TILE, tid, wid);
    if (wid == 0) dma_bytes(sb + it * 32, (a.Tq - it * 32) * 16, dst + 2 * TILE, lane);
  };
  constexpr int NA = 4 * KC, LEAD = HD == 128 && sizeof(T) == 2 ? 2 : AHEAD<T>, R = LEAD + 1;   // (3 at hd 128: 251 registers and no faster)
  const bool late = NS == 3 && wid >= NW / 2;                               // as in dq_kernel
  f32x4 dp[2], p[2], s[2][2];
  Frag<T> ring[R], pf, df[2], pl, dl[2];
  auto scores = [&](int at) {
    int rq = rb + at;
    asm volatile("" : "+v"(rq));
    auto rows = [&](int u, int i) { return row16<T, HD>(smem + (i & 1 ? 0 : TILE), rq, 16 * u, i / 2); };
#pragma unroll
    for (int i = 0; i < LEAD; ++i) ring[i] = rows(0, i);
    PIN();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      dp[u] = s[0][u] = s[1][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        const int n = u * NA + i + LEAD;
        if (n < 2 * NA) ring[n % R] = rows(n / NA, n % NA);
        const Frag<T>& f = ring[(u * NA + i) % R];
        if (i & 1) s[i / 2 / KC][u] = mma16(f, kf[i / 2], s[i / 2 / KC][u]);
        else dp[u] = mma16(f, vf[i / 2], dp[u]);
        PIN();
      }
    }
    float part = 0.f;
    const f32x4* ts = reinterpret_cast<const f32x4*>(smem + 2 * TILE + 64 * (opaque(lane) >> 4) + at);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 st = ts[16 * u + r];
        const float p0 = exp2_fast(s[0][u][r] * a.c2 - st[0]), p1 = exp2_fast(s[1][u][r] * a.c2 - st[1]);
        const float d = sign * dp[u][r];
        p[u][r] = p0 - lam * p1;
        if constexpr (sizeof(T) == 2) part += p1 * d;
        s[0][u][r] = p0 * (d - st[2]);
        s[1][u][r] = p1 * (d - st[3]);                                       // -lam: at the end, once
      }
    if constexpr (sizeof(T) == 2) dlam += opaque(part);                                                    // here, not behind the products: its terms would be kept over them
    frag_pair(pf, pl, p[0], p[1]);
#pragma unroll
    for (int m = 0; m < 2; ++m) frag_pair(df[m], dl[m], s[m][0], s[m][1]);
  };
  auto products = [&](int at) {
    int cq = cb + at;
    asm volatile("" : "+v"(cq));
    auto cols = [&](int i) { return col16<T, HD>(smem + (i & 1 ? 0 : TILE), cq, i / 2); };
#pragma unroll
    for (int i = 0; i < LEAD; ++i) ring[i] = cols(i);
    PIN();
#pragma unroll
    for (int i = 0; i < 4 * CT; ++i) {
      const int t = i / 2;
      if (i + LEAD < 4 * CT) ring[(i + LEAD) % R] = cols(i + LEAD);
      if (i & 1) dk[t] = mma16(ring[i % R], df[t / CT], dk[t]);
      else dv[t] = mma16(ring[i % R], pf, dv[t]);
      if constexpr (sizeof(T) == 2) {
        if (i & 1) dk[t] = mma16(ring[i % R], dl[t / CT], dk[t]);
        else dv[t] = mma16(ring[i % R], pl, dv[t]);
      }
      PIN();
    }
  };
  int before = 0, now = 0;
  if (n > 0) fetch(0, 0);
  for (int it = 0; it < n; ++it) {
    tile_barrier<0>();
    const int next = now + STAGE == NS * STAGE ? 0 : now + STAGE;
    if (it + 1 < n) fetch(it + 1, next);
    if (late && it > 0) products(before);
    scores(now);
    if (!late) products(now);
    before = now;
    now = next;
  }
  if (late && n > 0) products(before);
  // a masked key's lane has computed with zeros for its operands and another row's statistics: it gives zeros
  if constexpr (sizeof(T) == 2) {
    const float sum = wave_sum(ok ? (float)dlam : 0.f);
    if (lane == 0) a.dlam_part[(((int64_t)h * a.B + b) * a.q_splits + split) * (blocks * NW) + block * NW + wid] = sum;
  }
  if (key >= a.Tk) return;
  auto store = [&](auto* dkr, auto* dvr) {
    const f32x4 none = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 2 * CT; ++t) {
      store4(dkr + t * 16, ok ? dk[t] * (t < CT ? a.scale : -lam * a.scale) : none);
      store4(dvr + t * 16, ok ? dv[t] : none);
    }
  };
  if (a.q_splits > 1) {
    const int64_t at = (((int64_t)split * a.B * a.H + pair) * a.Tk + key) * (2 * HD) + 4 * g;
    store(a.dk_part + at, a.dv_part + at);
  } else {
    store((T*)a.dk + (int64_t)b * a.bsdk + (int64_t)key * a.lddk + h * 2 * HD + 4 * g,
          (T*)a.dv + (int64_t)b * a.bsdv + (int64_t)key * a.lddv + h * 2 * HD + 4 * g);
  }
}

// dlam[h] = -(sum of the head's partial sums): a workgroup, each thread every 256th in index order, then a fixed tree
__device__ __forceinline__ void sum_dlam(const float* __restrict__ part, int64_t n, int h, float* __restrict__ dlam) {
  __shared__ float red[4];
  const float* p = part + (int64_t)h * n;
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 256) s += p[i];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) dlam[h] = -((red[0] + red[1]) + (red[2] + red[3]));
}
__global__ __launch_bounds__(256) void dlam_kernel(const float* __restrict__ part, int64_t n, float* __restrict__ dlam) {
  sum_dlam(part, n, blockIdx.x, dlam);
}

// the spans' sums of dQ (where the keys were split) and of dK, dV (where the queries were), added in the spans' order: a thread owns 4
// columns of a row.  The first n_head workgroups sum dlam instead
template <typename T, int HD>
__global__ __launch_bounds__(256) void join_kernel(Args a, int64_t parts, float* dlam) {
  constexpr int W = 2 * HD, PER = W / 4;
  const int64_t pairs = (int64_t)a.B * a.H, nq = a.k_splits > 1 ? pairs * a.Tq : 0, nk = a.q_splits > 1 ? pairs * a.Tk : 0;
  if ((int)blockIdx.x < a.H) return sum_dlam(a.dlam_part, parts, blockIdx.x, dlam);
  const int64_t i = (int64_t)(blockIdx.x - a.H) * 256 + threadIdx.x;
  int64_t row = i / PER;
  const int c = (int)(i - row * PER) * 4;
  if (row >= nq + 2 * nk) return;
  const bool is_q = row < nq, is_k = !is_q && row < nq + nk;
  row -= is_q ? 0 : is_k ? nq : nq + nk;
  const int n = is_q ? a.Tq : a.Tk, splits = is_q ? a.k_splits : a.q_splits;
  const float* p = (is_q ? a.dq_part : is_k ? a.dk_part : a.dv_part) + row * W + c;
  const int64_t step = (is_q ? nq : nk) * W;
  f32x4 sum = *reinterpret_cast<const f32x4*>(p);
  for (int s = 1; s < splits; ++s) sum += *reinterpret_cast<const f32x4*>(p + s * step);
  const int64_t pair = row / n, t = row - pair * n;
  const int64_t b = pair / a.H, h = pair - b * a.H;
  T* out = (T*)(is_q ? a.dq : is_k ? a.dk : a.dv) + b * (is_q ? a.bsdq : is_k ? a.bsdk : a.bsdv) + t * (is_q ? a.lddq : is_k ? a.lddk : a.lddv);
  store4(out + h * W + c, sum);
}

// waves of 16 rows per workgroup: eight share the tiles where that still gives every CU a workgroup; fp32 from hd 96 on: four, which may
// have 512 registers each (eight would spill)
template <typename T, int HD>
constexpr int MANY = sizeof(T) == 4 && HD >= 96 ? 4 : 8;
// dK / dV in bf16 at hd 64: three waves per SIMD in workgroups of four, which the launch bounds ask for (unasked it took 176 registers:
// 16 samples of up to 515 tokens 67 us, now 57), two in workgroups of eight (4 x 4096 tokens, 8 heads: 870 and 930 us; 16 x 515: 93 and
// 115.  At hd 32, 4 x 4096: 656 and 591; hd 128, T = 4096: 1092 and 760)
template <typename T, int HD>
constexpr int MANY_KEYS = sizeof(T) == 2 && HD == 64 ? 4 : MANY<T, HD>;
// ... else four, one per SIMD: two workgroups of two waves share SIMDs while others idle (32 (sample, head) x 512 tokens, hd 128: dK / dV
// and dQ 51 and 48 us in bf16, 45 and 34 by fours; in fp32 180 and 226, 168 and 126)
constexpr int FEW = 4;
bool many_waves(int64_t pairs, int T) { return T > 32 && pairs * ((T + 127) / 128) >= 192; }

// How a call is cut.  Workgroups of four waves that do not fill the CUs have their sweep split into spans, up to one workgroup per CU
// (two where registers and LDS leave room: hd <= 64), whose sums are joined by a launch of their own (6 to 10 us): worth it from 5
// tiles of 32 rows per span in bf16 and, the matrix rate being an eighth there, from 2 in fp32.  dK / dV and dQ, unsplit and split:
// 16 (sample, head) x 257 tokens, hd 96, fp32: 67 and 52 us, 32 and 24; 2 x 2048, hd 128, bf16: 129 and 106, 46 and 35.
struct Plan {
  bool many_q, many_k;
  int q_splits = 1, q_tiles, k_splits = 1, k_tiles;
  int64_t stats, dlam, dq, dkv;                                            // bytes of the workspace's parts (dkv: each of the two)
  int64_t bytes() const { return stats + dlam + dq + 2 * dkv; }
};
int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }
void spans(int64_t wgs, int64_t fill, int tiles, int least, int* splits, int* per) {
  const int64_t want = fill / wgs, most = tiles / least, n = want < most ? want : most;
  *per = n > 1 ? (int)((tiles + n - 1) / n) : tiles;
  *splits = (tiles + *per - 1) / *per;
}
Plan plan_for(int dtype, int B, int Tq, int Tk, int H, int hd) {
  Plan p;
  const int64_t pairs = (int64_t)B * H;
  const int qt = (Tq + 31) / 32, kt = (Tk + 31) / 32, least = dtype == GPT_BF16 ? 5 : 2, fill = hd <= 64 ? 512 : 256;
  p.many_q = many_waves(pairs, Tq);
  p.many_k = many_waves(pairs, Tk);
  p.q_tiles = qt;
  p.k_tiles = kt;
  if (!p.many_k) spans(pairs * ((kt + 1) / 2), fill, qt, least, &p.q_splits, &p.q_tiles);
  if (!p.many_q) spans(pairs * ((qt + 1) / 2), fill, kt, least, &p.k_splits, &p.k_tiles);
  p.stats = 16 * pairs * Tq;
  // one per 16 keys of the workgroups' blocks and span, in fp32 one per 16 queries
  p.dlam = round16((dtype == GPT_BF16 ? pairs * p.q_splits * (((int64_t)Tk + 127) / 128 * 8) : pairs * (((int64_t)Tq + 127) / 128 * 8)) * 4);
  p.dq = p.k_splits > 1 ? pairs * p.k_splits * Tq * 2 * hd * 4 : 0;
  p.dkv = p.q_splits > 1 ? pairs * p.q_splits * Tk * 2 * hd * 4 : 0;
  return p;
}

template <typename T, int HD, int NW>
int launch_dq(const Args& a, hipStream_t s) {
  const char* who = "gpt_diff_attention_bwd";
  static GptPerDevice once;
  const int64_t grid = ((int64_t)a.Tq + 16 * NW - 1) / (16 * NW) * a.k_splits * a.H * a.B;
  GPT_REQUIRE(grid * NW * 64 < (1ll << 32) && grid < (1ll << 31), "%s: too many workgroups (%lld)", who, (long long)grid);
  if (int st = grant_lds(dq_kernel<T, HD, NW>, once, who)) return st;
  hipLaunchKernelGGL((dq_kernel<T, HD, NW>), dim3((unsigned)grid), dim3(NW * 64), (STAGES<T, NW> * 64 * Tile<T, HD>::PITCH), s, a);
  return gpt_launch_status(who);
}

template <typename T, int HD, int NW>
int launch_dkv(const Args& a, hipStream_t s) {
  const char* who = "gpt_diff_attention_bwd";
  static GptPerDevice once;
  const int64_t grid = ((int64_t)a.Tk + 16 * NW - 1) / (16 * NW) * a.q_splits * a.H * a.B;
  GPT_REQUIRE(grid * NW * 64 < (1ll << 32) && grid < (1ll << 31), "%s: too many workgroups (%lld)", who, (long long)grid);
  if (int st = grant_lds(dkv_kernel<T, HD, NW>, once, who)) return st;
  hipLaunchKernelGGL((dkv_kernel<T, HD, NW>), dim3((unsigned)grid), dim3(NW * 64), (STAGES<T, NW> * (64 * Tile<T, HD>::PITCH + 512)), s, a);
  return gpt_launch_status(who);
}

template <typename T, int HD>
int launch(const Args& a, const Plan& plan, f32x4* stats, float* dlam, hipStream_t s) {
  const char* who = "gpt_diff_attention_bwd";
  const int64_t pairs = (int64_t)a.B * a.H, rows = pairs * a.Tq, nd = (rows + 15) / 16;
  GPT_REQUIRE(nd < (1ll << 24), "%s: too many rows (%lld)", who, (long long)rows);
  hipLaunchKernelGGL((stats_kernel<T, HD>), dim3((unsigned)nd), dim3(256), 0, s, a, stats);
  if (int st = gpt_launch_status(who)) return st;
  constexpr int M = MANY<T, HD>, MK = MANY_KEYS<T, HD>;
  if (int st = plan.many_k ? launch_dkv<T, HD, MK>(a, s) : launch_dkv<T, HD, FEW>(a, s)) return st;
  if (int st = plan.many_q ? launch_dq<T, HD, M>(a, s) : launch_dq<T, HD, FEW>(a, s)) return st;
  const int nk = plan.many_k ? MK : FEW, nq = plan.many_q ? M : FEW;                    // parts of dlam per head
  const int64_t parts = sizeof(T) == 2 ? (int64_t)a.B * a.q_splits * (((int64_t)a.Tk + 16 * nk - 1) / (16 * nk) * nk)
                                       : (int64_t)a.B * (((int64_t)a.Tq + 16 * nq - 1) / (16 * nq) * nq);
  const int64_t joined = ((a.k_splits > 1 ? rows : 0) + (a.q_splits > 1 ? 2 * pairs * a.Tk : 0)) * (HD / 2);
  if (joined > 0)
    hipLaunchKernelGGL((join_kernel<T, HD>), dim3((unsigned)(a.H + (joined + 255) / 256)), dim3(256), 0, s, a, parts, dlam);
  else
    hipLaunchKernelGGL(dlam_kernel, dim3(a.H), dim3(256), 0, s, a.dlam_part, parts, dlam);
  return gpt_launch_status(who);
}

}  // namespace
}  // namespace diffattn

using namespace diffattn;

static int64_t bwd_workspace(int dtype, int B, int Tq, int Tk, int n_head, int hd) {
  if (Tq <= SHORT && Tk <= SHORT) return round16((int64_t)n_head * B * 4);
  return plan_for(dtype, B, Tq, Tk, n_head, hd).bytes();
}

extern "C" int gpt_diff_attention_bwd_workspace(int dtype, int B, int Tq, int Tk, int n_head, int hd, int64_t* host_bytes) {
  GPT_REQUIRE(host_bytes && (dtype == GPT_F32 || dtype == GPT_BF16) && B > 0 && Tq > 0 && Tk > 0 && n_head > 0 && hd > 0,
              "gpt_diff_attention_bwd_workspace: bad arguments");
  *host_bytes = bwd_workspace(dtype, B, Tq, Tk, n_head, hd);
  return 0;
}

extern "C" int gpt_diff_attention_bwd(const gpt_diff_attention_t* f, const gpt_diff_attention_bwd_t* p, void* stream) {
  return gpt_diff_attention_bwd_kept(f, nullptr, p, stream);
}

extern "C" int gpt_diff_attention_bwd_kept(const gpt_diff_attention_t* f, const void* rest, const gpt_diff_attention_bwd_t* p, void* stream) {
  const char* who = "gpt_diff_attention_bwd";
  Args a;
  if (int st = make_args(f, who, &a)) return st;
  if (int st = check_rest(f, const_cast<void*>(rest), who, &a)) return st;
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
  const int64_t need = bwd_workspace(f->dtype, f->B, f->Tq, f->Tk, f->n_head, f->hd);
  GPT_REQUIRE(p->ws && (uintptr_t)p->ws % 16 == 0 && p->ws_bytes >= need, "%s: needs %lld bytes of scratch", who, (long long)need);
  a.dout = p->dout; a.lddo = row_step(p->lddo, f->Tq, w); a.bsdo = p->bsdo;
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
  const Plan plan = plan_for(f->dtype, f->B, f->Tq, f->Tk, f->n_head, f->hd);
  f32x4* stats = (f32x4*)p->ws;
  a.stats = stats;
  a.dlam_part = (float*)((char*)p->ws + plan.stats);
  a.dq_part = (float*)((char*)a.dlam_part + plan.dlam);
  a.dk_part = (float*)((char*)a.dq_part + plan.dq);
  a.dv_part = (float*)((char*)a.dk_part + plan.dkv);
  a.q_splits = plan.q_splits; a.q_tiles = plan.q_tiles;
  a.k_splits = plan.k_splits; a.k_tiles = plan.k_tiles;
#define GO(T)                                          \
  switch (f->hd) {                                     \
    case 32: return launch<T, 32>(a, plan, stats, p->dlam, s);  \
    case 64: return launch<T, 64>(a, plan, stats, p->dlam, s);  \
    case 96: return launch<T, 96>(a, plan, stats, p->dlam, s);  \
    default: return launch<T, 128>(a, plan, stats, p->dlam, s); \
  }
  if (f->dtype == GPT_BF16) GO(bf16_t)
  GO(float)
#undef GO
}
