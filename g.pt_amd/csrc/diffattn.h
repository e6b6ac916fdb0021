// What the differential-attention kernels share: the launch's arguments, tiles in LDS and their loads, 32 x 32 matrix products of both
// types.
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
  bf16_t* rest;               // bf16, or NULL: [2][B][Tq][H * 2 hd], what the roundings of out and of out2 leave
  float* part;                // split forward: [splits][B * H][Tq][4 hd + 4]
  int B, Tq, Tk, H, splits, split_keys;
  float scale, c2;            // c2 = scale * log2(e): exp(scale s - m) = exp2(c2 s - m')
  // backward
  const void* dout;
  int64_t lddo, bsdo;
  void *dq, *dk, *dv;
  int64_t lddq, bsdq, lddk, bsdk, lddv, bsdv;
  const f32x4* stats;         // [B][H][Tq]: lse_1, lse_2, D_1, D_2
  float* dlam_part;           // [H][B * splits * key tiles], fp32 [H][B * query tiles]
  // split sweeps: spans of q_tiles / k_tiles tiles of 32, sums of a span [span][B * H][Tq or Tk][2 hd]
  int q_splits, q_tiles, k_splits, k_tiles;
  float *dq_part, *dk_part, *dv_part;
};

// A single row's stride may be anything; the kernels' tiles end where the row after it would begin
inline int64_t row_step(int64_t ld, int T, int64_t w) { return T == 1 ? w : ld; }

// Tq, Tk <= 32 (diffattn_short.hip); the backward needs dlam_part [H][B], no lse, out, out2 or delta
constexpr int SHORT = 32;
int short_attention(const Args& a, int dtype, int hd, bool backward, hipStream_t s);

// dynamic LDS beyond 64 KiB has to be granted per kernel and device
template <typename K>
static int grant_lds(K kernel, GptPerDevice& once, const char* who) {
  if (once.here()) return 0;
  const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
  GPT_REQUIRE(e == hipSuccess, "%s: %s", who, hipGetErrorString(e));
  once.here() = true;
  return 0;
}

__device__ __forceinline__ int valid_keys(const Args& a, int b) {
  if (!a.lengths) return a.Tk;
  const int n = a.lengths[b];
  return n < 0 ? 0 : n > a.Tk ? a.Tk : n;
}

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s* lds_v4s_ptr;
typedef __attribute__((address_space(3))) void* lds_ptr;

// ---- LDS tiles: rows of 2 hd elements (both maps' halves of q or k, or the values of one head).  16-byte chunk c of row r lies at
// chunk c ^ f(r); f has 4 bits where rows start at the same bank (PITCH % 256 == 0), else 3: there bit 3 comes from the row.  No two
// lanes that the LDS serves together hit the same bank:
//   ds_read_b128 serves lanes 0-3, 12-15, 20-27 (measured by its conflicts; the other phases likewise): with one chunk per 32 rows
//     that is one row of each residue mod 16, with chunk C + (lane >> 4) per 16 rows the quads of rows 0, 3 at chunk C and 1, 2 at
//     C + 1 - hence quads 1 and 2 in the same half of a 64-byte group;
//   a transposing read serves 32 lanes: 4 rows x 64 bytes, or 8 rows x 32 (neighbouring quads in different halves).
template <typename T, int HD>
struct Tile {
  static constexpr int ES = sizeof(T), COLS = 2 * HD, PITCH = COLS * ES, CPR = PITCH / 16, CM = CPR / 2;   // bytes per row, chunks per row and per map
  static constexpr int REAL = CPR;
  static constexpr int MASK = PITCH % 256 == 0 ? 15 : 7;
  __device__ static __forceinline__ int f(int r) {
    const int b0 = (r >> 2) & 1, b1 = (r >> 3) & 1, pair = ((b0 ^ b1) << 1) | b1;   // quads of rows 0, 1, 2, 3 -> 0, 2, 3, 1
    if constexpr (PITCH % 256 == 0) return ((r & 3) << 2) | pair;
    return (((r >> 1) & 1) << 2) | pair;
  }
  __device__ static __forceinline__ int at(int r, int chunk) { return r * PITCH + ((chunk ^ f(r)) << 4); }
  // the same in two steps: `base` = at(r, c) of the lane's part c of a chunk number C + c (no common bits), then C
  __device__ static __forceinline__ int add(int base, int C) { return (base ^ ((C & MASK) << 4)) + ((C & ~MASK) << 4); }
};

__device__ __forceinline__ f32x16 zero16() {
  f32x16 v;
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = 0.f;
  return v;
}

// ---- 32 x 32 tiles: the accumulator holds column lane & 31 and rows row_of(register, lane >> 5)
__device__ __forceinline__ int row_of(int reg, int half) { return (reg & 3) + 8 * (reg >> 2) + 4 * half; }

// acc[row of A][row of B] += one 16-byte chunk of each row per lane half (bf16: 16 k-values, one instruction; fp32: 8, four)
template <typename T>
__device__ __forceinline__ f32x16 mma_chunk(const u32x4& a, const u32x4& b, f32x16 c) {
  if constexpr (sizeof(T) == 2) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
  }
}

// A 32 x 32 matrix as an operand that contracts over its rows.  bf16: step s, half hh, slot j holds row 16 s + 8 (j >> 2) + 4 hh +
// (j & 3), which is what an accumulator's registers hold; fp32: register e holds row row_of(e, hh).
struct Operand {
  bf16x8 p[2];
  float f[16];
};
template <typename T>
__device__ __forceinline__ void operand_from(Operand& o, const f32x16& x) {   // bf16: rounded once, here
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = pack_bf16x2(x[8 * s + 2 * j], x[8 * s + 2 * j + 1]);
      o.p[s] = __builtin_bit_cast(bf16x8, w);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) o.f[e] = x[e];
  }
}

// bf16: what the rounding of operand_from left of x, as a second operand (together 16 bits of mantissa)
__device__ __forceinline__ void operand_rest(Operand& rest, const f32x16& x, const Operand& o) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const u32x4 w = __builtin_bit_cast(u32x4, o.p[s]);
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = pack_bf16x2(x[8 * s + 2 * j] - __uint_as_float(w[j] << 16), x[8 * s + 2 * j + 1] - __uint_as_float(w[j] & 0xffff0000u));
    rest.p[s] = __builtin_bit_cast(bf16x8, v);
  }
}

// 4 consecutive values to memory
__device__ __forceinline__ void store4(bf16_t* p, const f32x4& v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}
__device__ __forceinline__ void store4(float* p, const f32x4& v) { *reinterpret_cast<f32x4*>(p) = v; }
// the same, and what the rounding leaves to `rest` (NULL: nowhere)
__device__ __forceinline__ void store4(bf16_t* p, bf16_t* rest, const f32x4& v) {
  const uint32_t a = pack_bf16x2(v[0], v[1]), b = pack_bf16x2(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(a, b);
  if (rest)
    store4(rest, f32x4{v[0] - __uint_as_float(a << 16), v[1] - __uint_as_float(a & 0xffff0000u), v[2] - __uint_as_float(b << 16),
                       v[3] - __uint_as_float(b & 0xffff0000u)});
}
__device__ __forceinline__ void store4(float* p, bf16_t*, const f32x4& v) { store4(p, v); }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }   // v_exp_f32, 1 ulp; exp2(-inf) = 0

// ---- tiles shared by a workgroup of NT threads
// NROWS rows from `src` (row stride ld) by LDS-DMA; rows from `valid` on arrive as zeros (they lie outside the buffer's range).
// The load is written out because the compiler, which knows the builtin's LDS write, would wait for the tile in flight before every
// transposing read of the other one.  It has no register result; tile_barrier() waits for it.
// (A load may read scalar registers that a vector instruction wrote five wait states later at the earliest, and the compiler does not
// look into the text: the descriptor comes from scalar instructions in every kernel, which tests/test_build_cpu.py checks in the built code; a
// wait before each tile's loads would cost dK / dV 1 %.)
template <typename T, int HD, int NROWS, int NT>
__device__ __forceinline__ void dma_tile(const T* src, int64_t ld, int valid, char* dst, int tid, int wid) {
  using L = Tile<T, HD>;
  const int n = valid < NROWS ? valid : NROWS;
  const uint64_t base = (uint64_t)src;
  const u32x4 rsrc = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)base), (uint32_t)__builtin_amdgcn_readfirstlane((int)(base >> 32)) & 0xffffu,
                      (uint32_t)__builtin_amdgcn_readfirstlane(n > 0 ? (int)(((int64_t)(n - 1) * ld + 2 * HD) * L::ES) : 0), 0x00020000u};
  const uint32_t lds = (uint32_t)(uint64_t)(lds_ptr)dst + wid * 1024, row_bytes = (uint32_t)(ld * L::ES);
  constexpr int CHUNKS = NROWS * L::CPR, STEP = NT / L::CPR;
  // threads NT chunks apart: whole rows apart where NT is a multiple of a row's chunks, at the same swizzle where of 16 rows'
  constexpr bool EVEN = NT % (16 * L::CPR) == 0;
  asm volatile("" : "+v"(tid));                                    // the offset is formed anew each time: no register over the loop
  uint32_t off = 0;
#pragma unroll
  for (int c0 = 0; c0 < CHUNKS; c0 += NT) {
    if (CHUNKS % NT != 0 && c0 + wid * 64 >= CHUNKS) break;        // wave-uniform
    if (!EVEN || c0 == 0) {
      const int ci = c0 + tid, row = ci / L::CPR, pos = ci - row * L::CPR;
      off = (uint32_t)row * row_bytes + (uint32_t)((pos ^ L::f(row)) << 4);
    }
    const uint32_t more = EVEN ? (uint32_t)(c0 / NT * STEP) * row_bytes : 0u;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(
                     __builtin_amdgcn_readfirstlane((int)(lds + c0 * 16))),
                 "v"(off + more), "s"(rsrc)
                 : "memory", "m0");
  }
}

// up to 512 consecutive bytes (32 lanes x 16), zeros from `bytes` on
__device__ __forceinline__ void dma_bytes(const void* src, int bytes, char* dst, int lane) {
  const uint64_t base = (uint64_t)src;
  const u32x4 rsrc = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)base), (uint32_t)__builtin_amdgcn_readfirstlane((int)(base >> 32)) & 0xffffu,
                      (uint32_t)__builtin_amdgcn_readfirstlane(bytes < 512 ? bytes : 512), 0x00020000u};
  if (lane < 32)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(
                     __builtin_amdgcn_readfirstlane((int)(uint32_t)(uint64_t)(lds_ptr)dst)),
                 "v"(lane * 16), "s"(rsrc)
                 : "memory", "m0");
}

// this lane's row of 32 in a tile, as the base that Tile::add takes with an even chunk number C (the lane half reads chunk C + hh)
template <typename T, int HD>
__device__ __forceinline__ int row_base(int lane) {
  return Tile<T, HD>::at(lane & 31, lane >> 5);
}

// the lane's place in transposed reads of 32 rows x 32 columns (see columns_frag): bf16 reads 4 x 16 blocks (lane group gq = lane >> 4
// reads rows .. + tq, columns 16 (gq & 1) ..), fp32 single values
template <typename T, int HD>
struct ColBase {
  int lo, hi;
  __device__ __forceinline__ ColBase(int lane) {
    using L = Tile<T, HD>;
    if constexpr (sizeof(T) == 2) {
      const int gq = lane >> 4, tq = (lane & 15) >> 2, tp = lane & 3, c = 2 * (gq & 1) + (tp >> 1), in = 8 * (tp & 1);
      lo = L::at(4 * (gq >> 1) + tq, c) + in;
      hi = L::at(8 + 4 * (gq >> 1) + tq, c) + in;
    } else {
      lo = hi = L::at(4 * (lane >> 5), (lane & 31) >> 2) + (lane & 3) * 4;
    }
  }
};

// acc[column of the tile][lane's column of X] += sum over rows [row0, row0 + 32) of tile[row][..] X[row][..] for the 32 columns that
// start at chunk C (a multiple of 4 chunks in bf16, 8 in fp32); rest: X's second operand, if any
template <typename T, int HD, typename... Rest>
__device__ __forceinline__ f32x16 columns_product(const char* tile, const ColBase<T, HD>& cb, int row0, int C, const Operand& x, f32x16 acc,
                                                  const Rest&... rest) {
  using L = Tile<T, HD>;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const char* p = tile + (row0 + 16 * s) * L::PITCH;
      const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_ptr)(p + L::add(cb.lo, C)));
      const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_ptr)(p + L::add(cb.hi, C)));
      const bf16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, x.p[s], acc, 0, 0, 0);
      ((acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, rest.p[s], acc, 0, 0, 0)), ...);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      constexpr int M = L::MASK;                                     // 15: fp32 rows are multiples of 256 bytes
      const int swz = ((e & 3) << 2) | (3 * ((e >> 2) & 1));           // f(row_of(e, hh)) = swz ^ f(4 hh)
      const char* p = tile + (row0 + (e & 3) + 8 * (e >> 2)) * L::PITCH;
      const float v = *reinterpret_cast<const float*>(p + (cb.lo ^ (((C ^ swz) & M) << 4)) + ((C & ~M) << 4));
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(v, x.f[e], acc, 0, 0, 0);
    }
  }
  return acc;
}

// bf16: the 32 columns from chunk C of 16 rows of a tile as such a product's left operand; lo, hi: ColBase, moved to the rows
template <int HD>
__device__ __forceinline__ bf16x8 columns_frag(const char* tile, int lo, int hi, int C) {
  using L = Tile<bf16_t, HD>;
  const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_ptr)(tile + L::add(lo, C)));
  const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_ptr)(tile + L::add(hi, C)));
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// everything this wave has asked of memory and LDS is there, then everyone's is
template <int LEFT>
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LEFT) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// workgroup -> (pair, block of the pair).  All blocks of a (sample, head) on one XCD (workgroups go round them), whose L2 then holds the
// rows they share, and the pairs dealt out in turn: samples of different lengths spread over the XCDs.  The last pairs % 8 are not.
__device__ __forceinline__ void xcd_block(int id, int n, int per_pair, int* pair, int* block) {
  const int whole = n / per_pair / 8 * 8 * per_pair, j = id < whole ? id >> 3 : id;
  const int p = j / per_pair;
  *pair = id < whole ? p * 8 + (id & 7) : p;
  *block = j - p * per_pair;
}

// max / sum over the two lanes that hold one column of a 32 x 32 accumulator
__device__ __forceinline__ float col_max(float v) { return fmaxf(v, __shfl_xor(v, 32, 64)); }
__device__ __forceinline__ float col_sum(float v) { return v + __shfl_xor(v, 32, 64); }

}  // namespace diffattn
