// RMS norm of the residual stream with the residual's addition and its dropout, forward and backward:
//   x = resid + drop(h),  rho = (mean x^2 + eps)^-1/2,  y = x rho w            (stands beside layernorm_kernel of norm.hip)
//   dx = gx + rho (w gy) - x rho^3 mean(w gy x),  dresid = dx,  dh = drop(dx),  dw = sum_rows gy x rho
// HBM-bound: every operand once.  A row stays in registers between its sum and its use; the mask is drawn again in the backward.
// 13312 x 2048, bf16 h and y, fp32 stream: forward 59 us (327 MB, 5.5 TB/s), backward 84 (436 MB, 5.2) and 5 for dw's partial rows;
// 8320 x 1536 to 8 bits 27 us (141 MB, 5.2).
#include "philox.h"

// the addition, the product x * rho and the product with w are rounded one by one, as separate tensor operations round them: the
// 8-bit rounding and the stored stream then meet their ties at the same values
#pragma clang fp contract(off)

namespace {

// ------------------------------------------------------------------------------------------------------------- 8-bit blocks
// E8M0 byte of a block of 32: the smallest e with amax <= 448 * 2^e, biased by 127.  448 = 1.75 * 2^8: with amax = 1.f * 2^(E - 127)
// that is E - 127 - 8 (+ 1 where 1.f > 1.75), i.e. byte E - 8 (+ 1).  0 (2^-127) for zeros, subnormals and whatever lies below.
__device__ __forceinline__ uint32_t mx_scale_byte(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)(e > 0 ? e : 0);
}
// 2^-(byte - 127); byte <= 247
__device__ __forceinline__ float mx_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// four e4m3 values.  |t| <= 448 for every finite t here; Inf and NaN become NaN (0x7f)
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return (uint32_t)w;
}
__device__ __forceinline__ float finite_or_nan(float t) { return fabsf(t) <= 448.f ? t : __uint_as_float(0x7fc00000u); }

struct Fwd {
  const void *h, *resid;
  void *x, *y;
  const float* w;
  uint8_t* scales;
  float* rho;
  int64_t ldh, ldr, ldx, ldy, rows, d;
  float eps, inv_d;
  DropoutRng rng;
  int64_t first;                // row of this launch's first workgroup
};

__device__ __forceinline__ float4 sq4(const float (&v)[8]) {
  return make_float4(v[0] * v[0] + v[4] * v[4], v[1] * v[1] + v[5] * v[5], v[2] * v[2] + v[6] * v[6], v[3] * v[3] + v[7] * v[7]);
}

// sum over the W waves of a workgroup (one row)
template <int W>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < W; ++i) v += red[i];
  }
  return v;
}

// Vector path: 8 | d, 16-byte aligned rows, d <= 512 W NC.  One workgroup of W waves per row; a lane owns NC groups of 8 columns (one
// Philox block each).  W = ceil(d / 512), so that few lanes idle and a lane holds little: the waves in flight hide the row's one
// round trip (a wave per row, 3 - 4 groups per lane: 13312 x 2048 training 71 -> 60 us, 8-bit 8320 x 1536 30.4 -> 28.3 us).
// H: type of h and of y (unless MX); X: type of the stream.
template <typename H, typename X, bool MX, int NC, int W>
__global__ __launch_bounds__(64 * W) void add_rmsnorm_kernel(Fwd a) {
  __shared__ float red[W];
  constexpr int LANES = 64 * W;
  const int lane = threadIdx.x;
  const int64_t row = a.first + blockIdx.x;
  const int n8 = (int)(a.d >> 3);
  const X* rr = (const X*)a.resid + row * a.ldr;
  float x[NC][8];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = lane + LANES * i;
    if (c < n8) load8(rr + c * 8, x[i]);
    else
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = 0.f;
  }
  if (a.h) {
    const H* hr = (const H*)a.h + row * a.ldh;
    X* xr = (X*)a.x + row * a.ldx;
    const uint64_t off = a.rng.thr ? dropout_offset(a.rng) : 0;
    float h[NC][8];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + LANES * i;
      if (c < n8) load8(hr + c * 8, h[i]);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + LANES * i;
      if (c < n8) {
        const uint32_t keep = a.rng.thr ? dropout_keep8(a.rng, off, (uint64_t)(row * n8 + c)) : 0xffu;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] += (keep >> j) & 1u ? h[i][j] * a.rng.scale : 0.f;
        store8(xr + c * 8, x[i]);
        if constexpr (sizeof(X) == 2) {                          // the norm reads the stream as it is stored
#pragma unroll
          for (int j = 0; j < 8; ++j) x[i][j] = bf16_to_f32(f32_to_bf16(x[i][j]));
        }
      }
    }
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const float4 q = sq4(x[i]);
    s += (q.x + q.y) + (q.z + q.w);
  }
  const float rho = 1.0f / sqrtf(row_sum<W>(s, red) * a.inv_d + a.eps);
  if (a.rho && lane == 0) a.rho[row] = rho;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = lane + LANES * i;
    const bool in = c < n8;
    float y[8];
    if (in) load8(a.w + c * 8, y);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = in ? x[i][j] * rho * y[j] : 0.f;
    if constexpr (MX) {
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(y[j]));
      m = fmaxf(m, __shfl_xor(m, 1, 64));                        // a block of 32 columns = 4 neighbouring lanes
      m = fmaxf(m, __shfl_xor(m, 2, 64));
      const uint32_t byte = mx_scale_byte(m);
      const float inv = mx_inverse(byte);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = finite_or_nan(y[j] * inv);
      if (in) {
        uint2 q;
        q.x = e4m3x4(y[0], y[1], y[2], y[3]);
        q.y = e4m3x4(y[4], y[5], y[6], y[7]);
        *reinterpret_cast<uint2*>((uint8_t*)a.y + row * a.ldy + c * 8) = q;
        if ((lane & 3) == 0) a.scales[row * (a.d >> 5) + (c >> 2)] = (uint8_t)byte;
      }
    } else if (in) {
      store8((H*)a.y + row * a.ldy + c * 8, y);
    }
  }
}

// Any d, alignment and stride: one workgroup per row, element by element; the second sweep reads the stream back (from x_out where
// it was written: each thread reads its own columns).
template <typename H, typename X, bool MX>
__global__ __launch_bounds__(256) void add_rmsnorm_any_kernel(Fwd a) {
  __shared__ float red[4];
  const int64_t row = a.first + blockIdx.x;
  const X* rr = (const X*)a.resid + row * a.ldr;
  const uint64_t off = a.rng.thr ? dropout_offset(a.rng) : 0;
  const X* src = rr;
  float s = 0.f;
  if (a.h) {
    const H* hr = (const H*)a.h + row * a.ldh;
    X* xr = (X*)a.x + row * a.ldx;
    src = xr;
    for (int64_t c = threadIdx.x; c < a.d; c += 256) {
      const bool keep = !a.rng.thr || dropout_keep1(a.rng, off, (uint64_t)(row * a.d + c));
      const float v = elem<X>::load(rr + c) + (keep ? elem<H>::load(hr + c) * a.rng.scale : 0.f);
      elem<X>::store(xr + c, v);
      const float t = elem<X>::load(xr + c);
      s += t * t;
    }
  } else {
    for (int64_t c = threadIdx.x; c < a.d; c += 256) {
      const float t = elem<X>::load(rr + c);
      s += t * t;
    }
  }
  const float rho = 1.0f / sqrtf(row_sum<4>(s, red) * a.inv_d + a.eps);
  if (a.rho && threadIdx.x == 0) a.rho[row] = rho;
  // MX: 32 | d, so every group of 32 lanes covers one block of 32 columns of the row per sweep, or none
  for (int64_t c = threadIdx.x; c < a.d; c += 256) {
    float y = elem<X>::load(src + c) * rho * a.w[c];
    if constexpr (MX) {
      float m = fabsf(y);
      if (!(m >= 0.f)) m = 0.f;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
      const uint32_t byte = mx_scale_byte(m);
      y = finite_or_nan(y * mx_inverse(byte));
      ((uint8_t*)a.y)[row * a.ldy + c] = (uint8_t)(e4m3x4(y, y, y, y) & 0xffu);
      if ((c & 31) == 0) a.scales[row * (a.d >> 5) + (c >> 5)] = (uint8_t)byte;
    } else {
      elem<H>::store((H*)a.y + row * a.ldy + c, y);
    }
  }
}

constexpr int64_t LAUNCH_ROWS = 1 << 23;   // a workgroup per row: a grid of at most 2^32 threads

template <typename H, typename X, bool MX>
int launch_fwd(Fwd a, bool vec, hipStream_t s) {
  for (a.first = 0; a.first < a.rows; a.first += LAUNCH_ROWS) {
    const dim3 grid((unsigned)(a.rows - a.first < LAUNCH_ROWS ? a.rows - a.first : LAUNCH_ROWS));
#define RN(NC, W) hipLaunchKernelGGL((add_rmsnorm_kernel<H, X, MX, NC, W>), grid, dim3(64 * W), 0, s, a)
    if (!vec || a.d > 8192) hipLaunchKernelGGL((add_rmsnorm_any_kernel<H, X, MX>), grid, dim3(256), 0, s, a);
    else if (a.d <= 512) RN(1, 1);
    else if (a.d <= 1024) RN(1, 2);
    else if (a.d <= 1536) RN(1, 3);
    else if (a.d <= 2048) RN(1, 4);
    else if (a.d <= 4096) RN(2, 4);
    else RN(4, 4);
#undef RN
    if (int st = gpt_launch_status("gpt_add_rmsnorm")) return st;
  }
  return 0;
}

// ---------------------------------------------------------------------------------------------------------------- backward
struct Bwd {
  const void *gy, *gx, *x;
  const float *w, *rho;
  void *dresid, *dh;
  float* part;                  // [gridDim.x][d] column sums of the workgroups, or NULL
  int64_t ldgy, ldgx, ldx, lddr, lddh, rows, d;
  float inv_d;
  DropoutRng rng;
};

// rho^3 m, m = mean(w gy x): from m, which is of the order of 1 / rho, up - rho^3 alone leaves the range of fp32 where the rows are below
// 1e-13 or above 1e13
__device__ __forceinline__ float cube_scaled(float rho, float m) { return rho * (rho * (rho * m)); }

constexpr int BWD_BLOCKS = 768;  // workgroups at most: rows are dealt out round robin, each keeps its columns' dw sums in registers

// Vector path, one workgroup of W waves per row at a time
template <typename H, typename X, int NC, int W>
__global__ __launch_bounds__(64 * W) void add_rmsnorm_bwd_kernel(Bwd a) {
  __shared__ float red[W];
  constexpr int LANES = 64 * W;
  const int lane = threadIdx.x;
  const int n8 = (int)(a.d >> 3);
  const uint64_t off = a.rng.thr ? dropout_offset(a.rng) : 0;
  float dw[NC][8];
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = 0.f;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float x[NC][8], t[NC][8], g[NC][8];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + LANES * i;
      if (c < n8) {
        load8((const X*)a.x + row * a.ldx + c * 8, x[i]);
        load8((const H*)a.gy + row * a.ldgy + c * 8, t[i]);
        if (a.gx) load8((const X*)a.gx + row * a.ldgx + c * 8, g[i]);
      }
    }
    const float rho = a.rho[row];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + LANES * i;
      if (c < n8) {
        float w[8];
        load8(a.w + c * 8, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          dw[i][j] += t[i][j] * (x[i][j] * rho);
          t[i][j] *= w[j];
          s += t[i][j] * x[i][j];
        }
      }
    }
    if constexpr (W > 1) __syncthreads();                         // the previous row's sums have been read
    const float k = cube_scaled(rho, row_sum<W>(s, red) * a.inv_d);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + LANES * i;
      if (c < n8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = t[i][j] * rho - x[i][j] * k;
          t[i][j] = a.gx ? g[i][j] + v : v;
        }
        store8((X*)a.dresid + row * a.lddr + c * 8, t[i]);
        if (a.dh) {
          const uint32_t keep = a.rng.thr ? dropout_keep8(a.rng, off, (uint64_t)(row * n8 + c)) : 0xffu;
#pragma unroll
          for (int j = 0; j < 8; ++j) t[i][j] = (keep >> j) & 1u ? t[i][j] * a.rng.scale : 0.f;
          store8((H*)a.dh + row * a.lddh + c * 8, t[i]);
        }
      }
    }
  }
  if (!a.part) return;
  float* out = a.part + (int64_t)blockIdx.x * a.d;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = lane + LANES * i;
    if (c < n8) store8(out + c * 8, dw[i]);
  }
}

// Any d, alignment and stride: a workgroup per row at a time; a thread's columns of the workgroup's partial row are read, added to
// and written back by that thread alone
template <typename H, typename X>
__global__ __launch_bounds__(256) void add_rmsnorm_bwd_any_kernel(Bwd a) {
  __shared__ float red[4];
  const uint64_t off = a.rng.thr ? dropout_offset(a.rng) : 0;
  float* part = a.part ? a.part + (int64_t)blockIdx.x * a.d : nullptr;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const X* xr = (const X*)a.x + row * a.ldx;
    const H* gyr = (const H*)a.gy + row * a.ldgy;
    const X* gxr = a.gx ? (const X*)a.gx + row * a.ldgx : nullptr;
    const float rho = a.rho[row];
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < a.d; c += 256) {
      const float x = elem<X>::load(xr + c), gy = elem<H>::load(gyr + c);
      s += gy * a.w[c] * x;
      if (part) part[c] = (row == (int64_t)blockIdx.x ? 0.f : part[c]) + gy * (x * rho);
    }
    __syncthreads();
    const float k = cube_scaled(rho, row_sum<4>(s, red) * a.inv_d);
    for (int64_t c = threadIdx.x; c < a.d; c += 256) {
      const float x = elem<X>::load(xr + c), gy = elem<H>::load(gyr + c);
      float v = gy * a.w[c] * rho - x * k;
      if (gxr) v = elem<X>::load(gxr + c) + v;
      elem<X>::store((X*)a.dresid + row * a.lddr + c, v);
      if (a.dh) {
        const bool keep = !a.rng.thr || dropout_keep1(a.rng, off, (uint64_t)(row * a.d + c));
        elem<H>::store((H*)a.dh + row * a.lddh + c, keep ? v * a.rng.scale : 0.f);
      }
    }
  }
}

// out[c] = sum over the partial rows in index order, within 16 interleaved groups and then over the groups
__global__ __launch_bounds__(1024) void rmsnorm_dw_kernel(const float* __restrict__ part, int n, float* __restrict__ out, int64_t d) {
  __shared__ float red[16][64];
  const int64_t c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const int grp = threadIdx.x >> 6;
  float s = 0.f;
  if (c < d) {
#pragma unroll 8
    for (int r = grp; r < n; r += 16) s += part[(int64_t)r * d + c];
  }
  red[grp][threadIdx.x & 63] = s;
  __syncthreads();
  if (grp == 0 && c < d) {
#pragma unroll
    for (int q = 1; q < 16; ++q) s += red[q][threadIdx.x];
    out[c] = s;
  }
}

template <typename H, typename X>
int launch_bwd(const Bwd& a, bool vec, float* dweight, hipStream_t s) {
  const int nb = (int)(a.rows < BWD_BLOCKS ? a.rows : BWD_BLOCKS);
#define RB(NC, W) hipLaunchKernelGGL((add_rmsnorm_bwd_kernel<H, X, NC, W>), dim3(nb), dim3(64 * W), 0, s, a)
  if (!vec || a.d > 8192) hipLaunchKernelGGL((add_rmsnorm_bwd_any_kernel<H, X>), dim3(nb), dim3(256), 0, s, a);
  else if (a.d <= 512) RB(1, 1);
  else if (a.d <= 1024) RB(1, 2);
  else if (a.d <= 1536) RB(1, 3);
  else if (a.d <= 2048) RB(1, 4);
  else if (a.d <= 4096) RB(2, 4);
  else RB(4, 4);
#undef RB
  if (int st = gpt_launch_status("gpt_add_rmsnorm_bwd")) return st;
  if (dweight) {
    hipLaunchKernelGGL(rmsnorm_dw_kernel, dim3((unsigned)((a.d + 63) / 64)), dim3(1024), 0, s, a.part, nb, dweight, a.d);
    return gpt_launch_status("gpt_add_rmsnorm_bwd");
  }
  return 0;
}

bool fp_dtype(int t) { return t == GPT_F32 || t == GPT_BF16; }
size_t fp_size(int t) { return t == GPT_BF16 ? 2 : 4; }
bool elem_aligned(const void* p, size_t es) { return (uintptr_t)p % es == 0; }

}  // namespace

extern "C" int gpt_add_rmsnorm(const gpt_add_rmsnorm_t* p, void* stream) {
  const char* who = "gpt_add_rmsnorm";
  GPT_REQUIRE(p, "%s: null descriptor", who);
  const bool mx = p->y_dtype == GPT_MXFP8;
  GPT_REQUIRE(fp_dtype(p->h_dtype) && fp_dtype(p->x_dtype) && (mx || fp_dtype(p->y_dtype)), "%s: bad dtype (%d, %d, %d)", who, p->h_dtype,
              p->x_dtype, p->y_dtype);
  GPT_REQUIRE(p->resid && p->weight && p->y && (!p->h || p->x_out), "%s: null operand", who);
  GPT_REQUIRE(p->rows > 0 && p->d > 0 && p->rows <= INT64_MAX / 8 / p->d && p->d < (1ll << 31), "%s: bad size (rows=%lld d=%lld)", who,
              (long long)p->rows, (long long)p->d);
  GPT_REQUIRE(!mx || (p->d % 32 == 0 && p->scales), "%s: 8-bit output needs d %% 32 == 0 and a scales buffer (d=%lld)", who, (long long)p->d);
  GPT_REQUIRE(mx || !p->h || p->y_dtype == p->h_dtype, "%s: y has the type of h (%d, %d)", who, p->y_dtype, p->h_dtype);
  GPT_REQUIRE(p->eps >= 0.f, "%s: eps %g < 0", who, p->eps);
  GPT_REQUIRE(p->rows == 1 || ((!p->h || p->ldh >= 0) && p->ldr >= 0 && (!p->h || p->ldx >= p->d) && p->ldy >= p->d), "%s: bad row stride", who);
  const size_t hs = fp_size(mx ? p->h_dtype : p->y_dtype), xs = fp_size(p->x_dtype), ys = mx ? 1 : hs;
  GPT_REQUIRE(elem_aligned(p->h, hs) && elem_aligned(p->resid, xs) && elem_aligned(p->x_out, xs) && elem_aligned(p->weight, 4) &&
                  elem_aligned(p->y, ys) && elem_aligned(p->rho, 4),
              "%s: misaligned element", who);
  Fwd a{p->h, p->resid, p->x_out, p->y, p->weight, p->scales, p->rho, p->ldh, p->ldr, p->ldx, p->ldy, p->rows, p->d, p->eps, 1.0f / (float)p->d, {}, 0};
  if (int st = gpt_dropout_rng(p->drop, &a.rng, who)) return st;
  const bool vec = p->d % 8 == 0 && rows_aligned16(p->resid, p->ldr, xs) && aligned16(p->weight) &&
                   (!p->h || (rows_aligned16(p->h, p->ldh, hs) && rows_aligned16(p->x_out, p->ldx, xs))) &&
                   (mx ? ((uintptr_t)p->y % 8 == 0 && p->ldy % 8 == 0) : rows_aligned16(p->y, p->ldy, hs));
  hipStream_t s = (hipStream_t)stream;
  const int ht = mx ? p->h_dtype : p->y_dtype;
#define GO(H, X) (mx ? launch_fwd<H, X, true>(a, vec, s) : launch_fwd<H, X, false>(a, vec, s))
  if (ht == GPT_BF16) return p->x_dtype == GPT_BF16 ? GO(bf16_t, bf16_t) : GO(bf16_t, float);
  return p->x_dtype == GPT_BF16 ? GO(float, bf16_t) : GO(float, float);
#undef GO
}

static int64_t bwd_workspace(int64_t rows, int64_t d) { return (rows < BWD_BLOCKS ? rows : BWD_BLOCKS) * d * (int64_t)sizeof(float); }

extern "C" int gpt_add_rmsnorm_bwd_workspace(int64_t rows, int64_t d, int64_t* host_bytes) {
  GPT_REQUIRE(host_bytes && rows > 0 && d > 0 && d < (1ll << 31), "gpt_add_rmsnorm_bwd_workspace: bad arguments");
  *host_bytes = bwd_workspace(rows, d);
  return 0;
}

extern "C" int gpt_add_rmsnorm_bwd(const gpt_add_rmsnorm_bwd_t* p, void* stream) {
  const char* who = "gpt_add_rmsnorm_bwd";
  GPT_REQUIRE(p, "%s: null descriptor", who);
  GPT_REQUIRE(fp_dtype(p->h_dtype) && fp_dtype(p->x_dtype) && fp_dtype(p->y_dtype), "%s: bad dtype (%d, %d, %d)", who, p->h_dtype, p->x_dtype,
              p->y_dtype);
  GPT_REQUIRE(p->gy && p->x && p->weight && p->rho && p->dresid, "%s: null operand", who);
  GPT_REQUIRE(!p->dh || p->h_dtype == p->y_dtype, "%s: dh has the type of gy (%d, %d)", who, p->h_dtype, p->y_dtype);
  GPT_REQUIRE(p->rows > 0 && p->d > 0 && p->rows <= INT64_MAX / 8 / p->d && p->d < (1ll << 31), "%s: bad size (rows=%lld d=%lld)", who,
              (long long)p->rows, (long long)p->d);
  GPT_REQUIRE(p->rows == 1 || (p->ldgy >= 0 && (!p->gx || p->ldgx >= 0) && p->ldx >= 0 && p->lddr >= p->d && (!p->dh || p->lddh >= p->d)),
              "%s: bad row stride", who);
  GPT_REQUIRE(!p->dweight || (p->ws && aligned16(p->ws) && p->ws_bytes >= bwd_workspace(p->rows, p->d)),
              "%s: the weight gradient needs %lld bytes of scratch", who, (long long)bwd_workspace(p->rows, p->d));
  const size_t hs = fp_size(p->y_dtype), xs = fp_size(p->x_dtype);
  GPT_REQUIRE(elem_aligned(p->gy, hs) && elem_aligned(p->gx, xs) && elem_aligned(p->x, xs) && elem_aligned(p->weight, 4) &&
                  elem_aligned(p->rho, 4) && elem_aligned(p->dresid, xs) && elem_aligned(p->dh, hs) && elem_aligned(p->dweight, 4),
              "%s: misaligned element", who);
  Bwd a{p->gy, p->gx, p->x, p->weight, p->rho, p->dresid, p->dh, p->dweight ? (float*)p->ws : nullptr, p->ldgy, p->ldgx, p->ldx, p->lddr,
        p->lddh, p->rows, p->d, 1.0f / (float)p->d, {}};
  if (int st = gpt_dropout_rng(p->drop, &a.rng, who)) return st;
  const bool vec = p->d % 8 == 0 && rows_aligned16(p->gy, p->ldgy, hs) && (!p->gx || rows_aligned16(p->gx, p->ldgx, xs)) &&
                   rows_aligned16(p->x, p->ldx, xs) && aligned16(p->weight) && rows_aligned16(p->dresid, p->lddr, xs) &&
                   (!p->dh || rows_aligned16(p->dh, p->lddh, hs));
  hipStream_t s = (hipStream_t)stream;
  if (p->y_dtype == GPT_BF16)
    return p->x_dtype == GPT_BF16 ? launch_bwd<bf16_t, bf16_t>(a, vec, p->dweight, s) : launch_bwd<bf16_t, float>(a, vec, p->dweight, s);
  return p->x_dtype == GPT_BF16 ? launch_bwd<float, bf16_t>(a, vec, p->dweight, s) : launch_bwd<float, float>(a, vec, p->dweight, s);
}
