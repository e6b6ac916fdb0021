// Dropout from a counter-based generator (philox.h), with the residual's addition:
//   out = resid + keep(i) * h * s          nn.Dropout of Gpt/models/transformer.py:34-72 and the "x + f(x)" of :70-71
// The mask is a function of (seed, offset, element index) alone, so the backward, dh = keep(i) * g * s, is the same kernel on the
// gradient and nothing is stored between the two.
// HBM-bound: read h and resid, write out, once each.  26624 x 1536, bf16 h, fp32 stream: 71 us with the residual (410 MB, 5.8 TB/s),
// 45 the masked gradient (245 MB, 5.5 TB/s); 208 x 1536 4.5 us, a launch.
#include "philox.h"

// h * s and the addition are rounded separately, as two tensor operations round them
#pragma clang fp contract(off)

namespace {

template <typename T>
__device__ __forceinline__ float load1(const T* p) { return elem<T>::load(p); }

__device__ __forceinline__ float drop(float h, bool keep, float s) { return keep ? h * s : 0.f; }   // a select: NaN and Inf are dropped too

// Contiguous operands: the flat index is the element index.  One Philox block = one thread's 8 elements = one 16-byte load per
// bf16 operand, two per fp32 operand.
template <typename H, typename X, bool RES>
__global__ __launch_bounds__(256) void dropout_flat_kernel(const H* h, const X* resid, X* out, int64_t n, DropoutRng r) {
  const uint64_t off = dropout_offset(r);
  const int64_t n8 = n >> 3, stride = (int64_t)gridDim.x * 256;
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int64_t c = first; c < n8; c += stride) {
    float v[8], x[8];
    load8(h + c * 8, v);
    if constexpr (RES) load8(resid + c * 8, x);
    const uint32_t keep = dropout_keep8(r, off, (uint64_t)c);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float t = drop(v[j], (keep >> j) & 1u, r.scale);
      x[j] = RES ? x[j] + t : t;
    }
    store8(out + c * 8, x);
  }
  const int64_t i = n8 * 8 + first;                            // the last n % 8 elements
  if (i < n) {
    const float t = drop(load1(h + i), dropout_keep1(r, off, (uint64_t)i), r.scale);
    elem<X>::store(out + i, RES ? load1(resid + i) + t : t);
  }
}

// Rows with a stride: one workgroup walks rows; VEC: 8 | d and every row 16-byte aligned, else element by element (a Philox block
// per element: eight times the generator's work, for shapes that no vector access fits)
template <typename H, typename X, bool RES, bool VEC>
__global__ __launch_bounds__(256) void dropout_rows_kernel(const H* h, int64_t ldh, const X* resid, int64_t ldr, X* out,
                                                           int64_t ldo, int64_t rows, int64_t d, DropoutRng r) {
  const uint64_t off = dropout_offset(r);
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const H* hr = h + row * ldh;
    const X* rr = RES ? resid + row * ldr : nullptr;
    X* orow = out + row * ldo;
    if constexpr (VEC) {
      for (int64_t c = threadIdx.x; c < (d >> 3); c += 256) {
        float v[8], x[8];
        load8(hr + c * 8, v);
        if constexpr (RES) load8(rr + c * 8, x);
        const uint32_t keep = dropout_keep8(r, off, (uint64_t)(row * (d >> 3) + c));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float t = drop(v[j], (keep >> j) & 1u, r.scale);
          x[j] = RES ? x[j] + t : t;
        }
        store8(orow + c * 8, x);
      }
    } else {
      for (int64_t c = threadIdx.x; c < d; c += 256) {
        const float t = drop(load1(hr + c), dropout_keep1(r, off, (uint64_t)(row * d + c)), r.scale);
        elem<X>::store(orow + c, RES ? load1(rr + c) + t : t);
      }
    }
  }
}

template <typename H, typename X>
int launch(const void* h, int64_t ldh, const void* resid, int64_t ldr, void* out, int64_t ldo, int64_t rows, int64_t d, const DropoutRng& r,
           hipStream_t s) {
  const H* hp = (const H*)h;
  const X* rp = (const X*)resid;
  X* op = (X*)out;
  const bool flat = rows == 1 || (ldh == d && ldo == d && (!resid || ldr == d));
  if (flat && aligned16(h) && aligned16(resid) && aligned16(out)) {
    const int64_t n = rows * d, want = ((n + 7) / 8 + 255) / 256;
    const dim3 grid((unsigned)(want < (1 << 22) ? want : (1 << 22)));
    if (resid) hipLaunchKernelGGL((dropout_flat_kernel<H, X, true>), grid, dim3(256), 0, s, hp, rp, op, n, r);
    else hipLaunchKernelGGL((dropout_flat_kernel<H, X, false>), grid, dim3(256), 0, s, hp, rp, op, n, r);
    return gpt_launch_status("gpt_dropout_add");
  }
  const bool vec = d % 8 == 0 && rows_aligned16(h, ldh, sizeof(H)) && rows_aligned16(out, ldo, sizeof(X)) &&
                   (!resid || rows_aligned16(resid, ldr, sizeof(X)));
  const dim3 grid((unsigned)(rows < (1 << 20) ? rows : (1 << 20)));
#define DR(RES, VEC) hipLaunchKernelGGL((dropout_rows_kernel<H, X, RES, VEC>), grid, dim3(256), 0, s, hp, ldh, rp, ldr, op, ldo, rows, d, r)
  if (resid) { if (vec) DR(true, true); else DR(true, false); }
  else { if (vec) DR(false, true); else DR(false, false); }
#undef DR
  return gpt_launch_status("gpt_dropout_add");
}

}  // namespace

extern "C" int gpt_dropout_add(int h_dtype, const void* h, int64_t ldh, int x_dtype, const void* resid, int64_t ldr, void* out, int64_t ldo,
                               int64_t rows, int64_t d, const gpt_dropout_t* drop, void* stream) {
  GPT_REQUIRE((h_dtype == GPT_F32 || h_dtype == GPT_BF16) && (x_dtype == GPT_F32 || x_dtype == GPT_BF16), "gpt_dropout_add: bad dtype (%d, %d)",
              h_dtype, x_dtype);
  GPT_REQUIRE(drop && h && out, "gpt_dropout_add: null operand");
  GPT_REQUIRE(rows > 0 && d > 0, "gpt_dropout_add: need rows > 0 and d > 0 (rows=%lld d=%lld)", (long long)rows, (long long)d);
  GPT_REQUIRE(rows <= INT64_MAX / 8 / d, "gpt_dropout_add: rows * d too large");
  GPT_REQUIRE((rows == 1 || (ldh >= 0 && ldo >= d && (!resid || ldr >= 0))), "gpt_dropout_add: bad row stride (ldh=%lld ldr=%lld ldo=%lld d=%lld)",
              (long long)ldh, (long long)ldr, (long long)ldo, (long long)d);
  const size_t hs = h_dtype == GPT_BF16 ? 2 : 4, xs = x_dtype == GPT_BF16 ? 2 : 4;
  GPT_REQUIRE((uintptr_t)h % hs == 0 && (uintptr_t)resid % xs == 0 && (uintptr_t)out % xs == 0, "gpt_dropout_add: misaligned element");
  DropoutRng r;
  if (int st = gpt_dropout_rng(drop, &r, "gpt_dropout_add")) return st;
  hipStream_t s = (hipStream_t)stream;
  if (h_dtype == GPT_BF16)
    return x_dtype == GPT_BF16 ? launch<bf16_t, bf16_t>(h, ldh, resid, ldr, out, ldo, rows, d, r, s)
                               : launch<bf16_t, float>(h, ldh, resid, ldr, out, ldo, rows, d, r, s);
  return x_dtype == GPT_BF16 ? launch<float, bf16_t>(h, ldh, resid, ldr, out, ldo, rows, d, r, s)
                             : launch<float, float>(h, ldh, resid, ldr, out, ldo, rows, d, r, s);
}
