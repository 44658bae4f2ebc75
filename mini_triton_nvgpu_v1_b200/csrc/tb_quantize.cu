// tb_quantize.cu — 8-bit operands with a scale per block of 128.
//
//   m = max(max |block|, 448 · 2^-63)     S = m / 448     Q = e4m3(448 · X / m)
//
// Blocks are 1 × 128 (a row's scale along k), 128 × 1 (a column's, for
// operands whose rows are k) or 128 × 128. 448 is the largest e4m3 value, so
// a block's largest element lands on it. The floor of m keeps every scale at
// 2^-63 or above: the product of two scales is then a normal f32.
//
// HBM bound: el + 1 bytes per element and nothing read twice. A CTA takes a
// 128 × 128 tile, which is whole blocks in all three shapes; a thread holds 8
// columns of 8 rows in registers (all 8 loads in flight at once: 32 KB per
// CTA of 16-bit inputs), the maxima meet through shuffles and, for blocks
// that span rows, 4 KB of shared memory.
//
// The quotient 448 X / m has to be rounded as the division rounds it: X and m
// are often multiples of each other's last places, so quotients that lie on
// the border of two e4m3 values exactly are common (1 of 400 in bf16), and a
// product with a rounded 1 / m would send them either way. One residual step
// (Markstein, 1990: q' = q + r·(a − b·q), r = 1 / b) gives the division's
// result for two more multiply-adds per element. 448 and m enter as 0.4375
// and m / 1024: 0.4375 X is exact for 16-bit X and never overflows.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "tb_plan.h"

namespace {

constexpr float kLeastMax = 448.f * 1.0842021724855044e-19f;  // 448 · 2^-63

struct QParams {
  const void* x;
  uint8_t* q;
  float* s;
  int64_t ldx, ldq, batch_x, batch_q, batch_s, s_row, s_col;  // elements
  int64_t rows, cols;
  int32_t tiles_r, tiles_c;
  int32_t vec_x, vec_q;
};

__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
struct In;
template <>
struct In<float> {
  static __device__ __forceinline__ float one(const float* p) { return __ldcs(p); }
  static __device__ __forceinline__ void eight(const float* p, float (&v)[8]) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
};
template <>
struct In<__half> {
  static __device__ __forceinline__ float one(const __half* p) {
    return __half2float(__ushort_as_half(__ldcs(reinterpret_cast<const unsigned short*>(p))));
  }
  static __device__ __forceinline__ void eight(const __half* p, float (&v)[8]) {
    const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __half2 h;
      memcpy(&h, &w[i], 4);
      const float2 f = __half22float2(h);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};
template <>
struct In<__nv_bfloat16> {
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) {
    return __uint_as_float((uint32_t)__ldcs(reinterpret_cast<const unsigned short*>(p)) << 16);
  }
  static __device__ __forceinline__ void eight(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

// BR × BC: the block's extent, 1 × 128, 128 × 1 or 128 × 128.
template <typename T, int BR, int BC>
__global__ void __launch_bounds__(256) tb_quantize_kernel(const QParams p) {
  __shared__ float part[8][128];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t per = (int64_t)p.tiles_r * p.tiles_c;
  const int64_t b = blockIdx.x / per;
  const int32_t u = (int32_t)(blockIdx.x - b * per);
  const int32_t tr = u / p.tiles_c, tc = u - tr * p.tiles_c;
  const int64_t r0 = (int64_t)tr * 128 + ty, c0 = (int64_t)tc * 128 + tx * 8;
  const int ncol = (int)min((int64_t)8, max((int64_t)0, p.cols - c0));
  const T* x = static_cast<const T*>(p.x) + b * p.batch_x + c0;

  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + 16 * i;
    if (r < p.rows && ncol == 8 && p.vec_x) {
      In<T>::eight(x + r * p.ldx, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = r < p.rows && j < ncol ? In<T>::one(x + r * p.ldx + j) : 0.f;
    }
  }

  // block maxima: of row i (BR = 1), of column j (BC = 1), or of all
  float m[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) m[i] = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float& d = m[BR == 1 ? i : j];
      d = max_nan(d, fabsf(v[i][j]));
    }
  if constexpr (BR == 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int d = 8; d > 0; d /= 2) m[i] = max_nan(m[i], __shfl_xor_sync(0xffffffffu, m[i], d));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = max_nan(m[j], __shfl_xor_sync(0xffffffffu, m[j], 16));
    if constexpr (BC == 128) {
#pragma unroll
      for (int j = 1; j < 8; ++j) m[0] = max_nan(m[0], m[j]);
#pragma unroll
      for (int d = 8; d > 0; d /= 2) m[0] = max_nan(m[0], __shfl_xor_sync(0xffffffffu, m[0], d));
      if (lane == 0) part[warp][0] = m[0];
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 8; ++w) m[0] = max_nan(m[0], part[w][0]);
    } else {
      if (lane < 16) {
#pragma unroll
        for (int j = 0; j < 8; j += 4)
          *reinterpret_cast<float4*>(&part[warp][tx * 8 + j]) = make_float4(m[j], m[j + 1], m[j + 2], m[j + 3]);
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 8; ++w)
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          const float4 f = *reinterpret_cast<const float4*>(&part[w][tx * 8 + j]);
          m[j] = max_nan(m[j], f.x);
          m[j + 1] = max_nan(m[j + 1], f.y);
          m[j + 2] = max_nan(m[j + 2], f.z);
          m[j + 3] = max_nan(m[j + 3], f.w);
        }
    }
  }
  constexpr int kMaxima = BR == 128 && BC == 128 ? 1 : 8;
#pragma unroll
  for (int i = 0; i < kMaxima; ++i) m[i] = max_nan(m[i], kLeastMax);

  float* s = p.s + b * p.batch_s;
  if constexpr (BR == 1) {
    if (tx == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (r0 + 16 * i < p.rows) s[(r0 + 16 * i) * p.s_row + (int64_t)tc * p.s_col] = m[i] / 448.f;
    }
  } else if constexpr (BC == 1) {
    if (ty == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < ncol) s[(int64_t)tr * p.s_row + (c0 + j) * p.s_col] = m[j] / 448.f;
    }
  } else {
    if (threadIdx.x == 0) s[(int64_t)tr * p.s_row + (int64_t)tc * p.s_col] = m[0] / 448.f;
  }

  float rcp[kMaxima], den[kMaxima];
#pragma unroll
  for (int i = 0; i < kMaxima; ++i) {
    const float d = m[i] * 0.0009765625f;  // m / 1024
    rcp[i] = __frcp_rn(d);
    den[i] = isinf(d) ? 0.f : d;         // an infinite block: 0, and NaN for the infinities (as X / m)
  }
  uint8_t* q = p.q + b * p.batch_q + c0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + 16 * i;
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t two[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float2 f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = 4 * h + 2 * k + e;
          const int g = kMaxima == 1 ? 0 : BR == 1 ? i : j;
          const float y = v[i][j] * 0.4375f;
          const float t = y * rcp[g];
          (e ? f.y : f.x) = fmaf(fmaf(-t, den[g], y), rcp[g], t);
        }
        two[k] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
      }
      w[h] = two[0] | (two[1] << 16);
    }
    if (r >= p.rows) continue;
    if (ncol == 8 && p.vec_q) {
      *reinterpret_cast<uint2*>(q + r * p.ldq) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < ncol) q[r * p.ldq + j] = (uint8_t)(w[j / 4] >> (8 * (j % 4)));
    }
  }
}

template <typename T>
cudaError_t launch_q(const QParams& p, int br, int bc, unsigned grid, cudaStream_t st) {
  if (br == 1) tb_quantize_kernel<T, 1, 128><<<grid, 256, 0, st>>>(p);
  else if (bc == 1) tb_quantize_kernel<T, 128, 1><<<grid, 256, 0, st>>>(p);
  else tb_quantize_kernel<T, 128, 128><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace

extern "C" tbStatus tb_quantize_blocks(const tb_quantize_desc* d, const void* X, int64_t ldx, int64_t stride_x,
                                       void* Q, int64_t ldq, int64_t stride_q, float* S, int64_t stride_s,
                                       int64_t s_row, int64_t s_col, void* stream) {
  tb_clear_error();
  if (!d) return tb_fail(TB_ERR_INVALID_ARGUMENT, "desc must not be NULL");
  if (d->batch < 0 || d->rows < 0 || d->cols < 0)
    return tb_fail(TB_ERR_INVALID_ARGUMENT, "batch, rows and cols must not be negative");
  if (!((d->block_rows == 1 && d->block_cols == 128) || (d->block_rows == 128 && d->block_cols == 1) ||
        (d->block_rows == 128 && d->block_cols == 128)))
    return tb_fail(TB_ERR_INVALID_ARGUMENT, "blocks are 1 x 128, 128 x 1 or 128 x 128");
  if (d->x_dtype != TB_F32 && d->x_dtype != TB_F16 && d->x_dtype != TB_BF16)
    return tb_fail(TB_ERR_INVALID_ARGUMENT, "the input must be f32, f16 or bf16");
  if (d->batch == 0 || d->rows == 0 || d->cols == 0) return TB_OK;
  if (!X || !Q || !S) return tb_fail(TB_ERR_INVALID_ARGUMENT, "X, Q and S must not be NULL");
  if (d->rows > 1 && (ldx < d->cols || ldq < d->cols))
    return tb_fail(TB_ERR_INVALID_ARGUMENT, "leading dimensions must be >= the row length");
  const int el = d->x_dtype == TB_F32 ? 4 : 2;
  const uintptr_t xa = reinterpret_cast<uintptr_t>(X), qa = reinterpret_cast<uintptr_t>(Q);
  if (xa % el || reinterpret_cast<uintptr_t>(S) % 4)
    return tb_fail(TB_ERR_INVALID_ARGUMENT, "X and S must be aligned to their element sizes");
  const int64_t tr = (d->rows + 127) / 128, tc = (d->cols + 127) / 128;
  if (tr > INT32_MAX || tc > INT32_MAX || tr * tc > INT32_MAX || tr * tc * d->batch > INT32_MAX)
    return tb_fail(TB_ERR_UNSUPPORTED, "the matrix has too many blocks");
  QParams p;
  p.x = X;
  p.q = static_cast<uint8_t*>(Q);
  p.s = S;
  p.ldx = ldx;
  p.ldq = ldq;
  p.batch_x = stride_x;
  p.batch_q = stride_q;
  p.batch_s = stride_s;
  p.s_row = s_row;
  p.s_col = s_col;
  p.rows = d->rows;
  p.cols = d->cols;
  p.tiles_r = (int32_t)tr;
  p.tiles_c = (int32_t)tc;
  p.vec_x = xa % 16 == 0 && (d->rows == 1 || ldx * el % 16 == 0) && (d->batch == 1 || stride_x * el % 16 == 0);
  p.vec_q = qa % 8 == 0 && (d->rows == 1 || ldq % 8 == 0) && (d->batch == 1 || stride_q % 8 == 0);
  const unsigned grid = (unsigned)(tr * tc * d->batch);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int br = (int)d->block_rows, bc = (int)d->block_cols;
  const cudaError_t e = d->x_dtype == TB_F32   ? launch_q<float>(p, br, bc, grid, st)
                        : d->x_dtype == TB_F16 ? launch_q<__half>(p, br, bc, grid, st)
                                               : launch_q<__nv_bfloat16>(p, br, bc, grid, st);
  if (e != cudaSuccess) return tb_fail(TB_ERR_CUDA, std::string("tb_quantize launch: ") + cudaGetErrorString(e));
  return TB_OK;
}
