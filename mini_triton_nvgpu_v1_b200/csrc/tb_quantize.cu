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
// columns of 8 rows in registers as they were read, all 8 loads in flight at
// once and 32 KB per CTA of 16-bit inputs. The maxima are taken on the bits of
// |x| as unsigned integers (the order of the magnitudes, with NaN above
// infinity, two 16-bit values to an instruction) and meet through shuffles
// and, for blocks that span rows, shared memory.
//
// The quotient 448 X / m has to be rounded as the division rounds it: X and m
// are often multiples of each other's last places, so quotients that lie on
// the border of two e4m3 values exactly are common (1 of 400 in bf16), and a
// product with a rounded 1 / m would send them either way. One residual step
// (Markstein, 1990: q' = q + r·(a − b·q), r = 1 / b) gives the division's
// result for two more multiply-adds per element. 448 and m enter as 0.4375
// and m / 1024: 0.4375 X is exact for 16-bit X and never overflows. Of f32 X it
// is rounded, and the quotient is rounded to f32 before it is to e4m3 (2^-24 and
// 2^-23): one that lies that near to a border may go to either side.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstring>
#include <string>
#include <type_traits>

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

// Two f32 in a register pair.
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Eight values of a row as they are in memory: kWords words of kPer values.
template <typename T>
struct In {
  static constexpr int kPer = 4 / (int)sizeof(T), kWords = 8 / kPer;
  static __device__ __forceinline__ void eight(const T* p, uint32_t (&w)[kWords]) {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p) + i);
      w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
    }
  }
  static __device__ __forceinline__ void some(const T* p, int n, uint32_t (&w)[kWords]) {  // the first n, then zeros
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      w[i] = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int k = i * kPer + j;
        if (k < n) {
          if constexpr (kPer == 1) w[i] = __ldcs(reinterpret_cast<const uint32_t*>(p) + k);
          else w[i] |= (uint32_t)__ldcs(reinterpret_cast<const unsigned short*>(p) + k) << (16 * j);
        }
      }
    }
  }
  static constexpr uint32_t kAbs = kPer == 1 ? 0x7fffffffu : 0x7fff7fffu;
  static __device__ __forceinline__ uint32_t max3(uint32_t a, uint32_t b, uint32_t c) {
    if constexpr (kPer == 1) return __vimax3_u32(a, b, c);
    else return __vimax3_u16x2(a, b, c);
  }
  static __device__ __forceinline__ float value(uint32_t bits) {  // of the low 16 (or all 32) bits
    if constexpr (kPer == 1) return __uint_as_float(bits);
    else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)bits));
    else return __uint_as_float(bits << 16);
  }
  // values 2k and 2k + 1
  static __device__ __forceinline__ uint64_t pair(const uint32_t (&w)[kWords], int k) {
    if constexpr (kPer == 1) {
      return two(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
    } else if constexpr (std::is_same<T, __half>::value) {
      __half2 h;
      memcpy(&h, &w[k], 4);
      const float2 f = __half22float2(h);
      return two(f.x, f.y);
    } else {
      return two(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
    }
  }
};

// BR × BC: the block's extent, 1 × 128, 128 × 1 or 128 × 128. 16-bit inputs:
// at most 64 registers, so that four CTAs (128 KB of loads) are at work on an SM.
template <typename T, int BR, int BC>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2) tb_quantize_kernel(const QParams p) {
  using I = In<T>;
  constexpr int W = I::kWords;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t per = (int64_t)p.tiles_r * p.tiles_c;
  const int64_t b = blockIdx.x / per;
  const int32_t u = (int32_t)(blockIdx.x - b * per);
  const int32_t tr = u / p.tiles_c, tc = u - tr * p.tiles_c;
  const int64_t r0 = (int64_t)tr * 128 + ty, c0 = (int64_t)tc * 128 + tx * 8;
  const int ncol = (int)min((int64_t)8, max((int64_t)0, p.cols - c0));
  const int nrow = (int)min((int64_t)8, max((int64_t)0, (p.rows - r0 + 15) / 16));  // this thread's rows
  const T* x = static_cast<const T*>(p.x) + b * p.batch_x + r0 * p.ldx + c0;
  // Launched while the kernel before it in the stream ends: nothing of memory
  // is touched before that one's writes are there. The next may do the same.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  uint32_t v[8][W];
  if (p.vec_x && (int64_t)tr * 128 + 128 <= p.rows && (int64_t)tc * 128 + 128 <= p.cols) {
#pragma unroll
    for (int i = 0; i < 8; ++i) I::eight(x + 16 * i * p.ldx, v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int n = i < nrow ? ncol : 0;
      if (n == 8 && p.vec_x) I::eight(x + 16 * i * p.ldx, v[i]);
      else I::some(x + 16 * i * p.ldx, n, v[i]);
    }
  }

  // Block maxima, and for the pairs of columns that meet them 1 / d and -d of
  // d = m / 1024: one pair for the block, one for each row, or one for two
  // columns. Each maximum's reciprocal and scale (a division) are worked out
  // by one thread and handed to the others: every thread doing its own eight
  // took as long as the rest of the arithmetic (16384 × 8192 bf16: 1 × 128 blocks 80 µs, 128 × 1 77 µs; now 72 and 68,
  // 128 × 128 63).
  constexpr int kPairs = BR == 1 ? 8 : BC == 1 ? 4 : 1;
  uint64_t rcp[kPairs], neg[kPairs];
  float* s = p.s + b * p.batch_s;
  auto floor_of = [](float m) { return m < kLeastMax ? kLeastMax : m; };  // a NaN stays
  auto den_of = [](float m) { return m * 0.0009765625f; };
  auto neg_of = [](float d) { return isinf(d) ? 0.f : -d; };  // an infinite block: 0, and NaN for the infinities
  if constexpr (BR == 1) {
    uint32_t a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = 0;
#pragma unroll
      for (int j = 0; j < W; j += 2) a[i] = I::max3(a[i], v[i][j] & I::kAbs, v[i][j + 1] & I::kAbs);
    }
    if constexpr (I::kPer == 2) {
      // rows i and i + 1 in one word
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        uint32_t x = __vimax3_u16x2(__byte_perm(a[i], a[i + 1], 0x5410), __byte_perm(a[i], a[i + 1], 0x7632), 0);
#pragma unroll
        for (int d = 8; d > 0; d /= 2) x = I::max3(x, __shfl_xor_sync(0xffffffffu, x, d), 0);
        a[i] = x & 0xffffu;
        a[i + 1] = x >> 16;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int d = 8; d > 0; d /= 2) a[i] = I::max3(a[i], __shfl_xor_sync(0xffffffffu, a[i], d), 0);
    }
    // of row tx mod 8, by halves (an index into a[] would put it into memory)
    const bool t1 = tx & 1, t2 = tx & 2;
    const uint32_t lo = t2 ? (t1 ? a[3] : a[2]) : (t1 ? a[1] : a[0]), hi = t2 ? (t1 ? a[7] : a[6]) : (t1 ? a[5] : a[4]);
    const uint32_t mine = tx & 4 ? hi : lo;
    const float m = floor_of(I::value(mine)), d = den_of(m), r = __frcp_rn(d), n = neg_of(d);
    if (tx < nrow) s[(r0 + 16 * tx) * p.s_row + (int64_t)tc * p.s_col] = m / 448.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float ri = __shfl_sync(0xffffffffu, r, (lane & 16) + i), ni = __shfl_sync(0xffffffffu, n, (lane & 16) + i);
      rcp[i] = two(ri, ri);
      neg[i] = two(ni, ni);
    }
  } else {
    __shared__ __align__(16) uint32_t part[8][16 * W];
    uint32_t a[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
      a[j] = 0;
#pragma unroll
      for (int i = 0; i < 8; i += 2) a[j] = I::max3(a[j], v[i][j] & I::kAbs, v[i + 1][j] & I::kAbs);
      a[j] = I::max3(a[j], __shfl_xor_sync(0xffffffffu, a[j], 16), 0);
    }
    if constexpr (BC == 128) {
#pragma unroll
      for (int j = 1; j < W; ++j) a[0] = I::max3(a[0], a[j], 0);
      if constexpr (I::kPer == 2) a[0] = max(a[0] & 0xffffu, a[0] >> 16);
      a[0] = __reduce_max_sync(0xffffffffu, a[0]);
      if (lane == 0) part[warp][0] = a[0];
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 8; ++w) a[0] = max(a[0], part[w][0]);
      const float m = floor_of(I::value(a[0])), d = den_of(m), r = __frcp_rn(d), n = neg_of(d);
      if (threadIdx.x == 0) s[(int64_t)tr * p.s_row + (int64_t)tc * p.s_col] = m / 448.f;
      rcp[0] = two(r, r);
      neg[0] = two(n, n);
    } else {
      __shared__ __align__(16) float col_rcp[128], col_neg[128];
      if (lane < 16) {
#pragma unroll
        for (int j = 0; j < W; j += 4)
          *reinterpret_cast<uint4*>(&part[warp][tx * W + j]) = make_uint4(a[j], a[j + 1], a[j + 2], a[j + 3]);
      }
      __syncthreads();
      if (threadIdx.x < 16 * W) {  // one word of maxima to a thread
        uint32_t x = 0;
#pragma unroll
        for (int w = 0; w < 8; w += 2) x = I::max3(x, part[w][threadIdx.x], part[w + 1][threadIdx.x]);
#pragma unroll
        for (int e = 0; e < I::kPer; ++e) {
          const int c = threadIdx.x * I::kPer + e;
          const float m = floor_of(I::value(I::kPer == 1 ? x : e ? x >> 16 : x & 0xffffu)), d = den_of(m);
          col_rcp[c] = __frcp_rn(d);
          col_neg[c] = neg_of(d);
          if ((int64_t)tc * 128 + c < p.cols) s[(int64_t)tr * p.s_row + ((int64_t)tc * 128 + c) * p.s_col] = m / 448.f;
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&col_rcp[tx * 8 + 2 * i]);
        const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(&col_neg[tx * 8 + 2 * i]);
        rcp[i] = x.x;
        rcp[i + 1] = x.y;
        neg[i] = y.x;
        neg[i + 1] = y.y;
      }
    }
  }
  uint8_t* q = p.q + b * p.batch_q + r0 * p.ldq + c0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t o[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t e[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int c = 2 * h + k;  // columns 2c and 2c + 1
        const int g = BR == 1 ? i : BC == 1 ? c : 0;
        const uint64_t y = mul2(I::pair(v[i], c), two(0.4375f, 0.4375f));
        const uint64_t t = mul2(y, rcp[g]);
        const uint64_t z = fma2(fma2(t, neg[g], y), rcp[g], t);
        float2 f;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(z));
        e[k] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
      }
      o[h] = __byte_perm(e[0], e[1], 0x5410);
    }
    if (i >= nrow) break;
    uint8_t* row = q + 16 * i * p.ldq;
    if (ncol == 8 && p.vec_q) {
      *reinterpret_cast<uint2*>(row) = make_uint2(o[0], o[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < ncol) row[j] = (uint8_t)(o[j / 4] >> (8 * (j % 4)));
    }
  }
}

template <typename T>
cudaError_t launch_q(const QParams& p, int br, int bc, unsigned grid, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kern = br == 1 ? tb_quantize_kernel<T, 1, 128> : bc == 1 ? tb_quantize_kernel<T, 128, 1>
                                                                : tb_quantize_kernel<T, 128, 128>;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  return e == cudaSuccess ? cudaGetLastError() : e;
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
