// tb_grouped.cu — matrix products whose rows belong to groups (experts) and
// matrix products of 8-bit operands with a scale per block of 128.
//
//   rows grouped   C[r, :] = beta·C[r, :] + A[r, :] · B[e]     r in group e
//   K grouped      G[e] = beta·G[e] + A[rows of e]^T · D[rows of e]
//   8-bit          C = beta·C + Σ_b SA[:, b] SB[b, :] (A_b · B_b), b = blocks of 128 along K
//
// One kernel family, tb_grouped_sm100_kernel<KIND, BN, G>, in the manner of
// the dense GEMM: persistent, warp-specialised, TMA into a ring of 128-byte
// rows, tcgen05.mma into two TMEM accumulators, an epilogue that overlaps the
// next accumulation. Group sizes are read on the device (the offsets are a
// router's output), so no call waits for the host to learn them:
// every CTA builds the table of tiles from the offsets when it starts.
//
//   warp 0   TMA producer              warp 3      scheduler: the next tiles, worked out
//   warp 1   MMA issuer                            once and handed over in shared memory
//   warp 2   row fixer (K grouped)     warps 4-11  epilogue, two per lane quarter
//
// Rows grouped: a tile's rows begin at any row of A (a TMA coordinate other
// than the innermost has no alignment rule); the rows past the group's end
// are other groups' rows, whose results are not stored. A row of the result
// depends on that row of A alone, so nothing of them can leak.
//
// K grouped: the K range of a tile is a range of rows, which ends anywhere
// inside the last ring fill. Rows behind it up to the next multiple of the
// MMA's K step would add another group's products, so the fixer warp zeroes
// them in shared memory, in both operands (0 · NaN is NaN), between the
// TMA's arrival and the MMA; all other fills go from TMA to MMA directly.
//
// 8-bit: one ring fill is one block of 128 along K, and one accumulation in
// TMEM. The epilogue warps take each block's sums from TMEM, scale them and
// add them to f32 registers while the MMAs of the next block run into the
// other accumulator. The sum of 128 products of two e4m3 values is held in
// f32 by the MMA, and the sum over blocks in f32 registers.
//
// Few tiles (a decoding step): the K range is split over the CTAs of a
// cluster, which add their partial sums through distributed shared memory in
// a fixed order — no workspace, no atomics, results repeat bit for bit.
//
// What bounds it (B200, 148 SMs; "burst": a few calls after a pause, at 1965 MHz;
// in a loop the power cap lowers the clock):
// * Training sizes: the operands' way from L2 into the SMs, 43–46 bytes a cycle
//   and SM for 32 KB per fill of a 256 × 256 pair tile (the MMAs of a fill
//   need 512 cycles), and below that the power cap: 16384 rows over 8 experts
//   of 4096 × 4096 bf16 in 387 µs in a burst (1420 TFLOP/s), 455 in a loop.
// * 8-bit products: besides, the epilogue takes 64 KB of sums per block and
//   CTA out of TMEM, 1140 cycles a block: 8192³ e4m3 in 494 µs in a burst (2230
//   TFLOP/s; 437 µs with the epilogue's arithmetic left out), 580 in a loop.
//   With a scale per column (weight gradients) 952 and 954.
// * Decoding steps: HBM, once the weights flow (6.2 TB/s), and some 4 µs of
//   start and end around it: offsets, first tile, first fill, exchange.
//   96 rows over 32 experts of 2048 × 1408 f16 (179 MB): 38 µs in a CUDA graph.
//
// Every wait is bounded, as in the dense GEMM.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <string>
#include <type_traits>

#include "tb_plan.h"
#include "tb_sm100.cuh"
#include "tb_wait.cuh"

using namespace tb::sm100;

namespace {

constexpr int kThreadsG = 384;
constexpr int kMaxGroups = 1024;
constexpr int kMaxStages = 10;
constexpr size_t kSmemLimitG = 232448;  // 227 KB opt-in per CTA

// kHalf      16-bit operands (f16 / bf16) and outputs, the whole K range (at most kOneSum) summed in TMEM
// kHalfSum   16-bit operands, segments of GParams::seg fills summed in f32 registers
// kByte      8-bit operands (e4m3), a scale of B per 128 columns
// kByteCol   8-bit operands, a scale of B per column
enum Kind : int { kHalf = 0, kHalfSum = 1, kByte = 2, kByteCol = 3 };
// The MMA truncates when it adds to its accumulator: the error of a sum grows
// with the number of additions (one for 16 elements of K) and leans one way, and
// K may be a number of rows without a bound. So a segment of K is taken out of
// TMEM and the segments are added in registers, rounded to nearest: every 8
// fills (512 elements of K) for f32 outputs, every 16 for 16-bit outputs, whose
// own rounding is hundreds of times as large. Relative error of f16 products
// against 64 bits, f32 outputs: 3.4e-7 at K = 256, 6.5e-7 from K = 512 on, where
// f32 arithmetic has 4.0e-7 at 512, 5.7e-7 at 1032 and 1.1e-6 at 4096. (Segments
// of 4 fills: 3.5e-7 from 256 on; 16384 rows over 8 experts of 4096 × 4096 took
// 534 µs in place of 470, their weight gradient 308 in place of 246.) bf16
// outputs of K = 4096 and 16384 that are not the nearest value: 0.064 % and
// 0.063 %; in one sum 0.12 % and 0.47 %, by f32 arithmetic 0.03 %. It costs 2 %
// (16384 rows, 8 × 4096 × 4096 bf16), and 10 % where rows are off 16 bytes.
// What one segment holds stays one sum in TMEM, without registers for it (4096
// rows over 8 experts of 512 × 2048 bf16 11.5 µs, with them 13.6; 32768 rows of
// 256 × 4096 88 and 116).
constexpr int kSegF32 = 8, kSegHalf = 16;
constexpr int64_t kOneSum = 64 * kSegHalf;  // elements of K

// KIND's ring fill is 128 bytes of K: 64 or 128 elements, four MMA K steps.
template <int KIND, int BN, int G>
struct GCfg {
  static constexpr bool kBytes = KIND == kByte || KIND == kByteCol;
  static constexpr bool kSums = KIND != kHalf;          // sums held in registers
  static constexpr int kEl = kBytes ? 1 : 2;
  static constexpr int kKB = 128 / kEl;                 // K elements per fill
  static constexpr int kMmaK = 32 / kEl;                // K elements per MMA
  static constexpr int kBM = 128 * G;                   // tile rows
  static constexpr int kBnCta = BN / G;                 // B columns a CTA loads
  static constexpr uint32_t kABytes = 128 * 128;
  static constexpr uint32_t kBBytes = kBnCta * 128;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes;
  static constexpr int kMnBox = 128 / kEl;              // columns of an MN-major box
  static constexpr uint32_t kMnBoxBytes = kKB * 128;
  static constexpr uint32_t kMnStep = kMmaK * 128;      // bytes per MMA K step, MN-major
  static constexpr int kAccs = 2;
  static constexpr uint32_t kTmemCols = kAccs * BN;
  static constexpr int kHalfCols = BN / 2;              // columns per epilogue warp
  static constexpr int kChunks = kHalfCols / 32;
  // One CTA's tile may be shared by a cluster, but not with 128 sums per
  // thread: the exchange does not fit beside them into the registers.
  static constexpr bool kShares = G == 1 && !(kSums && BN == 256);
  // Outputs that no vector access reaches go through emit32_spread, but for the
  // same reason not straight from 128 sums: those of 16-bit operands go through
  // local memory, those of 8-bit operands are stored by the element (either way's
  // spills made e4m3 products 1.5 to 1.8 times as long).
  static constexpr bool kSpreads = !(kSums && BN == 256);
  static constexpr uint32_t kRedStride = (BN + 4) * 4;  // bytes per row of the cluster's partial sums
};

// Tiles of every group, built by each CTA from the offsets.
struct GroupTable {
  int32_t start[kMaxGroups];
  int32_t rows[kMaxGroups];
  int32_t cum[kMaxGroups + 1];  // rows grouped: tiles before group e
};

struct GTile {
  int32_t e;         // group
  int32_t row0;      // first row of A and C (rows grouped) or of G[e] (K grouped)
  int32_t rows, n0, cols;
  int32_t k0, k_end; // K range of the tile
  int32_t f0, f1;    // this CTA's ring fills of it
};

constexpr int kTileSlots = 4;

struct GBars {
  uint64_t full[kMaxStages], empty[kMaxStages], fix[kMaxStages];
  uint64_t tfull[2], tempty[2];
  uint64_t drain, ready, consumed;
  // tiles that the scheduler warp has worked out for the other roles
  uint64_t tile_full[kTileSlots], tile_empty[kTileSlots];
  GTile tile[kTileSlots];
  alignas(16) float col_scale[8][128];  // per epilogue warp: SB of its columns in the block at hand
  uint32_t tmem_holder;
  uint32_t issued;  // the producer's fills
  int abort_flag;
};

constexpr size_t kTailBytes = sizeof(GroupTable) + sizeof(GBars) + 64;

struct GScale {           // scale of element (mn, k-block b): p[(mn >> shift)·smn + b·sk], per group + sg
  const float* p;
  int64_t sg, smn, sk;
  int32_t shift;          // 7: one scale per 128 rows / columns; 0: per row / column
};

struct GParams {
  int32_t k_grouped;      // 1: K ranges are the groups (weight gradient)
  int32_t groups;
  int32_t M, N, K;        // rows grouped: A is M × K; K grouped: A is K × M, D is K × N (K = rows of both)
  int32_t tiles_m, tiles_n;  // K grouped: tiles of one group; rows grouped: tiles_n only
  int32_t most_tiles;     // as many as offsets that do not fall can give
  const void* offsets;    // groups + 1 entries, or null: one group of all rows
  int32_t offsets_64;
  int32_t a_mn, b_kmaj;
  uint32_t fmt;           // MMA operand format (idesc bits 7 and 10)
  int32_t beta, c_dtype, vec;  // vec: what C's rows are multiples of (128, 32, 16 bytes, or 0)
  void* C;
  int64_t ldc, group_c;
  GScale sa, sb;
  int64_t budget;         // cycles until a wait gives up
  int32_t stages;         // ring depth
  int32_t seg;            // fills per accumulation in TMEM, a power of two (kinds with sums)
  int32_t split, split_log2;  // CTAs per cluster that share a tile's K range (G = 1)
  int32_t block;          // rows whose partial sums they exchange at a time: 32, 64 or 128
  int32_t small_log2;     // log2 of the rows of tmAs's boxes: a K-major A tile of few rows comes in these (G = 1)
};

// Offset i, clamped to [0, rows]: whatever the offsets are, no access leaves the operands.
__device__ __forceinline__ int32_t read_offset(const void* offsets, bool wide, int32_t rows, int32_t i) {
  long long v;
  if (!offsets) v = i ? rows : 0;
  else if (wide) v = static_cast<const long long*>(offsets)[i];
  else v = static_cast<const int32_t*>(offsets)[i];
  return (int32_t)(v < 0 ? 0 : v > rows ? rows : v);
}

// Tile t, worked out by a whole warp. Inside a group, tiles go in bands of 8
// tile rows, rows fastest: the CTAs at work share few panels of A and B.
// `cursor`: a group at or before the tile's; it moves on with t.
template <int BM, int BN, int KB>
__device__ __forceinline__ GTile tile_at(const GParams& p, const GroupTable& tab, int32_t t, int32_t part,
                                         int32_t& cursor, int lane) {
  GTile g;
  uint32_t u;
  int32_t group_rows, tiles_m;
  if (p.k_grouped) {
    const uint32_t per = (uint32_t)p.tiles_m * (uint32_t)p.tiles_n;
    g.e = (int32_t)((uint32_t)t / per);
    u = (uint32_t)t - (uint32_t)g.e * per;
    tiles_m = p.tiles_m;
    group_rows = p.M;
    g.row0 = 0;
    g.k0 = tab.start[g.e];
    g.k_end = g.k0 + tab.rows[g.e];
  } else {
    uint32_t before;  // groups from the cursor on that end at or before t: 32 looked at together
    do {
      const int32_t i = cursor + lane;
      before = __ballot_sync(0xffffffffu, i < p.groups && tab.cum[i + 1] <= t);
      cursor += __popc(before);
    } while (before == 0xffffffffu);
    g.e = cursor;
    u = (uint32_t)(t - tab.cum[cursor]);
    group_rows = tab.rows[cursor];
    tiles_m = (group_rows + BM - 1) / BM;
    g.row0 = tab.start[cursor];
    g.k0 = 0;
    g.k_end = p.K;
  }
  uint32_t m = 0, n = u;
  if (tiles_m > 1) {
    const uint32_t band = u / (8u * (uint32_t)p.tiles_n), v = u - band * 8u * (uint32_t)p.tiles_n;
    const uint32_t height = min(8u, (uint32_t)tiles_m - band * 8u);
    n = v / height;
    m = band * 8u + v - n * height;
  }
  g.row0 += (int32_t)m * BM;
  g.rows = min(BM, group_rows - (int32_t)m * BM);
  g.n0 = (int32_t)n * BN;
  g.cols = min(BN, p.N - g.n0);
  const uint32_t fills = (uint32_t)(g.k_end - g.k0 + KB - 1) / KB;  // < 2^25: 8 parts of it fit in 32 bits
  g.f0 = (int32_t)(fills * (uint32_t)part >> p.split_log2);
  g.f1 = (int32_t)(fills * (uint32_t)(part + 1) >> p.split_log2);
  return g;
}

__device__ __forceinline__ float load_out(const GParams& p, const char* q) {
  if (p.c_dtype == TB_F32) return *reinterpret_cast<const float*>(q);
  if (p.c_dtype == TB_F16) return __half2float(*reinterpret_cast<const __half*>(q));
  return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(q));
}
__device__ __forceinline__ void store_out(const GParams& p, char* q, float v) {
  if (p.c_dtype == TB_F32) *reinterpret_cast<float*>(q) = v;
  else if (p.c_dtype == TB_F16) *reinterpret_cast<__half*>(q) = __float2half_rn(v);
  else *reinterpret_cast<__nv_bfloat16*>(q) = __float2bfloat16_rn(v);
}
__device__ __forceinline__ uint32_t pack2(const GParams& p, float a, float b) {
  uint32_t w;
  if (p.c_dtype == TB_F16) {
    const __half2 h = __floats2half2_rn(a, b);
    memcpy(&w, &h, 4);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    memcpy(&w, &h, 4);
  }
  return w;
}
__device__ __forceinline__ float2 unpack2(const GParams& p, uint32_t w) {
  if (p.c_dtype == TB_F16) {
    __half2 h;
    memcpy(&h, &w, 4);
    return __half22float2(h);
  }
  __nv_bfloat162 h;
  memcpy(&h, &w, 4);
  return __bfloat1622float2(h);
}
// 32 bytes in one store: a whole sector, so that a warp's rows need no merging
// in L2. (The output through shared memory, by TMA or in whole rows, gained 3 to
// 13 % where little but the output is written and lost as much elsewhere.)
__device__ __forceinline__ void st_32(void* q, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(q), "r"(w[0]), "r"(w[1]),
               "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Row lane of n registers to register lane of n rows, in every n lanes: n − 1
// exchanges of half the registers with the lane n / 2, … 1 away. Its own inverse.
template <typename T, int N>
__device__ __forceinline__ void transpose(T (&v)[N], int lane) {
#pragma unroll
  for (int d = N / 2; d > 0; d /= 2) {
    const bool up = lane & d;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i & d) continue;
      const T got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + d], d);
      if (up) v[i] = got;
      else v[i + d] = got;
    }
  }
}

// beta·C + v of `ncol` of 32 consecutive columns, whatever the alignment: v is
// a lane's row, which begins at q; the first `rows` lanes' rows are stored. The
// values are transposed in registers, so that an access of the warp covers
// consecutive columns of one row (f32) or the 32-bit words of two (16 bits; a
// row that begins inside a word has its first column alone). Each lane storing
// its own row, an element at a time, touched 32 sectors with every access
// (5481 × 2679 of 8-bit operands, k = 128: bf16 143 µs, now 28.5; f32 98, now 31).
template <int KIND>
__device__ __forceinline__ void emit32_spread(const GParams& p, char* q, float (&v)[32], int rows, int ncol, int lane) {
  if (KIND != kHalf && p.c_dtype == TB_F32) {
    const int64_t step = p.ldc * 4;
    transpose(v, lane);
    if (lane >= ncol) return;
    q += lane * (4 - step);
    constexpr int kAhead = 4;  // rows whose loads run together
#pragma unroll
    for (int i0 = 0; i0 < 32; i0 += kAhead) {
      if (i0 >= rows) break;
      if (p.beta) {
        float c[kAhead];
        const char* at = q;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          c[i] = 0.f;
          if (i0 + i < rows) c[i] = *reinterpret_cast<const float*>(at);
          at += step;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) v[i0 + i] += c[i];
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (i0 + i < rows) *reinterpret_cast<float*>(q) = v[i0 + i];
        q += step;
        asm volatile("" : "+l"(q));  // one address, not 32
      }
    }
    return;
  }
  const int64_t step = p.ldc * 2;
  const bool odd = reinterpret_cast<uintptr_t>(q) & 2, mine = lane < rows;
  const int half = lane & 16, x = lane & 15;
  char* const first = q + (half - lane) * step;  // of this half's 16 rows
  // word x of row i of the 16: its columns and their address
  auto each_word = [&](auto&& f) {
    char* at = first;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int col = 2 * x + (int)((reinterpret_cast<uintptr_t>(at) >> 1) & 1);
      if (half + i < rows && col < ncol) f(i, at + col * 2, col + 1 < ncol);
      at += step;
      asm volatile("" : "+l"(at));
    }
  };
  if (p.beta) {
    uint32_t c[16] = {};
    each_word([&](int i, const char* at, bool both) {
      if (both) c[i] = *reinterpret_cast<const uint32_t*>(at);
      else c[i] = *reinterpret_cast<const unsigned short*>(at);
    });
    __syncwarp();
    transpose(c, lane);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float2 u = unpack2(p, c[j]);
      v[2 * j] += odd ? 0.f : u.x;
      v[2 * j + 1] += odd ? u.x : u.y;
      if (j < 15) v[2 * j + 2] += odd ? u.y : 0.f;
    }
    if (odd && mine) v[0] += load_out(p, q);
  }
  uint32_t w[16];
#pragma unroll
  for (int j = 0; j < 16; ++j)
    w[j] = pack2(p, odd ? v[2 * j + 1] : v[2 * j], odd ? (j < 15 ? v[2 * j + 2] : 0.f) : v[2 * j + 1]);
  if (odd && mine) store_out(p, q, v[0]);
  __syncwarp();
  transpose(w, lane);
  each_word([&](int i, char* at, bool both) {
    if (both) *reinterpret_cast<uint32_t*>(at) = w[i];
    else *reinterpret_cast<unsigned short*>(at) = (unsigned short)w[i];
  });
}

// beta·C + v of `ncol` of 32 consecutive columns at q.
__device__ __forceinline__ void emit32(const GParams& p, char* q, float (&v)[32], int ncol) {
  const int el = p.c_dtype == TB_F32 ? 4 : 2;
  if (ncol < 32 || !p.vec) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < ncol) store_out(p, q + i * el, p.beta ? v[i] + load_out(p, q + i * el) : v[i]);
    return;
  }
  if (p.c_dtype == TB_F32) {
    if (p.beta) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 c = reinterpret_cast<const float4*>(q)[i];
        v[4 * i] += c.x; v[4 * i + 1] += c.y; v[4 * i + 2] += c.z; v[4 * i + 3] += c.w;
      }
    }
    if (p.vec >= 32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(v[8 * i + j]);
        st_32(q + 32 * i, w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        reinterpret_cast<float4*>(q)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
    return;
  }
  if (p.beta) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 c = reinterpret_cast<const uint4*>(q)[i];
      const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack2(p, w[j]);
        v[8 * i + 2 * j] += f.x;
        v[8 * i + 2 * j + 1] += f.y;
      }
    }
  }
  uint32_t w[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) w[j] = pack2(p, v[2 * j], v[2 * j + 1]);
  if (p.vec >= 32) {
    st_32(q, w);
    st_32(q + 32, w + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<uint4*>(q)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
}

// beta·C + v of a warp's 32 rows × 32 columns where the rows of C begin on 128
// bytes: v is a lane's row, at q. Transposed in registers in units of 32 bytes,
// so that a store covers 128 (f32) or 64 consecutive bytes of a row. (Weight
// gradients, f32: 41 × 768 × 1024 from 26 rows 41.2 µs with each lane storing
// its own row, now 30.8; 8 × 1024 × 1024 from 2048 rows 19.6, now 16.5. Where
// rows begin off 128 bytes it is the other way round, 41 × 760 × 1048: 39 and
// 52; warps with fewer rows would pay for the exchange and store no faster.)
template <int KIND>
__device__ __forceinline__ void emit32_rows(const GParams& p, char* q, float (&v)[32], int lane) {
  auto run = [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;  // lanes of a row: 4 (f32) or 2
    const int64_t step = p.ldc * L;
    const int x = lane & (L - 1);
    char* const first = q + x * (32 - step);
    uint32_t w[L][8];
    auto turn = [&]() {  // word x of row i of the L to word i of row x
#pragma unroll
      for (int d = L / 2; d > 0; d /= 2) {
        const bool up = lane & d;
#pragma unroll
        for (int i = 0; i < L; ++i) {
          if (i & d) continue;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? w[i][k] : w[i + d][k], d);
            if (up) w[i][k] = got;
            else w[i + d][k] = got;
          }
        }
      }
    };
    if (p.beta) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
          const uint4 u = *reinterpret_cast<const uint4*>(first + i * step + 4 * h);
          w[i][h] = u.x; w[i][h + 1] = u.y; w[i][h + 2] = u.z; w[i][h + 3] = u.w;
        }
      }
      turn();
#pragma unroll
      for (int j = 0; j < 8 * L; ++j) {
        if constexpr (L == 4) {
          v[j] += __uint_as_float(w[j / 8][j % 8]);
        } else {
          const float2 f = unpack2(p, w[j / 8][j % 8]);
          v[2 * j] += f.x;
          v[2 * j + 1] += f.y;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8 * L; ++j) {
      if constexpr (L == 4) w[j / 8][j % 8] = __float_as_uint(v[j]);
      else w[j / 8][j % 8] = pack2(p, v[2 * j], v[2 * j + 1]);
    }
    turn();
#pragma unroll
    for (int i = 0; i < L; ++i) st_32(first + i * step, w[i]);
  };
  if (KIND != kHalf && p.c_dtype == TB_F32) run(std::integral_constant<int, 4>());
  else run(std::integral_constant<int, 2>());
}

// beta·C + v of `ncol` (at most 4) consecutive columns at q.
__device__ __forceinline__ void emit4(const GParams& p, char* q, float4 s, int ncol) {
  const float v[4] = {s.x, s.y, s.z, s.w};
  if (ncol >= 4 && p.vec && !p.beta) {
    if (p.c_dtype == TB_F32) *reinterpret_cast<float4*>(q) = s;
    else *reinterpret_cast<uint2*>(q) = make_uint2(pack2(p, s.x, s.y), pack2(p, s.z, s.w));
    return;
  }
  const int el = p.c_dtype == TB_F32 ? 4 : 2;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < ncol) store_out(p, q + i * el, p.beta ? v[i] + load_out(p, q + i * el) : v[i]);
}

// Two f32 in one register pair.
__device__ __forceinline__ uint64_t pack_u32x2(uint32_t a, uint32_t b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) {
  return pack_u32x2(__float_as_uint(a), __float_as_uint(b));
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float& a, float& b) {
  uint32_t x, y;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(x), "=r"(y) : "l"(v));
  a = __uint_as_float(x);
  b = __uint_as_float(y);
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

template <int KIND, int BN, int G>
__global__ void __launch_bounds__(kThreadsG, 1)
    tb_grouped_sm100_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmAs,
                            const __grid_constant__ CUtensorMap tmB, const __grid_constant__ GParams p) {
  using Cf = GCfg<KIND, BN, G>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const int S = p.stages;
  uint8_t* sA = smem;
  uint8_t* sB = smem + (size_t)S * Cf::kABytes;
  uint8_t* red = smem + (size_t)S * Cf::kStageBytes;
  uint8_t* tail = red + (Cf::kShares && p.split > 1 ? (uint32_t)p.block * Cf::kRedStride : 0u);
  GBars& bars = *reinterpret_cast<GBars*>(tail);
  GroupTable& tab = *reinterpret_cast<GroupTable*>(tail + ((sizeof(GBars) + 15) & ~size_t(15)));
  volatile int* abort_flag = &bars.abort_flag;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);
  const int lane = threadIdx.x % 32;
  const int cluster = G * p.split;
  const uint32_t crank = cluster > 1 ? cluster_ctarank() : 0u;
  const uint32_t rank = G == 2 ? crank : 0u;        // CTA of the pair
  const int32_t part = G == 2 ? 0 : (int32_t)crank; // part of the K range
  const bool leader = rank == 0;
  const int32_t first = blockIdx.x / cluster, stride = gridDim.x / cluster;

  if (warp == 0) {
    // one barrier to a lane
    auto init = [&](uint64_t* bar, int n, uint32_t count) {
      if (lane < n) mbar_init(smem_addr(bar + lane), count);
    };
    init(bars.full, S, p.k_grouped ? G : 1);  // K grouped pairs: both producers (or fixers) arrive for each fill
    init(bars.empty, S, 1);
    init(bars.fix, S, 1);
    init(bars.tfull, 2, 1);
    init(bars.tempty, 2, 8 * G);
    init(bars.tile_full, kTileSlots, 1);
    // producer, epilogue warps, and those of MMA issuer and fixer that are at work
    init(bars.tile_empty, kTileSlots, 9 + (leader ? 1 : 0) + (p.k_grouped ? 1 : 0));
    init(&bars.drain, 1, 1);
    init(&bars.ready, 1, 1);
    init(&bars.consumed, 1, 8 * p.split);
    if (lane == 0) bars.abort_flag = 0;
    fence_mbar_init();
    if (lane == 0) {
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmAs);
      tma_prefetch_desc(&tmB);
    }
  }
  if (G == 2 && warp == 1) {  // (one CTA: the MMA issuer allocates while the first fill is on its way)
    tmem_alloc_g<G>(smem_addr(&bars.tmem_holder), Cf::kTmemCols);
    tmem_relinquish_g<G>();
  }
  if (warp == 2) {
    // Every launch's parameters come into the constant cache anew, a miss of
    // some hundred cycles to a line: all lines are asked for at once here.
    uint32_t all = 0;
    for (int i = lane; i < (int)(sizeof(GParams) / 4); i += 32) all ^= reinterpret_cast<const uint32_t*>(&p)[i];
    asm volatile("" ::"r"(all));
  }
  // Barriers (and a pair's TMEM) are there. The scheduler joins when it has the first tile.
  auto start = [&]() {
    if constexpr (G == 2) {
      tc_fence_before();
      cluster_sync();
    }
    __syncthreads();
    if constexpr (G == 2) tc_fence_after();
    else if (cluster > 1) cluster_arrive();  // the epilogue waits before it sends to other CTAs
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  };

  // The tiles in turn, up to one without columns: take() waits for the next
  // (and says no after the last, or when it gave up), done() gives its slot back.
  int slot = 0;
  uint32_t slot_phase = 0;
  auto done = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_addr(&bars.tile_empty[slot]));
    if (++slot == kTileSlots) {
      slot = 0;
      slot_phase ^= 1u;
    }
  };
  // One read of a field of the tile at hand (not kept in a register).
  auto field = [&](int32_t GTile::*m) {
    return *const_cast<const volatile int32_t*>(&(bars.tile[slot].*m));
  };
  bool ok = true;  // false: a wait gave up
  auto take = [&](uint32_t site) {
    ok = ok && warp_poll(smem_addr(&bars.tile_full[slot]), slot_phase, abort_flag, site, lane, p.budget);
    return ok && field(&GTile::cols) > 0;
  };

  // Sums in registers, 256 columns: 128 per epilogue thread. 256 threads ×
  // 224 + 128 × 56 registers = the launch's 384 × 168.
  constexpr bool kMoveRegs = Cf::kSums && BN == 256;
  if (warp < 4) {
    if constexpr (kMoveRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp != 3) start();
    if (warp == 0) {
      // ------------------------------------------------------------ producer
      // An operand's fill is a few boxes: box j of fill f lies at coordinates
      // (x + f·fx + j·jx, y + f·fy + j·jy) and goes to dst + j·step. What
      // decides them is worked out once per tile; with the parameters read and
      // tested inside the loop a fill took 475 cycles to issue.
      const bool a_mn = p.a_mn, b_mn = !p.b_kmaj, grouped_k = p.k_grouped;
      const int32_t a_fx = a_mn ? 0 : Cf::kKB, a_fy = a_mn ? Cf::kKB : 0;
      const int32_t b_fx = b_mn ? 0 : Cf::kKB, b_fy = b_mn ? Cf::kKB : 0;
      const int32_t b_boxes = b_mn ? Cf::kBnCta / Cf::kMnBox : 1;
      const int32_t sr = 1 << p.small_log2;
      const uint32_t full0 = smem_addr(&bars.full[0]), empty0 = smem_addr(&bars.empty[0]), fix0 = smem_addr(&bars.fix[0]);
      const uint32_t full0_leader = G == 2 ? map_to_cta(full0, 0) : full0;
      const uint32_t sa0 = smem_addr(sA), sb0 = smem_addr(sB);
      int stage = 0;
      uint32_t phase = 0;
      uint32_t issued = 0;
      asm volatile("griddepcontrol.wait;" ::: "memory");
      while (take(kSiteProducer)) {
        const GTile g = bars.tile[slot];
        done();
        // K-major A of a tile with few rows: only the small boxes that hold them
        const bool few = G == 1 && !a_mn && g.rows <= 3 * sr;
        const CUtensorMap* const map_a = few ? &tmAs : &tmA;
        const int32_t a_boxes = a_mn ? 128 / Cf::kMnBox : few ? (g.rows + sr - 1) >> p.small_log2 : 1;
        const uint32_t a_step = a_mn ? Cf::kMnBoxBytes : (uint32_t)sr * 128u;
        const int32_t a_jx = a_mn ? Cf::kMnBox : 0, a_jy = a_mn ? 0 : sr;
        const uint32_t bytes = (few ? (uint32_t)a_boxes * a_step : Cf::kABytes) + Cf::kBBytes;
        const int32_t am = g.row0 + (int32_t)rank * 128, bn = g.n0 + (int32_t)rank * Cf::kBnCta;
        const int32_t k_first = g.k0 + g.f0 * Cf::kKB;
        int32_t ax = a_mn ? am : k_first, ay = a_mn ? k_first : am;
        int32_t bx = b_mn ? bn : k_first, by = b_mn ? k_first : bn;
        const int32_t be = grouped_k ? 0 : g.e;
        // the fill (if any) whose last rows the fixer takes out
        const int32_t fix_at = grouped_k && (g.k_end - g.k0) % Cf::kMmaK != 0 && g.f1 * Cf::kKB > g.k_end - g.k0 - Cf::kMmaK
                                   ? (g.k_end - g.k0) / Cf::kKB : -1;
        for (int32_t f = g.f0; f < g.f1; ++f) {
          if (issued >= (uint32_t)S && !warp_wait(empty0 + stage * 8, phase ^ 1u, abort_flag, kSiteProducer, lane, p.budget)) {
            ok = false;
            break;
          }
          if (elect_one()) {
            uint32_t bar;
            if (f == fix_at) {  // this CTA's fixer takes the fill on from here
              bar = fix0 + stage * 8;
              mbar_expect_tx(bar, bytes);
            } else {
              bar = full0_leader + stage * 8;
              if (leader) mbar_expect_tx(full0 + stage * 8, G * bytes);
              else if (grouped_k) mbar_arrive_remote(bar);
            }
            uint32_t dst = sa0 + (uint32_t)stage * Cf::kABytes;
            for (int32_t j = 0; j < a_boxes; ++j, dst += a_step) {
              if constexpr (G == 2) tma_load_2d_pair(dst, map_a, bar, ax + j * a_jx, ay + j * a_jy);
              else tma_load_2d(dst, map_a, bar, ax + j * a_jx, ay + j * a_jy);
            }
            dst = sb0 + (uint32_t)stage * Cf::kBBytes;
            for (int32_t j = 0; j < b_boxes; ++j, dst += Cf::kMnBoxBytes) {
              if constexpr (G == 2) tma_load_3d_pair(dst, &tmB, bar, bx + j * Cf::kMnBox, by, be);
              else tma_load_3d(dst, &tmB, bar, bx + j * Cf::kMnBox, by, be);
            }
          }
          __syncwarp();
          ax += a_fx;
          ay += a_fy;
          bx += b_fx;
          by += b_fy;
          ++issued;
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (lane == 0) bars.issued = issued;
    } else if (warp == 1) {
      // ---------------------------------------------------------- MMA issuer
      // (Issuer and fixer touch no memory, but a wait of theirs is not to count
      // the time of the kernel before.)
      if constexpr (G == 1) {
        tmem_alloc_g<G>(smem_addr(&bars.tmem_holder), Cf::kTmemCols);
        tmem_relinquish_g<G>();
      }
      asm volatile("griddepcontrol.wait;" ::: "memory");
      if (leader) {
        const uint32_t tmem_base = *const_cast<volatile uint32_t*>(&bars.tmem_holder);
        const uint32_t idesc = idesc_f16_f32(Cf::kBM, BN, p.a_mn ? 1 : 0, p.b_kmaj ? 0 : 1) | (p.fmt << 7) |
                               (p.fmt << 10);
        // descriptor words: the start address (16-byte units) moves in the low one
        const uint32_t a_step = (p.a_mn ? Cf::kMnStep : 32u) >> 4, b_step = (p.b_kmaj ? 32u : Cf::kMnStep) >> 4;
        const uint64_t da = smem_desc_sw128(smem_addr(sA), p.a_mn ? Cf::kMnBoxBytes : 16u, 1024);
        const uint64_t db = smem_desc_sw128(smem_addr(sB), p.b_kmaj ? 16u : Cf::kMnBoxBytes, 1024);
        const uint32_t a_hi = (uint32_t)(da >> 32), b_hi = (uint32_t)(db >> 32);
        const uint32_t full0 = smem_addr(&bars.full[0]), empty0 = smem_addr(&bars.empty[0]),
                       tfull0 = smem_addr(&bars.tfull[0]), tempty0 = smem_addr(&bars.tempty[0]);
        auto commit = [&](uint32_t bar) {
          if constexpr (G == 2) umma_commit_pair(bar, 0x3);
          else umma_commit(bar);
        };
        const int32_t seg_mask = Cf::kBytes ? 0 : p.seg - 1;
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool issued_any = false;
        while (take(kSiteMma)) {
          // this tile's fills, and the MMA steps of the last one
          const int32_t fills = field(&GTile::f1) - field(&GTile::f0);
          const int32_t last_valid = min(Cf::kKB, field(&GTile::k_end) - field(&GTile::k0) - (field(&GTile::f1) - 1) * Cf::kKB);
          const int last_steps = (last_valid + Cf::kMmaK - 1) / Cf::kMmaK;
          const int32_t fixed_at = p.k_grouped && last_valid % Cf::kMmaK != 0 ? fills - 1 : -1;
          done();
          bool here = false;  // the fill at hand was seen to have landed
          for (int32_t f = 0; f < fills; ++f) {
            // first and last fill of an accumulation
            const bool opens = Cf::kSums ? (f & seg_mask) == 0 : f == 0;
            const bool closes = f + 1 == fills || (Cf::kSums && ((f + 1) & seg_mask) == 0);
            if ((opens && !warp_poll(tempty0 + acc * 8, acc_phase ^ 1u, abort_flag, kSiteMma, lane, p.budget)) ||
                (!here && !warp_poll(full0 + stage * 8, phase, abort_flag, kSiteMma, lane, p.budget))) {
              ok = false;
              break;
            }
            // The other CTA's fixer wrote to its shared memory before it arrived here.
            if (G == 2 && !Cf::kBytes && f == fixed_at) mbar_test_wait_cluster(full0 + stage * 8, phase);
            tc_fence_after();
            const uint32_t a_lo = (uint32_t)da + (uint32_t)stage * (Cf::kABytes >> 4);
            const uint32_t b_lo = (uint32_t)db + (uint32_t)stage * (Cf::kBBytes >> 4);
            const uint32_t d = tmem_base + (uint32_t)(acc * BN);
            const uint32_t empty = empty0 + stage * 8;
            if (++stage == S) {
              stage = 0;
              phase ^= 1u;
            }
            // the next fill's barrier is read while this one's MMAs are issued
            const bool peek = f + 1 < fills && mbar_test_wait(full0 + stage * 8, phase);
            if (elect_one()) {
              if (f + 1 < fills || last_steps == 4) {
#pragma unroll
                for (uint32_t kk = 0; kk < 4; ++kk)
                  umma_words<G, Cf::kBytes>(d, a_lo + a_step * kk, a_hi, b_lo + b_step * kk, b_hi, idesc,
                                            (!opens || kk > 0) ? 1u : 0u);
              } else {
                for (uint32_t kk = 0; kk < (uint32_t)last_steps; ++kk)
                  umma_words<G, Cf::kBytes>(d, a_lo + a_step * kk, a_hi, b_lo + b_step * kk, b_hi, idesc,
                                            (!opens || kk > 0) ? 1u : 0u);
              }
              commit(empty);
              if (closes) commit(tfull0 + acc * 8);
            }
            here = __all_sync(0xffffffffu, peek);
            issued_any = true;
            if (closes && ++acc == 2) {
              acc = 0;
              acc_phase ^= 1u;
            }
          }
        }
        if (!ok && issued_any && lane == 0) {
          // Given up with MMAs possibly in flight: wait for them before TMEM goes.
          if constexpr (G == 2) umma_commit_pair(smem_addr(&bars.drain), 0x1);
          else umma_commit(smem_addr(&bars.drain));
          const long long t0 = clock64();
          while (!mbar_try_wait(smem_addr(&bars.drain), 0)) {
            if (clock64() - t0 > kWaitBudgetCycles) {
              record_error(TB_ERR_DEVICE_TIMEOUT, kSiteDrain);
              break;
            }
          }
        }
        __syncwarp();
      }
    } else if (warp == 2) {
      // --------------------------------------------------------------- fixer
      asm volatile("griddepcontrol.wait;" ::: "memory");
      if (p.k_grouped) {
        int stage = 0;
        uint32_t fix_phase = 0;  // bit s: parity of stage s's next fix
        while (take(kSiteFixer)) {
          const GTile g = bars.tile[slot];
          done();
          const int32_t n = g.f1 - g.f0;
          if (n <= 0) continue;
          const int32_t last = (stage + n - 1) % S;  // only a tile's last fill can be short
          const int32_t valid = min(Cf::kKB, g.k_end - (g.k0 + (g.f1 - 1) * Cf::kKB));
          stage = (stage + n) % S;
          if (valid % Cf::kMmaK == 0) continue;
          if (!warp_poll(smem_addr(&bars.fix[last]), (fix_phase >> last) & 1u, abort_flag, kSiteFixer, lane, p.budget)) {
            ok = false;
            break;
          }
          fix_phase ^= 1u << last;
          // K rows [valid, next multiple of the K step) of every box of both
          // operands: 128 bytes per row (the swizzle stays inside a row)
          const int32_t end = (valid + Cf::kMmaK - 1) / Cf::kMmaK * Cf::kMmaK;
          const int32_t words = (end - valid) * 8;
          auto zero = [&](uint8_t* stage_base, int nboxes) {
            for (int b = 0; b < nboxes; ++b) {
              uint4* q = reinterpret_cast<uint4*>(stage_base + (size_t)b * Cf::kMnBoxBytes + (size_t)valid * 128);
              for (int i = lane; i < words; i += 32) q[i] = make_uint4(0, 0, 0, 0);
            }
          };
          zero(sA + (size_t)last * Cf::kABytes, 128 / Cf::kMnBox);
          zero(sB + (size_t)last * Cf::kBBytes, Cf::kBnCta / Cf::kMnBox);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if constexpr (G == 2) mbar_arrive_cluster(map_to_cta(smem_addr(&bars.full[last]), 0));
            else mbar_arrive(smem_addr(&bars.full[last]));
          }
        }
      }
    } else {
      // ----------------------------------------------------------- scheduler
      const void* const offsets = p.offsets;
      const bool wide = p.offsets_64;
      const int32_t groups = p.groups, all_rows = p.k_grouped ? p.K : p.M, tiles_n = p.tiles_n,
                    most_tiles = p.most_tiles;
      // What this launch reads may be written by the kernel before it in the
      // stream, which each role waits for before its first access to memory
      // (programmatic launch).
      asm volatile("griddepcontrol.wait;" ::: "memory");
      int32_t before = 0;
      for (int32_t e0 = 0; e0 < groups; e0 += 32) {
        const int32_t e = e0 + lane;
        // every lane loads one offset; the last also the one behind its 32
        int32_t lo = e <= groups ? read_offset(offsets, wide, all_rows, e) : all_rows;
        const int32_t behind = lane == 31 && e < groups ? read_offset(offsets, wide, all_rows, e + 1) : 0;
        const int32_t up = __shfl_down_sync(0xffffffffu, lo, 1);
        const int32_t rows = e < groups ? max(0, (lane == 31 ? behind : up) - lo) : 0;
        if (e < groups) {
          tab.start[e] = lo;
          tab.rows[e] = rows;
        }
        // Offsets that fall and rise again give the same rows to several
        // groups; the sums stop at what others can reach, so they fit in 32
        // bits and the work is bounded whatever the offsets are.
        int32_t v = (rows + Cf::kBM - 1) / Cf::kBM * tiles_n;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
          const int32_t o = __shfl_up_sync(0xffffffffu, v, d);
          if (lane >= d) v = min(v + o, most_tiles);
        }
        v = min(before + v, most_tiles);
        if (e < groups) tab.cum[e + 1] = v;
        before = __shfl_sync(0xffffffffu, v, 31);
      }
      if (lane == 0) tab.cum[0] = 0;
      __syncwarp();
      const int32_t tiles = p.k_grouped ? groups * p.tiles_m * tiles_n : before;
      int32_t cursor = 0;
      for (int32_t t = first;; t += stride) {
        GTile tile = {};
        if (t < tiles) tile = tile_at<Cf::kBM, BN, Cf::kKB>(p, tab, t, part, cursor, lane);
        if (t == first) start();
        if (!warp_wait(smem_addr(&bars.tile_empty[slot]), slot_phase ^ 1u, abort_flag, kSiteScheduler, lane, p.budget)) break;
        if (lane == 0) {
          bars.tile[slot] = tile;
          mbar_arrive(smem_addr(&bars.tile_full[slot]));
        }
        if (t >= tiles) break;  // that was the tile without columns
        if (++slot == kTileSlots) {
          slot = 0;
          slot_phase ^= 1u;
        }
      }
    }
  } else {
    if constexpr (kMoveRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    start();
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;               // TMEM lane quarter
    const int half = (warp - 4) >> 2;     // column half
    const int row_in_tile = (int)rank * 128 + q * 32 + lane;
    const int c_half = half * Cf::kHalfCols;
    // this warp's lanes and columns of TMEM (one CTA: known once an accumulation is complete)
    const uint32_t tm_off = ((uint32_t)(q * 32) << 16) + (uint32_t)c_half;
    const uint32_t tm_pair = G == 2 ? bars.tmem_holder + tm_off : 0u;
    auto tm = [&]() {
      if constexpr (G == 2) return tm_pair;
      else return *const_cast<volatile uint32_t*>(&bars.tmem_holder) + tm_off;
    };
    const int el = p.c_dtype == TB_F32 ? 4 : 2;
    const uint32_t tempty0 = G == 2 ? map_to_cta(smem_addr(&bars.tempty[0]), 0) : smem_addr(&bars.tempty[0]);
    auto release = [&](int acc) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (G == 2) mbar_arrive_remote(tempty0 + acc * 8);
        else mbar_arrive(tempty0 + acc * 8);
      }
    };
    // the tile at hand in C, and this thread's row and column half of it
    auto tile_at_c = [&]() {
      const int64_t group = p.k_grouped ? (int64_t)field(&GTile::e) * p.group_c : 0;
      return static_cast<char*>(p.C) + (group + (int64_t)field(&GTile::row0) * p.ldc + field(&GTile::n0)) * el;
    };
    auto row_at = [&]() { return tile_at_c() + ((int64_t)row_in_tile * p.ldc + c_half) * el; };
    // The cluster's CTAs hold partial sums of one tile. `block` rows at a time,
    // each sends row r of its own (sums(c): this warp's chunk c) to CTA
    // r mod split, which adds them in CTA order and stores the row. The rows
    // come as st.async, counted on the receiver's barrier: no fence, and the
    // sums are read from the CTA's own shared memory. (Partial sums left
    // behind a cluster-scope release and read by the others took 4100 cycles
    // from the last fill to the stores.) False: a wait gave up.
    uint32_t red_phase = 0;
    // Rows read are handed back to the senders of the next ones by an arrival
    // that is released at cluster scope, so that what was read here is not
    // overwritten before. The release waits for this warp's stores, half a
    // microsecond and more: so a block has as many rows as the tiles have, and a
    // tile's last block is handed back behind the start of the next tile's sums,
    // or (no next tile) not at all. (8-bit, K = N = 4096, blocks of 32 rows and of
    // the tile's: 33 rows 9.9 and 8.6 µs, 128 rows 15.7 and 12.8; a release of
    // CTA scope, which orders nothing for the other CTAs: 9.4 and 14.2.)
    bool owed = false;
    auto hand_back = [&]() {
      __syncwarp();
      if (lane < p.split) mbar_arrive_cluster(map_to_cta(smem_addr(&bars.consumed), (uint32_t)lane));
      owed = false;
    };
    auto share = [&](auto&& sums) -> bool {
      const int rows = field(&GTile::rows), cols = field(&GTile::cols);
      char* tile = tile_at_c();
      const int per = p.block >> p.split_log2;  // rows of each CTA in a block
      const uint32_t red0 = smem_addr(red), ready0 = smem_addr(&bars.ready), consumed0 = smem_addr(&bars.consumed);
      for (int r0 = 0; r0 < rows; r0 += p.block) {
        const int here = min(p.block, rows - r0);
        const int mine = (here - part + p.split - 1) >> p.split_log2;  // rows part, part + split, … below `here`
        // Every CTA has read the rows before. All eight warps wait for it, not
        // only the senders: a CTA without a row of its own has nothing else to
        // wait for, and a warp that went on would arrive a second time and stand
        // in for one that still reads.
        if (!warp_poll<true>(consumed0, red_phase ^ 1u, abort_flag, kSiteCluster, lane, p.budget)) return false;
        if (warp == 4 && lane == 0)
          mbar_expect_tx(ready0, (uint32_t)(mine * p.split) * (uint32_t)((cols + 31) / 32 * 128));
        const int row = q * 32 - r0 + lane;  // of the block
        if (row >= lane && row - lane < here) {
          const uint32_t owner = (uint32_t)row & (uint32_t)(p.split - 1);
          const uint32_t to = map_to_cta(red0 + (uint32_t)(part * per + (row >> p.split_log2)) * Cf::kRedStride, owner);
          const uint32_t bar = map_to_cta(ready0, owner);
#pragma unroll
          for (int c = 0; c < Cf::kChunks; ++c) {
            if (c_half + c * 32 < cols) {
              const float(&s)[32] = sums(c);
              if (row < here) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  st_async_f4(to + (uint32_t)(c_half + c * 32 + 4 * i) * 4, bar, s[4 * i], s[4 * i + 1], s[4 * i + 2],
                              s[4 * i + 3]);
              }
              __syncwarp();
            }
          }
        }
        if (!warp_poll<true>(ready0, red_phase, abort_flag, kSiteCluster, lane, p.budget)) return false;
        for (int i = warp - 4; i < mine; i += 8) {
#pragma unroll
          for (int h = 0; h < BN / 128; ++h) {  // four columns of each 128 to a lane
            const int c0 = h * 128 + lane * 4;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (j < p.split) {
                const float4 x = *reinterpret_cast<const float4*>(red + (size_t)(j * per + i) * Cf::kRedStride + c0 * 4);
                s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
              }
            }
            emit4(p, tile + ((int64_t)(r0 + part + (i << p.split_log2)) * p.ldc + c0) * el, s, cols - c0);
          }
        }
        if (r0 + p.block < rows) hand_back();
        else owed = true;
        red_phase ^= 1u;
      }
      return true;
    };
    int acc = 0;
    uint32_t acc_phase = 0;
    if (Cf::kShares && cluster > 1) cluster_wait();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    while (take(kSiteEpilogue)) {
      if (Cf::kShares && owed) hand_back();
      // Only the count of accumulations and the scales' places stay in
      // registers during the sums; the rest is read again for the stores.
      const int32_t fills = field(&GTile::f1) - field(&GTile::f0);
      const bool warp_ok = (int)rank * 128 + q * 32 < field(&GTile::rows) && c_half < field(&GTile::cols);
      float v[Cf::kSums ? Cf::kChunks : 1][32];

      if constexpr (Cf::kSums) {
        // Each accumulation is taken from TMEM, scaled, and added to this
        // thread's sums two at a time. A chunk's load runs while the one
        // before it is added.
        uint64_t sum[Cf::kChunks][16];
#pragma unroll
        for (int c = 0; c < Cf::kChunks; ++c)
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[c][i] = 0;
        // Scales of the next block: this row's, and the columns' (one, or this
        // lane's of the warp's columns); fetched a block ahead.
        const float *sa = nullptr, *sb = nullptr;
        int64_t sb_col[4] = {0, 0, 0, 0};
        float xa = 1.f, xb = 1.f, xc[4] = {0.f, 0.f, 0.f, 0.f};
        // (Plain loads: the kernel before this one may have written them while
        // this one was already resident.)
        auto fetch = [&]() {
          xa = *sa;
          sa += p.sa.sk;
          if constexpr (KIND == kByte) xb = *sb;
          if constexpr (KIND == kByteCol) {
#pragma unroll
            for (int j = 0; j < Cf::kHalfCols / 32; ++j) xc[j] = sb[sb_col[j]];
          }
          sb += p.sb.sk;
        };
        if constexpr (Cf::kBytes) {
          const int32_t f0 = field(&GTile::f0);
          const int32_t arow = min(field(&GTile::row0) + row_in_tile, p.M - 1);  // masked rows read some valid scale
          const int32_t col0 = field(&GTile::n0) + c_half;
          sa = p.sa.p + (int64_t)(arow >> p.sa.shift) * p.sa.smn + (int64_t)f0 * p.sa.sk;
          sb = p.sb.p + (int64_t)field(&GTile::e) * p.sb.sg + (int64_t)f0 * p.sb.sk;
          if constexpr (KIND == kByte) {
            sb += (int64_t)(min(col0, p.N - 1) >> 7) * p.sb.smn;
          } else {
#pragma unroll
            for (int j = 0; j < Cf::kHalfCols / 32; ++j)
              sb_col[j] = (int64_t)min(col0 + 32 * j + lane, p.N - 1) * p.sb.smn;
          }
          if (fills > 0) fetch();
        }
        for (int32_t left = fills; left > 0; left -= Cf::kBytes ? 1 : p.seg) {
          const float x = xa * xb;
          float* cs = bars.col_scale[warp - 4];
          if constexpr (KIND == kByteCol) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < Cf::kHalfCols / 32; ++j) cs[32 * j + lane] = xc[j];
            __syncwarp();
          }
          if constexpr (Cf::kBytes) {
            if (left > 1) fetch();
          }
          if (!warp_poll(smem_addr(&bars.tfull[acc]), acc_phase, abort_flag, kSiteEpilogue, lane, p.budget)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (warp_ok) {
            uint32_t w[2][32];
            const uint32_t ta = tm() + (uint32_t)(acc * BN);
            const uint64_t x2 = pack_f32x2(x, x);
            tmem_ld_32x32b_x32_issue(ta, w[0]);
#pragma unroll
            for (int c = 0; c < Cf::kChunks; ++c) {
              tmem_ld_wait(w[c & 1]);
              if (c + 1 < Cf::kChunks) tmem_ld_32x32b_x32_issue(ta + (uint32_t)((c + 1) * 32), w[(c + 1) & 1]);
              else release(acc);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const uint64_t u = pack_u32x2(w[c & 1][2 * i], w[c & 1][2 * i + 1]);
                if constexpr (KIND == kHalfSum) {
                  sum[c][i] = add_f32x2(sum[c][i], u);
                } else if constexpr (KIND == kByte) {
                  sum[c][i] = fma_f32x2(u, x2, sum[c][i]);
                } else {
                  const uint64_t y = *reinterpret_cast<const uint64_t*>(cs + c * 32 + 2 * i);
                  sum[c][i] = fma_f32x2(u, mul_f32x2(x2, y), sum[c][i]);
                }
              }
            }
          } else {
            release(acc);
          }
          if (++acc == 2) {
            acc = 0;
            acc_phase ^= 1u;
          }
        }
        if (!ok) break;
        if (KIND == kHalfSum && !Cf::kSpreads && !p.vec) {
          // 128 sums: through local memory, so that they are not in registers
          // beside the exchange, and the loop above needs no room for it.
          if (warp_ok) {
            float all[Cf::kChunks][32];
#pragma unroll
            for (int c = 0; c < Cf::kChunks; ++c)
#pragma unroll
              for (int i = 0; i < 16; ++i) unpack_f32x2(sum[c][i], all[c][2 * i], all[c][2 * i + 1]);
            const int32_t rows = field(&GTile::rows) - (row_in_tile - lane);  // of this warp
            const int32_t cols = field(&GTile::cols) - c_half;
            char* row = row_at();
#pragma unroll 1
            for (int c = 0; c * 32 < cols && c < Cf::kChunks; ++c) {
              float one[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) one[i] = all[c][i];
              emit32_spread<KIND>(p, row + c * 32 * el, one, rows, min(32, cols - c * 32), lane);
              __syncwarp();
            }
          }
          done();
          continue;
        }
#pragma unroll
        for (int c = 0; c < Cf::kChunks; ++c)
#pragma unroll
          for (int i = 0; i < 16; ++i) unpack_f32x2(sum[c][i], v[c][2 * i], v[c][2 * i + 1]);
      } else {
        const bool row_ok = row_in_tile < field(&GTile::rows);
        const int32_t cols = field(&GTile::cols) - c_half;
        char* row = row_at();
        if (fills > 0) {
          if (!warp_poll(smem_addr(&bars.tfull[acc]), acc_phase, abort_flag, kSiteEpilogue, lane, p.budget)) {
            ok = false;
            break;
          }
          tc_fence_after();
        }
        if (Cf::kShares && p.split > 1) {
          if (!(ok = share([&](int c) -> const float (&)[32] {
                  if (fills > 0) {
                    tmem_ld_32x32b_x32(tm() + (uint32_t)(acc * BN + c * 32), v[0]);
                  } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[0][i] = 0.f;
                  }
                  return v[0];
                })))
            break;
        } else {
          auto chunks = [&](auto&& emit) {
#pragma unroll
            for (int c = 0; c < Cf::kChunks; ++c) {
              if (!warp_ok) break;
              if (fills > 0) {
                tmem_ld_32x32b_x32(tm() + (uint32_t)(acc * BN + c * 32), v[0]);
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[0][i] = 0.f;
              }
              const int ncol = min(32, cols - c * 32);
              if (ncol > 0) emit(row + c * 32 * el, ncol);
              __syncwarp();
            }
          };
          if (!Cf::kSpreads || p.vec) {
            const bool whole = p.vec == 128 && row_in_tile - lane + 32 <= field(&GTile::rows);
            chunks([&](char* at, int ncol) {
              if (whole && ncol == 32) emit32_rows<KIND>(p, at, v[0], lane);
              else if (row_ok) emit32(p, at, v[0], ncol);
            });
          } else {
            const int32_t rows = field(&GTile::rows) - (row_in_tile - lane);  // of this warp
            chunks([&](char* at, int ncol) { emit32_spread<KIND>(p, at, v[0], rows, ncol, lane); });
          }
        }
        if (fills > 0) {
          release(acc);
          if (++acc == 2) {
            acc = 0;
            acc_phase ^= 1u;
          }
        }
      }

      if constexpr (Cf::kSums) {
        if (Cf::kShares && p.split > 1) {
          if (!(ok = share([&](int c) -> const float (&)[32] { return v[c]; }))) break;
        } else {
          const bool row_ok = row_in_tile < field(&GTile::rows);
          const int32_t cols = field(&GTile::cols) - c_half;
          char* row = row_at();
          if (!Cf::kSpreads || p.vec) {
            bool whole = false;
            if constexpr (Cf::kSpreads) whole = p.vec == 128 && row_in_tile - lane + 32 <= field(&GTile::rows);
#pragma unroll
            for (int c = 0; c < Cf::kChunks; ++c) {
              const int ncol = min(32, cols - c * 32);
              bool stored = false;
              if constexpr (Cf::kSpreads) {
                stored = whole && ncol == 32;
                if (stored) emit32_rows<KIND>(p, row + c * 32 * el, v[c], lane);
              }
              if (!stored && row_ok && ncol > 0) emit32(p, row + c * 32 * el, v[c], ncol);
            }
          } else if constexpr (Cf::kSpreads) {
            const int32_t rows = field(&GTile::rows) - (row_in_tile - lane);  // of this warp; may be none
#pragma unroll
            for (int c = 0; c < Cf::kChunks; ++c) {
              const int ncol = min(32, cols - c * 32);
              if (ncol > 0) emit32_spread<KIND>(p, row + c * 32 * el, v[c], rows, ncol, lane);
              __syncwarp();
            }
          }
          __syncwarp();
        }
      }
      done();
    }
    // The last rows are not handed back, so nothing of another CTA is on its way
    // to this one any more (a cluster barrier at the end took 1200 cycles).
  }

  __syncthreads();
  if (*abort_flag && threadIdx.x == 0 && leader) {
    // Given up: the newest fill of each stage must land before the CTAs exit.
    // (Otherwise the MMAs have waited for every fill.)
    const uint32_t last = min(bars.issued, (uint32_t)S);
    for (uint32_t i = 0; i < last; ++i) {
      const uint32_t f = bars.issued - 1 - i;
      const long long t0 = clock64();
      while (!mbar_try_wait(smem_addr(&bars.full[f % S]), (f / S) & 1)) {
        if (clock64() - t0 > kWaitBudgetCycles) {
          record_error(TB_ERR_DEVICE_TIMEOUT, kSiteDrain);
          break;
        }
      }
    }
  }
  if (G == 2) {
    cluster_sync();
  } else if (cluster > 1 && *abort_flag) {
    // given up: no CTA leaves while another one may still send to it
    if (warp < 4) cluster_wait();
    cluster_sync();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_g<G>(bars.tmem_holder, Cf::kTmemCols);
  }
}

// Self-test of these kernels' waits: one warp polls a barrier that nothing
// arrives on until the budget is spent, and a second wait of the same CTA then
// sees the abort flag.
__global__ void tb_grouped_selftest_kernel(long long budget) {
  __shared__ __align__(8) uint64_t bars[2];
  __shared__ int abort_flag;
  if (threadIdx.x < 2) mbar_init(smem_addr(&bars[threadIdx.x]), 1);
  if (threadIdx.x == 0) abort_flag = 0;
  fence_mbar_init();
  __syncthreads();
  if (!warp_poll(smem_addr(&bars[0]), 0, &abort_flag, kSiteSelfTest, threadIdx.x, budget))
    warp_wait(smem_addr(&bars[1]), 0, &abort_flag, kSiteDrain, threadIdx.x, budget);
}

// Copies rows of `row_bytes` to rows of ld_dst bytes (a multiple of 16), the
// rest of each row zero: operands whose rows TMA cannot address. HBM bound: a
// lane reads the one or two aligned 16-byte words that hold its 16 bytes (they
// lie in the rows' own allocation: no word without a byte of the row is
// touched) and shifts them into place. A warp takes a row at a time.
__global__ void __launch_bounds__(256)
    tb_grouped_pack_kernel(const uint8_t* __restrict__ src, int64_t ld_src, int64_t batch_src, uint8_t* __restrict__ dst,
                           int64_t ld_dst, int64_t batch_dst, int64_t rows, int64_t row_bytes) {
  src += (int64_t)blockIdx.z * batch_src;
  dst += (int64_t)blockIdx.z * batch_dst;
  const int lane = threadIdx.x % 32;
  const int words = (int)(ld_dst / 16);
  for (int64_t r = blockIdx.x * 8 + threadIdx.x / 32; r < rows; r += (int64_t)gridDim.x * 8) {
    const uint8_t* row = src + r * ld_src;
    // every 16 bytes of a row are off a boundary by as much as its first
    const int shift = (int)(reinterpret_cast<uintptr_t>(row) & 15);
    const uint4* word = reinterpret_cast<const uint4*>(row - shift);
    const int have = (int)((shift + row_bytes + 15) / 16);  // words that hold bytes of the row
    const int first = shift >> 2, bits = (shift & 3) * 8;
    for (int w0 = lane; w0 < words; w0 += 128) {
      uint4 lo[4], hi[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // all loads at once
        const int w = w0 + 32 * u;
        lo[u] = w < have ? __ldg(word + w) : make_uint4(0, 0, 0, 0);
        hi[u] = shift && w + 1 < have ? __ldg(word + w + 1) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int w = w0 + 32 * u;
        if (w >= words) break;
        const uint32_t x[9] = {lo[u].x, lo[u].y, lo[u].z, lo[u].w, hi[u].x, hi[u].y, hi[u].z, hi[u].w, 0};
        uint32_t v[5] = {0, 0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 5; ++i)
#pragma unroll
          for (int f = 0; f < 4; ++f)
            if (first == f) v[i] = x[i + f];
        const int64_t left = row_bytes - (int64_t)w * 16;  // bytes of the row from here on
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = __funnelshift_r(v[i], v[i + 1], bits);
          const int64_t here = left - 4 * i;
          if (here < 4) v[i] = here <= 0 ? 0u : v[i] & (0xffffffffu >> (32 - 8 * (int)here));
        }
        *reinterpret_cast<uint4*>(dst + r * ld_dst + (int64_t)w * 16) = make_uint4(v[0], v[1], v[2], v[3]);
      }
    }
  }
}

// ------------------------------------------------------------------- host

constexpr int kMaxDev = 64;

std::atomic<PFN_cuTensorMapEncodeTiled_v12000> g_encode_fn{nullptr};

tbStatus encoder(PFN_cuTensorMapEncodeTiled_v12000* out) {
  PFN_cuTensorMapEncodeTiled_v12000 f = g_encode_fn.load();
  if (!f) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult qres;
    cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &qres);
    if (e != cudaSuccess || qres != cudaDriverEntryPointSuccess || !fn)
      return tb_fail(TB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    f = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    g_encode_fn.store(f);
  }
  *out = f;
  return TB_OK;
}

std::atomic<int> g_sms[kMaxDev];

tbStatus current_device(int* dev, int* sms) {
  cudaError_t e = cudaGetDevice(dev);
  if (e != cudaSuccess) return tb_fail(TB_ERR_CUDA, std::string("cudaGetDevice: ") + cudaGetErrorString(e));
  if (*dev < 0 || *dev >= kMaxDev) return tb_fail(TB_ERR_UNSUPPORTED, "device ordinal beyond the library's table");
  int n = g_sms[*dev].load();
  if (!n) {
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *dev);
    if (e != cudaSuccess)
      return tb_fail(TB_ERR_CUDA, std::string("cudaDeviceGetAttribute: ") + cudaGetErrorString(e));
    g_sms[*dev].store(n);
  }
  *sms = n;
  return TB_OK;
}

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
// Clusters of 2^i CTAs (one CTA to an SM) that the device holds at once: fewer
// than its SMs divide into, since a cluster stays inside a GPC.
std::atomic<int> g_clusters[kMaxDev][4];

bool al(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)n == 0; }

// One operand as the kernel reads it: `rows` rows of `cols` contiguous
// elements in each of `batch` matrices.
struct Operand {
  const void* p;
  int64_t rows, cols, ld, batch, stride;  // strides in elements
  bool pack(int el) const {
    return !al(p, 16) || (rows > 1 && ld * el % 16) || (batch > 1 && stride * el % 16);
  }
  int64_t packed_ld(int el) const { return (cols * el + 15) / 16 * 16; }  // bytes
  size_t packed_bytes(int el) const {
    return ((size_t)packed_ld(el) * (size_t)rows * (size_t)batch + 255) / 256 * 256;
  }
};

tbStatus pack(Operand* o, int el, void* ws, cudaStream_t stream) {
  if (o->batch > 65535) return tb_fail(TB_ERR_UNSUPPORTED, "too many groups to repack");
  const int64_t ld = o->packed_ld(el);
  const unsigned gx = (unsigned)std::min<int64_t>(std::max<int64_t>(1, cdiv(o->rows, 8)), 4096);
  tb_grouped_pack_kernel<<<dim3(gx, 1, (unsigned)o->batch), 256, 0, stream>>>(
      static_cast<const uint8_t*>(o->p), o->ld * el, o->stride * el, static_cast<uint8_t*>(ws), ld, ld * o->rows,
      o->rows, o->cols * el);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return tb_fail(TB_ERR_CUDA, std::string("tb_grouped_pack launch: ") + cudaGetErrorString(e));
  o->p = ws;
  o->ld = ld / el;
  o->stride = o->ld * o->rows;
  return TB_OK;
}

tbStatus encode(CUtensorMap* map, int dims_n, const Operand& o, int el, int is_bf16, uint32_t box0, uint32_t box1,
                const char* what) {
  PFN_cuTensorMapEncodeTiled_v12000 f;
  tbStatus st = encoder(&f);
  if (st != TB_OK) return st;
  cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)o.batch};
  const cuuint64_t ld = (cuuint64_t)(o.rows > 1 ? o.ld * el : (o.cols * el + 15) / 16 * 16);
  const cuuint64_t bs = (cuuint64_t)(o.batch > 1 ? (cuuint64_t)o.stride * el : ld * (cuuint64_t)o.rows);
  cuuint64_t strides[2] = {ld, bs};
  cuuint32_t box[3] = {box0, box1, 1}, es[3] = {1, 1, 1};
  const CUtensorMapDataType dt = el == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                 : is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                           : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUresult r = f(map, dt, (cuuint32_t)dims_n, const_cast<void*>(o.p), dims, strides, box, es,
                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return tb_fail(TB_ERR_CUDA, std::string("cuTensorMapEncodeTiled(") + what + ") failed with CUresult " +
                                    std::to_string((int)r));
  return TB_OK;
}

struct Launch {
  Operand a, b;
  int el, bf16;
  int64_t tiles;  // an upper bound of the tiles
  int64_t rows;   // mean rows of a group that has any
  int64_t tile_rows;  // and of a tile
  int64_t slots;  // clusters at once
  GParams p;
};

template <int KIND, int BN, int G>
tbStatus launch(Launch& L, int dev, cudaStream_t stream) {
  using Cf = GCfg<KIND, BN, G>;
  GParams& p = L.p;
  CUtensorMap ta, tas, tb_;
  std::memset(&tas, 0, sizeof(tas));
  tbStatus st = encode(&ta, 2, L.a, L.el, L.bf16, p.a_mn ? Cf::kMnBox : Cf::kKB, p.a_mn ? Cf::kKB : 128, "A");
  p.small_log2 = L.rows <= 16 ? 3 : 5;
  if (st == TB_OK && !p.a_mn && G == 1) st = encode(&tas, 2, L.a, L.el, L.bf16, Cf::kKB, 1u << p.small_log2, "A");
  if (st == TB_OK)
    st = encode(&tb_, 3, L.b, L.el, L.bf16, p.b_kmaj ? Cf::kKB : Cf::kMnBox, p.b_kmaj ? Cf::kBnCta : Cf::kKB, "B");
  if (st != TB_OK) return st;
  // Some waits last as long as the tiles that the scheduler may be ahead by: a
  // second, and 4096 cycles (three to eight times what it takes) for each of their fills.
  p.budget = kWaitBudgetCycles + (int64_t)kTileSlots * 4096 * cdiv(p.K, Cf::kKB);
  p.split_log2 = p.split == 8 ? 3 : p.split == 4 ? 2 : p.split == 2 ? 1 : 0;
  // A block holds the rows that a tile has on average, if the ring keeps three stages beside it.
  p.block = BN == 128 && L.tile_rows > 64 ? 128 : L.tile_rows > 32 ? 64 : 32;
  const size_t fixed = 1024 + kTailBytes + (p.split > 1 ? (size_t)p.block * Cf::kRedStride : 0);
  p.stages = (int)std::min<size_t>(kMaxStages, (kSmemLimitG - fixed) / Cf::kStageBytes);
  const size_t smem = fixed + (size_t)p.stages * Cf::kStageBytes;
  auto kern = tb_grouped_sm100_kernel<KIND, BN, G>;
  static std::atomic<bool> ready[kMaxDev];
  if (!ready[dev].load()) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimitG);
    if (e != cudaSuccess)
      return tb_fail(TB_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
    ready[dev].store(true);
  }
  const int cluster = G * p.split;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(L.slots, L.tiles) * cluster), 1, 1);
  cfg.blockDim = dim3(kThreadsG, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  // The set-up (barriers, TMEM) overlaps the end of the kernel before.
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, ta, tas, tb_, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return tb_fail(TB_ERR_CUDA, std::string("tb_grouped launch: ") + cudaGetErrorString(e));
  return TB_OK;
}

// Whether a call's sums are held in registers: all but 16-bit outputs of so few
// elements of K that one accumulation holds them.
bool sums_in_registers(const Launch& L) { return L.el == 1 || L.p.c_dtype == TB_F32 || L.p.K > kOneSum; }

// The kind of a tile's kernel, by the operands' and the output's types and K.
template <int BN, int G>
tbStatus launch_tile(Launch& L, int dev, cudaStream_t stream) {
  if (L.el == 1)
    return L.p.sb.shift ? launch<kByte, BN, G>(L, dev, stream) : launch<kByteCol, BN, G>(L, dev, stream);
  L.p.seg = L.p.c_dtype == TB_F32 ? kSegF32 : kSegHalf;
  return sums_in_registers(L) ? launch<kHalfSum, BN, G>(L, dev, stream) : launch<kHalf, BN, G>(L, dev, stream);
}

tbStatus resident_clusters(int dev, int sms, int (&out)[4]) {
  for (int i = 0; i < 4; ++i) {
    int n = g_clusters[dev][i].load();
    if (!n) {
      auto kern = tb_grouped_sm100_kernel<kHalf, 128, 1>;
      cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimitG);
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)(sms >> i << i), 1, 1);
      cfg.blockDim = dim3(kThreadsG, 1, 1);
      cfg.dynamicSmemBytes = kSmemLimitG;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1u << i;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
      if (e != cudaSuccess)
        return tb_fail(TB_ERR_CUDA, std::string("cudaOccupancyMaxActiveClusters: ") + cudaGetErrorString(e));
      n = std::max(1, std::min(n, sms >> i));
      g_clusters[dev][i].store(n);
    }
    out[i] = n;
  }
  return TB_OK;
}

// Tile and K split, by estimated cycles. `rows`: mean rows of a group that has any.
//
// One ring fill takes 512 cycles of MMAs whatever the tile's width: the loop
// took 118–132 cycles per tcgen05.mma of 128 (or a pair's 256) rows, barriers
// included, for 64, 128 and 256 columns alike (the instruction by itself was not
// measured), so a narrower tile only lowers the rate of this loop. The pass of
// the epilogue over each 8-bit accumulation (1140 cycles at 256 columns) has no
// term here. A
// fill takes longer where its bytes do: 23 bytes a cycle and SM are an SM's
// share of HBM, 45 the most that one SM was seen to draw while others idle,
// and L2 feeds all SMs together 46 bytes a cycle each (42 where a CTA takes
// 48 KB at a time). A pair's two cluster barriers take 600 cycles.
// Storing a tile overlaps the next tile's fills: 16 bytes a cycle and SM, or
// (rows off 16-byte boundaries) 8 elements, 4 by way of local memory, 0.6 where
// a lane stores its own row.
tbStatus choose_and_launch(Launch& L, int64_t groups, int64_t rows, int sms, int dev, cudaStream_t stream) {
  GParams& p = L.p;
  int resident[4];  // clusters of 1, 2, 4 and 8 CTAs
  tbStatus st = resident_clusters(dev, sms, resident);
  if (st != TB_OK) return st;
  L.rows = rows;
  L.tile_rows = std::min<int64_t>(p.k_grouped ? p.M : rows, 128);
  const int64_t n = p.N;
  const int64_t m = p.k_grouped ? p.M : rows;
  const int64_t busy = p.k_grouped ? groups : std::min<int64_t>(groups, p.M);
  const int64_t fills = std::max<int64_t>(1, cdiv(p.k_grouped ? cdiv(p.K, std::max<int64_t>(1, groups)) : p.K, 128 / L.el));
  const int ce = p.c_dtype == TB_F32 ? 4 : 2;
  const bool even = p.k_grouped || !p.offsets;  // every group has m rows
  const bool sums = sums_in_registers(L);
  double best = 0;
  int bn = 0, split = 1;
  bool pair = false;
  auto consider = [&](bool is_pair, int b, int s) {
    // Groups of uneven sizes fill their last tile by half on average.
    const int64_t high = is_pair ? 256 : 128;
    const double tiles_high = even ? (double)cdiv(m, high) : std::max(1.0, (double)m / (double)high + 0.5);
    const int64_t tiles = (int64_t)std::ceil((double)busy * tiles_high) * cdiv(n, b);
    const int64_t slots = resident[is_pair || s == 2 ? 1 : s == 1 ? 0 : s == 4 ? 2 : 3];
    const double rounds = (double)cdiv(tiles, slots);
    const double used = std::min(1.0, (double)tiles / (double)slots);
    const double tile_rows = (double)std::min<int64_t>(m, 128);
    // bytes of a fill from HBM: B's share of a tile whose other tiles read the same B, and A's rows
    const double bytes = 128.0 * ((double)(is_pair ? b / 2 : b) / tiles_high + tile_rows / (double)cdiv(n, b));
    const double near = 128.0 * (is_pair ? 256 : b + tile_rows);  // into the SM, from L2
    const double fill = std::max(std::max(512.0, near / (is_pair || b == 128 ? 46.0 : 42.0)), bytes / std::min(45.0, 23.0 / used));
    const double main = (double)cdiv(fills, s) * fill + (s > 1 ? 300.0 + 300.0 * cdiv((int64_t)tile_rows, 32) : 0.0);
    const double store = tile_rows * b / (p.vec ? 16.0 / ce : !sums || b == 128 ? 8.0 : L.el == 1 ? 0.6 : 4.0) / (s > 1 ? s : 1);
    const double cycles = rounds * std::max(main, store) + std::min(main, store) + (is_pair ? 600.0 : 0.0);
    if (!bn || cycles < best) {
      best = cycles;
      bn = b;
      split = s;
      pair = is_pair;
    }
  };
  if (m > 64) consider(true, 256, 1);
  for (int b : {128, 256})
    for (int s = 1; s <= (sums && b == 256 ? 1 : 8) && (s == 1 || fills >= 4 * s); s *= 2) consider(false, b, s);
  p.split = split;
  L.slots = resident[pair || split == 2 ? 1 : split == 1 ? 0 : split == 4 ? 2 : 3];
  p.tiles_m = (int32_t)cdiv(p.M, pair ? 256 : 128);
  p.tiles_n = (int32_t)cdiv(n, bn);
  L.tiles = p.k_grouped ? groups * p.tiles_m * p.tiles_n
                        : (p.M / (pair ? 256 : 128) + std::min<int64_t>(groups, p.M)) * p.tiles_n;
  p.most_tiles = (int32_t)L.tiles;
  return pair        ? launch_tile<256, 2>(L, dev, stream)
         : bn == 256 ? launch_tile<256, 1>(L, dev, stream)
                     : launch_tile<128, 1>(L, dev, stream);
}

int c_bytes(int32_t dt) { return dt == TB_F32 ? 4 : 2; }

int vector_bytes(const void* C, int64_t ldc, int64_t group, int el) {
  for (int b : {128, 32, 16})
    if (al(C, b) && ldc * el % b == 0 && group * el % b == 0) return b;
  return 0;
}

tbStatus check_desc(const tb_grouped_desc* d, bool bytes) {
  if (!d) return tb_fail(TB_ERR_INVALID_ARGUMENT, "desc must not be NULL");
  if (d->groups < 0 || d->rows < 0 || d->n < 0 || d->k < 0)
    return tb_fail(TB_ERR_INVALID_ARGUMENT, "groups, rows, n and k must not be negative");
  if (d->groups > kMaxGroups)
    return tb_fail(TB_ERR_UNSUPPORTED, "at most " + std::to_string(kMaxGroups) + " groups");
  if (d->rows > INT32_MAX - 512 || d->n > INT32_MAX - 512 || d->k > INT32_MAX - 512)
    return tb_fail(TB_ERR_UNSUPPORTED, "problem dimensions must fit in 32 bits");
  if (bytes ? d->ab_dtype != TB_E4M3 : (d->ab_dtype != TB_F16 && d->ab_dtype != TB_BF16))
    return tb_fail(TB_ERR_INVALID_ARGUMENT, bytes ? "operands must be e4m3" : "operands must be f16 or bf16");
  if (d->c_dtype != TB_F32 && d->c_dtype != TB_F16 && d->c_dtype != TB_BF16)
    return tb_fail(TB_ERR_INVALID_ARGUMENT, "the output must be f32, f16 or bf16");
  if (d->beta != 0 && d->beta != 1) return tb_fail(TB_ERR_INVALID_ARGUMENT, "beta must be 0 or 1");
  const int64_t tiles = (d->rows / 128 + d->groups + 1) * (cdiv(d->n, 64) + 1);
  const int64_t tiles_k = (d->groups + 1) * (cdiv(d->k, 128) + 1) * (cdiv(d->n, 64) + 1);
  if (tiles > INT32_MAX / 2 || tiles_k > INT32_MAX / 2)
    return tb_fail(TB_ERR_UNSUPPORTED, "the problem has too many tiles");
  return TB_OK;
}

tbStatus check_ld(int64_t ld, int64_t row, int64_t rows, const char* name) {
  if (rows > 1 && ld < row)
    return tb_fail(TB_ERR_INVALID_ARGUMENT, std::string(name) + ": the leading dimension must be >= the row length");
  return TB_OK;
}

// Packs what TMA cannot address, then launches. `rows`: mean rows of a group.
tbStatus finish(Launch& L, int64_t groups, int64_t rows, void* ws, size_t ws_bytes, void* stream_v) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  const bool pa = L.a.pack(L.el), pb = L.b.pack(L.el);
  const size_t need = (pa ? L.a.packed_bytes(L.el) : 0) + (pb ? L.b.packed_bytes(L.el) : 0);
  if (need && (!ws || ws_bytes < need || !al(ws, 256)))
    return tb_fail(TB_ERR_WORKSPACE, "these operands' rows are not 16-byte aligned: they are repacked in a 256-byte "
                                     "aligned workspace of " + std::to_string(need) + " bytes");
  int dev, sms;
  tbStatus st = current_device(&dev, &sms);
  if (st != TB_OK) return st;
  uint8_t* w = static_cast<uint8_t*>(ws);
  if (pa) {
    const size_t b = L.a.packed_bytes(L.el);
    if ((st = pack(&L.a, L.el, w, stream)) != TB_OK) return st;
    w += b;
  }
  if (pb && (st = pack(&L.b, L.el, w, stream)) != TB_OK) return st;
  return choose_and_launch(L, groups, rows, sms, dev, stream);
}

// Operands of the row-grouped product: A rows × k, B groups × (k × n or n × k).
void row_operands(const tb_grouped_desc* d, const void* A, int64_t lda, const void* B, int64_t ldb, int64_t stride_b,
                  Operand* a, Operand* b) {
  *a = d->a_col_major ? Operand{A, d->k, d->rows, lda, 1, 0} : Operand{A, d->rows, d->k, lda, 1, 0};
  *b = d->b_col_major ? Operand{B, d->n, d->k, ldb, d->groups, stride_b}
                      : Operand{B, d->k, d->n, ldb, d->groups, stride_b};
}

size_t packing(const Operand& a, const Operand& b, int el) {
  return (a.pack(el) ? a.packed_bytes(el) : 0) + (b.pack(el) ? b.packed_bytes(el) : 0);
}

// beta = 0 and nothing to add: the rows of every group become zero.
// (K = 0; the kernel's tiles then have no fills and store zeros, so it runs
// with an operand that it never reads.)
alignas(16) const unsigned char kNothing[16] = {};

tbStatus run_rows(const tb_grouped_desc* d, bool bytes, const void* A, int64_t lda, const tb_scales* sa, const void* B,
                  int64_t ldb, int64_t stride_b, const tb_scales* sb, void* C, int64_t ldc, const void* offsets,
                  void* ws, size_t ws_bytes, void* stream) {
  tbStatus st = check_desc(d, bytes);
  if (st != TB_OK) return st;
  if (d->rows == 0 || d->n == 0 || d->groups == 0) return TB_OK;
  if (!C || (d->k > 0 && (!A || !B))) return tb_fail(TB_ERR_INVALID_ARGUMENT, "A, B and C must not be NULL");
  const int el = bytes ? 1 : 2;
  Launch L;
  row_operands(d, A, lda, B, ldb, stride_b, &L.a, &L.b);
  if ((st = check_ld(lda, L.a.cols, L.a.rows, "A")) != TB_OK) return st;
  if ((st = check_ld(ldb, L.b.cols, L.b.rows, "B")) != TB_OK) return st;
  if ((st = check_ld(ldc, d->n, d->rows, "C")) != TB_OK) return st;
  const int ce = c_bytes(d->c_dtype);
  if (!al(C, ce)) return tb_fail(TB_ERR_INVALID_ARGUMENT, "C is not aligned to its element size");
  if (offsets && !al(offsets, d->offsets_long ? 8 : 4))
    return tb_fail(TB_ERR_INVALID_ARGUMENT, "offsets are not aligned to their element size");
  GParams& p = L.p;
  std::memset(&p, 0, sizeof(p));
  if (bytes) {
    if (d->k > 0 && (!sa || !sb || !sa->ptr || !sb->ptr))
      return tb_fail(TB_ERR_INVALID_ARGUMENT, "8-bit operands need their scales");
    if (sa && sb) {
      if ((sa->block != 1 && sa->block != 128) || (sb->block != 1 && sb->block != 128))
        return tb_fail(TB_ERR_INVALID_ARGUMENT, "a scale covers 1 or 128 rows of A and 1 or 128 columns of B");
      if (offsets && sa->block != 1)
        return tb_fail(TB_ERR_UNSUPPORTED, "grouped rows need a scale for each row of A");
      p.sa = {sa->ptr, 0, sa->stride_mn, sa->stride_k, sa->block == 128 ? 7 : 0};
      p.sb = {sb->ptr, sb->stride_group, sb->stride_mn, sb->stride_k, sb->block == 128 ? 7 : 0};
    }
  }
  L.el = el;
  L.bf16 = d->ab_dtype == TB_BF16;
  p.k_grouped = 0;
  p.groups = (int32_t)d->groups;
  p.M = (int32_t)d->rows;
  p.N = (int32_t)d->n;
  p.K = (int32_t)d->k;
  p.offsets = offsets;
  p.offsets_64 = d->offsets_long;
  p.a_mn = d->a_col_major ? 1 : 0;
  p.b_kmaj = d->b_col_major ? 1 : 0;
  p.fmt = L.bf16 ? 1u : 0u;
  p.beta = d->beta;
  p.c_dtype = d->c_dtype;
  p.C = C;
  p.ldc = ldc;
  p.vec = vector_bytes(C, ldc, 0, ce);
  if (d->k == 0) {
    if (d->beta) return TB_OK;
    L.a = Operand{kNothing, 1, 16, 16, 1, 0};
    L.b = Operand{kNothing, 1, 16, 16, 1, 0};
  }
  const int64_t busy = std::min<int64_t>(d->groups, d->rows);
  return finish(L, d->groups, cdiv(d->rows, busy), ws, ws_bytes, stream);
}

}  // namespace

// The status word of this translation unit's kernels; read and cleared.
tbStatus tb_grouped_status(uint32_t* raw) {
  uint32_t v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_tb_status, sizeof(v));
  if (e != cudaSuccess)
    return tb_fail(TB_ERR_CUDA, std::string("cudaMemcpyFromSymbol: ") + cudaGetErrorString(e));
  if (v) {
    const uint32_t zero = 0;
    cudaMemcpyToSymbol(g_tb_status, &zero, sizeof(zero));
  }
  *raw = v;
  return TB_OK;
}

extern "C" tbStatus tb_selftest_grouped_wait(void* stream, uint64_t budget_cycles) {
  tb_clear_error();
  if (budget_cycles == 0 || budget_cycles > (uint64_t)kWaitBudgetCycles)
    return tb_fail(TB_ERR_INVALID_ARGUMENT, "budget_cycles must be in (0, 2e9]");
  tb_grouped_selftest_kernel<<<1, 32, 0, reinterpret_cast<cudaStream_t>(stream)>>>((long long)budget_cycles);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TB_OK
                          : tb_fail(TB_ERR_CUDA, std::string("tb_grouped_selftest launch: ") + cudaGetErrorString(e));
}

extern "C" tbStatus tb_grouped_desc_init(tb_grouped_desc* d) {
  tb_clear_error();
  if (!d) return tb_fail(TB_ERR_INVALID_ARGUMENT, "desc must not be NULL");
  std::memset(d, 0, sizeof(*d));
  d->groups = 1;
  d->ab_dtype = TB_F16;
  d->c_dtype = TB_F32;
  d->beta = 1;
  return TB_OK;
}

extern "C" size_t tb_grouped_matmul_workspace_bytes(const tb_grouped_desc* d, const void* A, int64_t lda,
                                                    const void* B, int64_t ldb, int64_t stride_b) {
  if (!d || d->rows <= 0 || d->n <= 0 || d->k <= 0 || d->groups <= 0) return 0;
  Operand a, b;
  row_operands(d, A, lda, B, ldb, stride_b, &a, &b);
  return packing(a, b, d->ab_dtype == TB_E4M3 ? 1 : 2);
}

extern "C" tbStatus tb_grouped_matmul(const tb_grouped_desc* d, const void* A, int64_t lda, const void* B, int64_t ldb,
                                      int64_t stride_b, void* C, int64_t ldc, const void* offsets, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  tb_clear_error();
  if (d && d->a_col_major) return tb_fail(TB_ERR_UNSUPPORTED, "grouped rows need a row-major A");
  if (d && d->groups > 0 && !offsets) return tb_fail(TB_ERR_INVALID_ARGUMENT, "offsets must not be NULL");
  return run_rows(d, false, A, lda, nullptr, B, ldb, stride_b, nullptr, C, ldc, offsets, workspace, workspace_bytes,
                  stream);
}

extern "C" size_t tb_grouped_matmul_wgrad_workspace_bytes(const tb_grouped_desc* d, const void* A, int64_t lda,
                                                          const void* D, int64_t ldd) {
  if (!d || d->rows <= 0 || d->n <= 0 || d->k <= 0 || d->groups <= 0) return 0;
  return packing(Operand{A, d->rows, d->k, lda, 1, 0}, Operand{D, d->rows, d->n, ldd, 1, 0}, 2);
}

extern "C" tbStatus tb_grouped_matmul_wgrad(const tb_grouped_desc* d, const void* A, int64_t lda, const void* D,
                                            int64_t ldd, void* Gp, int64_t ldg, int64_t stride_g, const void* offsets,
                                            void* workspace, size_t workspace_bytes, void* stream) {
  tb_clear_error();
  tbStatus st = check_desc(d, false);
  if (st != TB_OK) return st;
  if (d->a_col_major || d->b_col_major)
    return tb_fail(TB_ERR_UNSUPPORTED, "the weight gradient takes row-major operands");
  if (d->k == 0 || d->n == 0 || d->groups == 0) return TB_OK;
  if (!Gp || !offsets || (d->rows > 0 && (!A || !D)))
    return tb_fail(TB_ERR_INVALID_ARGUMENT, "A, D, G and offsets must not be NULL");
  if (d->rows == 0 && d->beta) return TB_OK;
  Launch L;
  L.a = Operand{A, d->rows, d->k, lda, 1, 0};
  L.b = Operand{D, d->rows, d->n, ldd, 1, 0};
  if ((st = check_ld(lda, d->k, d->rows, "A")) != TB_OK) return st;
  if ((st = check_ld(ldd, d->n, d->rows, "D")) != TB_OK) return st;
  if ((st = check_ld(ldg, d->n, d->k, "G")) != TB_OK) return st;
  const int ce = c_bytes(d->c_dtype);
  if (!al(Gp, ce)) return tb_fail(TB_ERR_INVALID_ARGUMENT, "G is not aligned to its element size");
  if (!al(offsets, d->offsets_long ? 8 : 4))
    return tb_fail(TB_ERR_INVALID_ARGUMENT, "offsets are not aligned to their element size");
  if (d->rows == 0) {  // every gradient is zero: the tiles have no fills
    L.a = Operand{kNothing, 1, 8, 8, 1, 0};
    L.b = Operand{kNothing, 1, 8, 8, 1, 0};
  }
  GParams& p = L.p;
  std::memset(&p, 0, sizeof(p));
  L.el = 2;
  L.bf16 = d->ab_dtype == TB_BF16;
  p.k_grouped = 1;
  p.groups = (int32_t)d->groups;
  p.M = (int32_t)d->k;
  p.N = (int32_t)d->n;
  p.K = (int32_t)d->rows;
  p.offsets = offsets;
  p.offsets_64 = d->offsets_long;
  p.a_mn = 1;
  p.b_kmaj = 0;
  p.fmt = L.bf16 ? 1u : 0u;
  p.beta = d->beta;
  p.c_dtype = d->c_dtype;
  p.C = Gp;
  p.ldc = ldg;
  p.group_c = stride_g;
  p.vec = vector_bytes(Gp, ldg, stride_g, ce);
  return finish(L, d->groups, 0, workspace, workspace_bytes, stream);
}

extern "C" tbStatus tb_matmul_blockscaled(const tb_grouped_desc* d, const void* A, int64_t lda, const tb_scales* sa,
                                          const void* B, int64_t ldb, const tb_scales* sb, void* C, int64_t ldc,
                                          void* workspace, size_t workspace_bytes, void* stream) {
  tb_clear_error();
  if (d && d->groups != 1) return tb_fail(TB_ERR_INVALID_ARGUMENT, "groups must be 1");
  return run_rows(d, true, A, lda, sa, B, ldb, 0, sb, C, ldc, nullptr, workspace, workspace_bytes, stream);
}

extern "C" tbStatus tb_grouped_matmul_blockscaled(const tb_grouped_desc* d, const void* A, int64_t lda,
                                                  const tb_scales* sa, const void* B, int64_t ldb, int64_t stride_b,
                                                  const tb_scales* sb, void* C, int64_t ldc, const void* offsets,
                                                  void* workspace, size_t workspace_bytes, void* stream) {
  tb_clear_error();
  if (d && d->a_col_major) return tb_fail(TB_ERR_UNSUPPORTED, "grouped rows need a row-major A");
  if (d && d->groups > 0 && !offsets) return tb_fail(TB_ERR_INVALID_ARGUMENT, "offsets must not be NULL");
  return run_rows(d, true, A, lda, sa, B, ldb, stride_b, sb, C, ldc, offsets, workspace, workspace_bytes, stream);
}
