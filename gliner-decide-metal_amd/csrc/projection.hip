// out = residual + scale * act(x w^T + bias), fp16 and bf16, any sizes.
//
// Sums are fp32 on the matrix cores (few rows: fp32 multiply-adds), the
// epilogue works on them in fp32 and rounds once.  Kernels:
//   * tile_kernel, many rows: a BM x BN tile of 32x32x16 MFMA sub-tiles, 64-wide
//     K steps brought into LDS by DMA two to four stages deep (rows of 16-byte
//     alignment) or through registers (any alignment), the tile staged through
//     LDS in fp32 so that the epilogue loads the residual and stores the
//     output in whole 16-byte pieces of rows.  8,192 x 4,096 x 16,384 bf16 onto a
//     residual: 854 to 875 us, 1.26 to 1.29 PFLOP/s, bound by the matrix cores and the card's
//     power (the vendor library's product alone: 789 us).  8,192 x 4,096 x 1,024
//     with GELU: 87 us, of which two epilogues of some 14 us run beside no MFMA
//     (74 us without an activation, the library's product alone 59).  777 x 1,000 x 4,096: 16.5 us, 64 x 64 tiles bound
//     by what the L2 gives (16.8 TB/s);
//   * strip_kernel, up to 32 rows (16 x 4,096 x 4,096: 10.6 us): W is read once, straight from global memory
//     into the MFMA operands; the waves of a workgroup share a strip of 16
//     columns and split K;
//   * row_kernel, up to 4 rows: a wave a column, lanes along K; bound by the bytes
//     of w (1 x 16,384 x 4,096: 20 us, 134 MB, part of them from the last-level
//     cache).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "elem16.hpp"
#include "gd_kernels.hpp"

namespace gd {
namespace {

// 0.5 erfc(|y| / sqrt(2)) as t q(t) exp(-y^2 / 2), t = 1 / (1 + 0.436 |y| / sqrt(2)),
// q a minimax fit of erfcx over [0, 10]: with the rounding of the exponent within
// 1e-5 of its value everywhere (a 50th of half a step of fp16), so GELU's lower
// tail keeps its digits.
__device__ __forceinline__ float half_erfc(float y) {
  const float z = fabsf(y);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.436f * 0.70710678f, z, 1.0f));
  float q = -0.07528479f;
  q = fmaf(q, t, 0.18845460f);
  q = fmaf(q, t, 0.00833212f);
  q = fmaf(q, t, 0.13616963f);
  q = fmaf(q, t, 0.11909175f);
  q = fmaf(q, t, 0.12323473f);
  return q * t * __builtin_amdgcn_exp2f(-0.72134752f * z * z);
}

template <int ACT>
__device__ __forceinline__ float activate(float y) {
  if (ACT == GD_ACT_RELU) return y > 0.f ? y : (y <= 0.f ? 0.f : y);
  if (ACT == GD_ACT_GELU) {
    const float h = half_erfc(y);
    return y * (y < 0.f ? h : 1.0f - h);
  }
  // 0.5 (1 + tanh(u)) = 1 / (1 + exp(-2 u))
  if (ACT == GD_ACT_GELU_TANH)
    return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-2.30220820f * fmaf(0.044715f * y * y, y, y)));
  if (ACT == GD_ACT_SILU) return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * y));
  return y;
}

// Eight elements at any alignment of the type; n < 8: the first n, then zeros.
template <class T>
__device__ __forceinline__ typename Elem<T>::v8 load8(const T* p, int n = 8) {
  typename Elem<T>::v8 r;
  if (n >= 8) {
    __builtin_memcpy(&r, p, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = e < n ? p[e] : (T)0.f;
  }
  return r;
}

// Epilogue of N consecutive elements of a row from column col (those below n).
template <class T, int ACT, int N, bool STREAM = false>
__device__ __forceinline__ void finish(const ProjectionArgs& a, int64_t row, int64_t col, const float* acc,
                                       const float* bias) {
  const T* res = a.residual ? (const T*)a.residual + row * a.ldr + col : nullptr;
  T* out = (T*)a.out + row * a.ldo + col;
  if (N == 8 && col + N <= a.n) {
    // One load and one store of 16 bytes at any alignment; STREAM: past the operand
    // tiles in the L2 (8,192 x 4,096 x 1,024: 81.9 -> 75.0 us without an activation, 92.0
    // -> 90.1 with GELU, against stores of 12 and 2 bytes; 75.7 and 91.6 not streamed).
    typedef T piece __attribute__((ext_vector_type(8), aligned(2)));
    piece r, add = {};
    if (res) add = *reinterpret_cast<const piece*>(res);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float y = a.scale * activate<ACT>(acc[e] + bias[e]);
      r[e] = (T)(res ? y + (float)add[e] : y);
    }
    if constexpr (STREAM)
      __builtin_nontemporal_store(r, reinterpret_cast<piece*>(out));
    else
      *reinterpret_cast<piece*>(out) = r;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (col + e < a.n) {
        const float y = a.scale * activate<ACT>(acc[e] + bias[e]);
        out[e] = (T)(res ? y + (float)res[e] : y);
      }
  }
}
template <class T, int N>
__device__ __forceinline__ void load_bias(const ProjectionArgs& a, int64_t col, float* b) {
#pragma unroll
  for (int e = 0; e < N; ++e) b[e] = a.bias && col + e < a.n ? (float)((const T*)a.bias)[col + e] : 0.f;
}

// ---------------------------------------------------------------------------
// Many rows.
// ---------------------------------------------------------------------------
constexpr int kBK = 64;

template <int V>
using ic = std::integral_constant<int, V>;

// LDS rows of 64 elements (128 bytes): 16-byte chunk c of row r at chunk
// c ^ ((r / 2) & 7), so that the 16 rows of a fragment read at one chunk cover
// the 64 banks.
__device__ __forceinline__ int tile_offset(int row, int chunk) { return row * kBK + ((chunk ^ ((row >> 1) & 7)) << 3); }

template <class T, int BM, int BN, int WAVES_M, int NW, int NST, int ACT, bool DMA>
__global__ __launch_bounds__(64 * NW) void tile_kernel(ProjectionArgs a, int tiles_m, int tiles_n) {
  typedef typename Elem<T>::v8 v8;
  constexpr int NT = 64 * NW, WAVES_N = NW / WAVES_M;
  constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, TM = WM / 32, TN = WN / 32;
  constexpr int A_IT = BM / 8 / NW, B_IT = BN / 8 / NW;  // 1 KiB DMA pieces (8 rows) a wave and stage
  constexpr int STAGE = (BM + BN) * kBK;
  constexpr int LPS = A_IT + B_IT;
  static_assert(TM >= 1 && TN >= 1 && A_IT >= 1 && B_IT >= 1, "tile shape");
  // (an array a stage, named at compile time: the compiler then waits for the
  // stage being read and leaves the DMA into the other in flight)
  __shared__ __attribute__((aligned(1024))) T st0[STAGE];
  __shared__ __attribute__((aligned(1024))) T st1[STAGE];
  __shared__ __attribute__((aligned(16))) T st2[NST > 2 ? STAGE : 8];
  __shared__ __attribute__((aligned(16))) T st3[NST > 3 ? STAGE : 8];
  static_assert(NST >= 2 && NST <= 4 && NST * STAGE * 2 <= 160 * 1024 && (NST - 1) * LPS < 64, "stages");
  auto stage = [&](auto i) -> T* {
    constexpr int I = decltype(i)::value % NST;
    if constexpr (I == 0) return st0;
    else if constexpr (I == 1) return st1;
    else if constexpr (I == 2) return st2;
    else return st3;
  };

  // Tile order: workgroups go round the 8 XCDs; each XCD takes a run of the
  // tiles in bands of four tile rows, whose x rows and w rows its L2 then serves.
  const int nwg = tiles_m * tiles_n, xcd = blockIdx.x & 7;
  const int bid = xcd * (nwg >> 3) + min(xcd, nwg & 7) + (blockIdx.x >> 3);
  const int band = bid / (4 * tiles_n), in_band = bid - band * 4 * tiles_n;
  const int gm = min(4, tiles_m - band * 4);
  const int64_t m0 = (int64_t)(band * 4 + in_band % gm) * BM, n0 = (int64_t)(in_band / gm) * BN;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WAVES_N, wn = wave % WAVES_N;
  const int lr = lane & 31, lk = lane >> 5;
  const int mrows = (int)min((int64_t)BM, a.m - m0), nrows = (int)min((int64_t)BN, a.n - n0);
  const T* xt = (const T*)a.x + m0 * a.ldx;
  const T* wt = (const T*)a.w + n0 * a.ldw;

  float16_t acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  v8 fa[2][TM], fb[2][TN];
  const int lane_row = lr * kBK, swz = (lr >> 1) & 7;
  auto read_frags = [&](const T* st, int s, int set) {
    const int lo = lane_row + (((2 * s + lk) ^ swz) << 3);
#pragma unroll
    for (int i = 0; i < TM; ++i) fa[set][i] = *reinterpret_cast<const v8*>(st + (wm * WM + i * 32) * kBK + lo);
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[set][j] = *reinterpret_cast<const v8*>(st + (BM + wn * WN + j * 32) * kBK + lo);
  };
  // w rows are the A operand: a lane holds four consecutive columns of a row
  auto mma = [&](int set) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = Elem<T>::mfma32(fb[set][j], fa[set][i], acc[i][j]);
  };
  // One MFMA, one fragment read, and so on: without an order the two fragment
  // sets fold into one with a wait before each group of MFMAs.
  auto interleave = [&]() {
#pragma unroll
    for (int r = 0; r < TM + TN; ++r) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    if constexpr (TM * TN > TM + TN) __builtin_amdgcn_sched_group_barrier(0x008, TM * TN - (TM + TN), 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  // A step of fewer than 64 columns, or one of unaligned rows: pieces of eight
  // elements through registers, zeros past the last column.
  constexpr int PIECES = (BM + BN) * 8 / NT;
  auto load_step = [&](int64_t k0, v8* r) {
    const int left = (int)min((int64_t)kBK, a.k - k0);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int p = tid + i * NT, row = p >> 3, c = (p & 7) * 8;
      const T* src = row < BM ? xt + min(row, mrows - 1) * a.ldx : wt + min(row - BM, nrows - 1) * a.ldw;
      r[i] = load8(src + k0 + c, left - c);
    }
  };
  auto store_step = [&](T* st, const v8* r) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int p = tid + i * NT;
      *reinterpret_cast<v8*>(st + tile_offset(p >> 3, p & 7)) = r[i];
    }
  };
  auto compute_step = [&](const T* st) {
    read_frags(st, 0, 0);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s < 3) read_frags(st, s + 1, (s + 1) & 1);
      mma(s & 1);
    }
  };

  if constexpr (DMA) {
    const int steps = (int)(a.k / kBK);
    // lane l of a piece brings the chunk that lands at chunk l % 8 of row l / 8
    uint32_t a_off[A_IT], b_off[B_IT];
#pragma unroll
    for (int i = 0; i < A_IT; ++i) {
      const int r = (wave * A_IT + i) * 8 + (lane >> 3);
      a_off[i] = (uint32_t)(min(r, mrows - 1) * (uint32_t)a.ldx + (((lane & 7) ^ ((r >> 1) & 7)) << 3));
    }
#pragma unroll
    for (int i = 0; i < B_IT; ++i) {
      const int r = (wave * B_IT + i) * 8 + (lane >> 3);
      b_off[i] = (uint32_t)(min(r, nrows - 1) * (uint32_t)a.ldw + (((lane & 7) ^ ((r >> 1) & 7)) << 3));
    }
    auto issue = [&](T* st, int step) {
      const T* xs = xt + (int64_t)min(step, steps - 1) * kBK;
      const T* ws = wt + (int64_t)min(step, steps - 1) * kBK;
#pragma unroll
      for (int i = 0; i < A_IT; ++i)
        __builtin_amdgcn_global_load_lds((const void*)(xs + a_off[i]), (lds_void_t*)(st + (wave * A_IT + i) * 512), 16,
                                         0, 0);
#pragma unroll
      for (int i = 0; i < B_IT; ++i)
        __builtin_amdgcn_global_load_lds((const void*)(ws + b_off[i]),
                                         (lds_void_t*)(st + BM * kBK + (wave * B_IT + i) * 512), 16, 0, 0);
    };
    // Every step issues one stage (past the last step that one again, which
    // nobody reads), so each wait is for a constant number of loads.
    auto step = [&](auto i, int t) {
      constexpr int I = decltype(i)::value;
      T* const st = stage(i);
#pragma unroll
      for (int s = 0; s < 3; ++s) {
        read_frags(st, s + 1, (s + 1) & 1);
        mma(s & 1);
        interleave();
      }
      wait_vmcnt<(NST - 2) * LPS>();
      stage_barrier();  // the next stage has landed, this one is in everyone's registers
      issue(st, t + NST);
      read_frags(stage(ic<I + 1>{}), 0, 0);
      mma(1);
      interleave();
    };
    if (steps > 0) {
      issue(st0, 0);
      issue(st1, 1);
      if constexpr (NST > 2) issue(st2, 2);
      if constexpr (NST > 3) issue(st3, 3);
      wait_vmcnt<(NST - 1) * LPS>();
      stage_barrier();
      read_frags(st0, 0, 0);
      // (whole rounds of the stages without a branch, which would cost a wait for
      // every load in flight)
      int t = 0;
      for (; t + NST <= steps; t += NST) {
        step(ic<0>{}, t);
        step(ic<1>{}, t + 1);
        if constexpr (NST > 2) step(ic<2>{}, t + 2);
        if constexpr (NST > 3) step(ic<3>{}, t + 3);
      }
      if (t < steps) step(ic<0>{}, t);
      if constexpr (NST > 2) if (t + 1 < steps) step(ic<1>{}, t + 1);
      if constexpr (NST > 3) if (t + 2 < steps) step(ic<2>{}, t + 2);
      wait_vmcnt<0>();
      __syncthreads();
    }
    if (a.k % kBK != 0) {
      v8 r[PIECES];
      load_step((int64_t)steps * kBK, r);
      store_step(st0, r);
      __syncthreads();
      compute_step(st0);
      __syncthreads();
    }
  } else {
    const int64_t steps = (a.k + kBK - 1) / kBK;
    v8 r[PIECES];
    load_step(0, r);
    for (int64_t t = 0; t < steps; ++t) {
      store_step(st0, r);
      __syncthreads();
      if (t + 1 < steps) load_step((t + 1) * kBK, r);
      compute_step(st0);
      __syncthreads();
    }
  }

  // ---- epilogue: the tile through LDS in fp32, 16-byte unit u of row r at
  // u ^ (r & 15) (16 rows at one unit cover the banks), out in rows ----
  constexpr int RP = STAGE / 2 / BN / 32 * 32;  // rows that a stage holds
  constexpr int UPR = BN / 8;                   // pieces of eight columns a row
  static_assert(RP >= 32 && NT % UPR == 0, "epilogue shape");
  const int u = tid % UPR;
  float bias[8];
  load_bias<T, 8>(a, n0 + 8 * u, bias);
#pragma unroll
  for (int pass = 0; pass < (BM + 2 * RP - 1) / (2 * RP); ++pass) {
    const int first = pass * 2 * RP;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row0 = wm * WM + i * 32 - first;
      if (row0 < 0 || row0 >= 2 * RP) continue;
      float* dst = reinterpret_cast<float*>(row0 < RP ? st0 : st1) + (row0 % RP + lr) * BN;
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int unit = (wn * WN + j * 32) / 4 + 2 * q + lk;
          *reinterpret_cast<float4_t*>(dst + 4 * (unit ^ (lr & 15))) =
              (float4_t){acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        }
    }
    __syncthreads();
    for (int r = tid / UPR; r < 2 * RP && first + r < mrows; r += NT / UPR) {
      const float* src = reinterpret_cast<const float*>(r < RP ? st0 : st1) + (r < RP ? r : r - RP) * BN;
      float v[8];
      *reinterpret_cast<float4_t*>(v) = *reinterpret_cast<const float4_t*>(src + 4 * ((2 * u) ^ (r & 15)));
      *reinterpret_cast<float4_t*>(v + 4) = *reinterpret_cast<const float4_t*>(src + 4 * ((2 * u + 1) ^ (r & 15)));
      finish<T, ACT, 8, BM == 256>(a, m0 + first + r, n0 + 8 * u, v, bias);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Few rows: 16 RB rows of x against a strip of 16 columns (rows of w); the NW
// waves take every NW-th block of 128 columns of K.  Operands come from global memory
// as they are (x from the L2).  Rows past the last repeat it.
// ---------------------------------------------------------------------------
template <class T, int RB, int NW, int ACT>
__global__ __launch_bounds__(64 * NW) void strip_kernel(ProjectionArgs a) {
  typedef typename Elem<T>::v8 v8;
  __shared__ float part[NW][16 * RB][17];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lc = lane & 15, lg = lane >> 4;
  const int64_t n0 = blockIdx.x * (int64_t)16;
  const T* w = (const T*)a.w + min(n0 + lc, a.n - 1) * a.ldw;
  const T* x[RB];
  float4_t acc[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    x[b] = (const T*)a.x + min((int64_t)(16 * b + lc), a.m - 1) * a.ldx;
    acc[b] = (float4_t){0.f, 0.f, 0.f, 0.f};
  }
  // blocks of U steps (whole 128-byte lines of a row) in flight, every NW-th a wave's
  constexpr int U = 4;
  int64_t k0 = wave * (32 * U);
  for (; k0 + 32 * U <= a.k; k0 += NW * 32 * U) {
    v8 fw[U], fx[U][RB];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t k = k0 + i * 32 + 8 * lg;
      fw[i] = load8(w + k);
#pragma unroll
      for (int b = 0; b < RB; ++b) fx[i][b] = load8(x[b] + k);
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int b = 0; b < RB; ++b) acc[b] = Elem<T>::mfma16(fw[i], fx[i][b], acc[b]);
  }
  for (const int64_t end = min(k0 + 32 * U, a.k); k0 < end; k0 += 32) {  // the wave that has the last, short block
    const int64_t k = k0 + 8 * lg;
    const int left = (int)max(min(a.k - k, (int64_t)8), (int64_t)0);
    const v8 fw = load8(w + k, left);
#pragma unroll
    for (int b = 0; b < RB; ++b) acc[b] = Elem<T>::mfma16(fw, load8(x[b] + k, left), acc[b]);
  }
  // lane: row of x lc, columns 4 lg + e
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wave][16 * b + lc][4 * lg + e] = acc[b][e];
  __syncthreads();
  for (int i = tid; i < 16 * RB * 16; i += 64 * NW) {
    const int r = i >> 4, c = i & 15;
    if (r >= a.m || n0 + c >= a.n) continue;
    float v = 0.f;
#pragma unroll
    for (int j = 0; j < NW; ++j) v += part[j][r][c];
    float bias;
    load_bias<T, 1>(a, n0 + c, &bias);
    finish<T, ACT, 1>(a, r, n0 + c, &v, &bias);
  }
}

// ---------------------------------------------------------------------------
// Up to four rows: a wave a column, 64 lanes x 8 elements of K a step.
// ---------------------------------------------------------------------------
template <class T, int M, int ACT>
__global__ __launch_bounds__(256) void row_kernel(ProjectionArgs a) {
  typedef typename Elem<T>::v8 v8;
  const int lane = threadIdx.x & 63;
  const int64_t col = blockIdx.x * (int64_t)4 + (threadIdx.x >> 6);
  if (col >= a.n) return;
  const T* w = (const T*)a.w + col * a.ldw;
  const T* x[M];
#pragma unroll
  for (int m = 0; m < M; ++m) x[m] = (const T*)a.x + min((int64_t)m, a.m - 1) * a.ldx;
  float acc[M] = {};
  auto add = [&](v8 fw, const v8* fx) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[m] = fmaf((float)fw[e], (float)fx[m][e], acc[m]);
  };
  int64_t k = lane * 8;
  for (; k + 512 + 8 <= a.k; k += 1024) {
    v8 fw[2], fx[2][M];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fw[i] = load8(w + k + 512 * i);
#pragma unroll
      for (int m = 0; m < M; ++m) fx[i][m] = load8(x[m] + k + 512 * i);
    }
    add(fw[0], fx[0]);
    add(fw[1], fx[1]);
  }
  for (; k < a.k; k += 512) {
    const int left = (int)min(a.k - k, (int64_t)8);
    v8 fx[M];
    const v8 fw = load8(w + k, left);
#pragma unroll
    for (int m = 0; m < M; ++m) fx[m] = load8(x[m] + k, left);
    add(fw, fx);
  }
#pragma unroll
  for (int m = 0; m < M; ++m) {
    float v = wave_sum_dpp(acc[m]);
    if (lane == m && m < a.m) {
      float bias;
      load_bias<T, 1>(a, col, &bias);
      finish<T, ACT, 1>(a, m, col, &v, &bias);
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
template <class T, int BM, int BN, int WAVES_M, int NW, int NST, int ACT, bool DMA>
int launch_tile(const ProjectionArgs& a, hipStream_t stream) {
  const int64_t tm = (a.m + BM - 1) / BM, tn = (a.n + BN - 1) / BN;
  if (tm * tn > 0x7fffffff || tn > 0x1fffffff) return fail(GD_ERR_SHAPE, "projection: too many tiles");
  tile_kernel<T, BM, BN, WAVES_M, NW, NST, ACT, DMA>
      <<<dim3((unsigned)(tm * tn)), dim3(64 * NW), 0, stream>>>(a, (int)tm, (int)tn);
  GD_LAUNCH_CHECK();
  return GD_OK;
}

// Tiles by the time that they would take, in us: a round of one workgroup a CU
// takes e + s a K step, where two fit, a round of two e2 + s2, and one that is
// partly of two a part of the way between.  The numbers are fits to 14 shapes
// of 128 to 8,192 rows, 1,024 to 4,096 columns and K of 1,024 and 4,096 on 256
// CUs (bf16 onto a residual), within 25% of the times measured and mostly 10%:
// 8,192 x 4,096 x 4,096 takes 238, 292, 355, 436 us with the four tiles, 2,048 x
// 4,096 x 1,024 35, 26, 30, 36, 2,048 x 1,024 x 4,096 83, 42, 25, 28, 512 x
// 1,024 x 4,096 83, 42, 23, 16.
int tile_choice(int64_t m, int64_t n, int64_t k) {
  struct Tile {
    int bm, bn;
    double e, s, e2, s2;  // e2 = 0: one workgroup a CU
  };
  static const Tile kTiles[4] = {{256, 256, 13.5, 1.1, 0, 0.6},  // (s grows by s2 as the CUs fill up)
                                 {128, 128, 3.5, 0.62, 8.5, 0.98},
                                 {128, 64, 4.0, 0.32, 5.0, 0.61},
                                 {64, 64, 3.5, 0.20, 4.5, 0.37}};
  const double cus = device_cu_count(), steps = (double)((k + kBK - 1) / kBK);
  int best = 0;
  double least = 0;
  for (int i = 0; i < 4; ++i) {
    const Tile& t = kTiles[i];
    const double tiles = (double)((m + t.bm - 1) / t.bm) * (double)((n + t.bn - 1) / t.bn);
    const double slots = t.e2 > 0 ? 2 * cus : cus, full = std::floor(tiles / slots), rest = tiles - full * slots;
    double time;
    if (t.e2 > 0) {
      const double one = t.e + t.s * steps, two = t.e2 + t.s2 * steps;
      time = full * two;
      if (rest > cus) time += one + (two - one) * (0.4 + 0.6 * (rest - cus) / cus);
      else if (rest > 0) time += one;
    } else {
      time = full * (t.e + (t.s + t.s2) * steps);
      if (rest > 0) time += t.e + (t.s + t.s2 * rest / cus) * steps;
    }
    if (i == 0 || time < least) best = i, least = time;
  }
  return best;
}

template <class T, int ACT>
int launch_act(const ProjectionArgs& a, hipStream_t stream) {
  if (a.m <= 4) {
    const int64_t blocks = (a.n + 3) / 4;
    if (a.m == 1)
      row_kernel<T, 1, ACT><<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(a);
    else if (a.m == 2)
      row_kernel<T, 2, ACT><<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(a);
    else
      row_kernel<T, 4, ACT><<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(a);
    GD_LAUNCH_CHECK();
    return GD_OK;
  }
  // Strips up to 32 rows and two workgroups a CU, where 64 x 64 tiles leave most
  // CUs idle: 16 x 4,096 x 4,096 10.6 against 15.1 us, 32 rows 13.1 against 15.2, 16
  // x 4,096 x 16,384 38 against 57; 48 rows 18.0 against 15.7, 16 x 16,384 x 4,096
  // 31.6 against 22.8.
  const int64_t strips = (a.n + 15) / 16;
  if (a.m <= 32 && strips <= 2 * device_cu_count()) {
    const dim3 grid((unsigned)strips);
    if (a.m <= 16)
      strip_kernel<T, 1, 8, ACT><<<grid, dim3(512), 0, stream>>>(a);
    else
      strip_kernel<T, 2, 8, ACT><<<grid, dim3(512), 0, stream>>>(a);
    GD_LAUNCH_CHECK();
    return GD_OK;
  }
  // DMA needs rows of 16-byte pieces and tile offsets within 32 bits
  auto rows16 = [](const void* p, int64_t ld) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && ld < (1 << 23);
  };
  if (!rows16(a.x, a.ldx) || !rows16(a.w, a.ldw)) {
    // (128 and 64 wide: 300 x 1,000 x 1,001 27 and 12 us, 3,784 x 502 x 3,126 103 and 40,
    // 148 x 192 x 3,711 79 and 35)
    const int64_t tiles = (a.m + 127) / 128 * ((a.n + 127) / 128);
    return tiles < device_cu_count() ? launch_tile<T, 64, 64, 2, 4, 2, ACT, false>(a, stream)
                                     : launch_tile<T, 128, 128, 2, 4, 2, ACT, false>(a, stream);
  }
  switch (tile_choice(a.m, a.n, a.k)) {
    case 0: return launch_tile<T, 256, 256, 2, 8, 2, ACT, true>(a, stream);
    case 1: return launch_tile<T, 128, 128, 2, 4, 2, ACT, true>(a, stream);
    case 2: return launch_tile<T, 128, 64, 2, 4, 3, ACT, true>(a, stream);
    default: return launch_tile<T, 64, 64, 2, 4, 4, ACT, true>(a, stream);
  }
}

template <class T>
int launch(const ProjectionArgs& a, hipStream_t stream) {
  switch (a.activation) {
    case GD_ACT_RELU: return launch_act<T, GD_ACT_RELU>(a, stream);
    case GD_ACT_GELU: return launch_act<T, GD_ACT_GELU>(a, stream);
    case GD_ACT_GELU_TANH: return launch_act<T, GD_ACT_GELU_TANH>(a, stream);
    case GD_ACT_SILU: return launch_act<T, GD_ACT_SILU>(a, stream);
    default: return launch_act<T, GD_ACT_NONE>(a, stream);
  }
}

}  // namespace

int launch_projection(const ProjectionArgs& a, hipStream_t stream) {
  return a.bf16 ? launch<bf16_t>(a, stream) : launch<half_t>(a, stream);
}

}  // namespace gd
