// Softmax attention over packed sequences with grouped heads:
//   out[t, h] = sum_j exp(scale q_t,h . k_j) v_j / sum_j exp(scale q_t,h . k_j)
// over the keys j of t's sequence that it sees, in one pass over the keys with
// a running maximum and sum in fp32.
//
// The G = heads / kv_heads query heads of one key head are rows of one tile:
// row r of a sequence and key head is token r / G, head r % G of the group, so
// keys and values are read once for the group and a tile's causal border is
// BM / G tokens wide.  Both kernels compute S^T = K Q^T, so that a lane holds
// the scores of one query row: row maxima and sums are in-lane operations and
// one swap between lanes, the rescale factor is the lane's own, and the
// exponentials are the B operand of O^T += V^T P^T as they stand -- the keys of
// a 16- or 32-wide step come in the order of the accumulators, and V^T is read
// from LDS (ds_read_b64_tr_b16) in that same order.
//   * prompt_kernel, many rows a sequence: tiles of 128 rows (four waves of 32)
//     on 32x32x16 MFMA, 64 keys a step, K and V straight from global memory
//     into two LDS stages.  Two workgroups a CU at head width 128.  16,384 tokens
//     of 32 / 8 heads of 128 (bf16) take 2.05 ms, 1.07 PFLOP/s of the pairs that
//     the mask leaves: the matrix cores are busy 52% of the cycles, the vector
//     unit about as long (the exponentials), and the card holds its clock at 1.8
//     to 2.0 GHz: a form with the scores one tile ahead of the softmax took 7%
//     fewer cycles at a clock 7% lower.  At head width 64 the exponentials bound it (0.79 PFLOP/s over
//     8,192 tokens of 16 heads);
//   * token_kernel, few rows a sequence (16 RB for RB = 1, 2, 4): each wave
//     walks 32 keys a step on 16x16x32 MFMA, K from global memory into
//     registers, V into the wave's own LDS; a sequence is cut into chunks of
//     keys and chunks are joined by join_kernel.  HBM bounds it: 16 tokens of 32 /
//     8 heads of 128 against 145,000 keys read 598 MB in 128 us (4.7 TB/s; a large
//     copy reaches 5.1), and the join takes 5 us more.
// The weights are rounded to the tensors' type for P V and, so rounded, summed (in
// fp32): the output stays a mean of the values with weights that are off by at
// most half a step of the type, a constant value comes out as itself, and the
// sum takes half the instructions.  Scores, maxima, sums and the output stay fp32
// until the one rounding at the end.
//
// Workgroups find their sequence from the offsets alone (no plan, no lengths
// on the host): with s tiles of BM rows before offset o being floor(o / BM),
// sequence i starts at slot floor(o_i / BM) + i, and has a slot for each of its
// tiles whatever the lengths are.
#include <algorithm>

#include "elem16.hpp"
#include "gd_kernels.hpp"

namespace gd {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ int clamp_to(int v, int hi) { return v < 0 ? 0 : (v > hi ? hi : v); }

struct Sequence {
  int q0, nq, k0, nk;
};
__device__ __forceinline__ Sequence sequence_of_offsets(const PackedAttentionArgs& a, int q0, int q1, int k0, int k1) {
  Sequence r;
  r.q0 = clamp_to(q0, (int)a.Tq);
  r.nq = max(clamp_to(q1, (int)a.Tq) - r.q0, 0);
  r.k0 = clamp_to(k0, (int)a.Tk);
  r.nk = max(clamp_to(k1, (int)a.Tk) - r.k0, 0);
  return r;
}
__device__ __forceinline__ Sequence sequence_at(const PackedAttentionArgs& a, int s) {
  return sequence_of_offsets(a, a.q_off[s], a.q_off[s + 1], a.k_off[s], a.k_off[s + 1]);
}

// The last entry i of n whose key, key_of(i), is at or before `at`, or -1: each
// round the lanes look at 64 entries that are a 64th of the rest apart, so up to
// 64 entries take one trip to memory and 4,096 two.  (Keys do not decrease; if
// they do, some entry is found.)  After the last round lane l holds what
// key_of(lo + l) has read; `lo` and `count` say of which entries.
template <class Key>
__device__ __forceinline__ int last_at_or_before(int n, int64_t at, Key key_of, int& lo, int& count) {
  const int lane = threadIdx.x & 63;
  lo = 0;
  for (;;) {
    const int step = (n + 63) / 64;
    const bool in = lane * (int64_t)step < n;
    const int64_t key = in ? key_of(lo + lane * step) : INT64_MAX;
    const int c = __popcll(__ballot(in && key <= at));
    if (step == 1) {
      count = n;
      return lo + c - 1;
    }
    if (c == 0) {
      count = 0;
      return lo - 1;
    }
    lo += (c - 1) * step;
    n = min(step, n - (c - 1) * step);
  }
}

// Sequence of a slot: the last i in [0, B] whose first slot, units(offset i) + i,
// is at or before it; -1 before the first, B behind the last sequence (sq is
// set for the others).  `first` is the found sequence's first slot (0 for -1).
// Its offsets come from the lanes that looked.
template <bool BY_KEYS, class Units>
__device__ __forceinline__ int sequence_of_slot(const PackedAttentionArgs& a, int64_t slot, Units units, int64_t& first,
                                                Sequence& sq) {
  const int B = (int)a.B;
  int qo = 0, ko = 0, lo, count;
  auto first_of = [&](int i, int q, int k) { return units(clamp_to(BY_KEYS ? k : q, (int)(BY_KEYS ? a.Tk : a.Tq))) + i; };
  const int s = last_at_or_before(
      B + 1, slot,
      [&](int i) {
        qo = a.q_off[i];
        ko = a.k_off[i];
        return first_of(i, qo, ko);
      },
      lo, count);
  first = 0;
  if (s < 0) return -1;
  const int at = s - lo;  // the lane that has seen it
  if (at >= 0 && at + 1 < count) {
    const int q0 = __builtin_amdgcn_readlane(qo, at), q1 = __builtin_amdgcn_readlane(qo, at + 1);
    const int k0 = __builtin_amdgcn_readlane(ko, at), k1 = __builtin_amdgcn_readlane(ko, at + 1);
    first = first_of(s, q0, k0);
    sq = sequence_of_offsets(a, q0, q1, k0, k1);
  } else {  // (the next offset was not looked at, or there is none)
    first = first_of(s, a.q_off[s], a.k_off[s]);
    if (s < B) sq = sequence_at(a, s);
  }
  return s;
}

// Sequence of a token: the last i with off[i] <= t, in [-1, B].
__device__ __forceinline__ int sequence_of_token(const int32_t* off, int B, int t) {
  int lo, count;
  return last_at_or_before(B + 1, t, [&](int i) { return (int64_t)off[i]; }, lo, count);
}

// What the host chooses for a call from its numbers alone.
struct Plan {
  int rb = 0;           // token_kernel's row blocks of 16; 0: prompt_kernel
  int split = 1;        // prompt_kernel's largest number of parts of the keys
  int chunk = 0;        // token_kernel's keys a workgroup
  int64_t k_slots = 0;  // its chunk slots
  int64_t floats = 0;   // workspace for the parts
};

// Workspace rows: D sums, then the running maximum (in units of log2) and sum.
__host__ __device__ constexpr int part_stride(int D) { return D + 4; }

// LDS rows of DP elements (the power of two at or above D).
constexpr int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256; }

// K rows: 16-byte chunk c of row r at chunk c ^ kswz(r), so that the 16 rows
// that a ds_read_b128 takes at a time at one chunk cover the 64 banks.
template <int DP>
__device__ __forceinline__ int k_swizzle(int row) {
  return DP == 32 ? (row >> 2) & 3 : DP == 64 ? (row >> 1) & 7 : row & 15;
}
// V rows: 32-byte unit u of row r at unit u ^ vswz(r).  A transposing read takes
// four rows at one unit a group of 16 lanes; the prompt kernel's two groups of
// a half wave read neighbouring units of the same rows, the token kernel's read
// the next four rows at the same unit.
template <int DP, bool PROMPT>
__device__ __forceinline__ int v_swizzle(int row) {
  if (PROMPT) return DP == 32 ? 0 : DP == 64 ? ((row >> 1) & 1) << 1 : (row & 3) << 1;
  return DP == 32 ? (row >> 2) & 1 : DP == 64 ? (row >> 1) & 3 : row & 7;
}

typedef short short4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4_t lds_short4_t;

template <class T>
__device__ __forceinline__ typename Elem<T>::v8 read_v(const T* lo, const T* hi) {
  const short4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)lo);
  const short4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)hi);
  typedef short short8_t __attribute__((ext_vector_type(8)));
  const short8_t r = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  return __builtin_bit_cast(typename Elem<T>::v8, r);
}

template <class T>
__device__ __forceinline__ void load_lds16t(const T* g, T* lds_block) {
  __builtin_amdgcn_global_load_lds(reinterpret_cast<const void*>(g), (lds_void_t*)(lds_block), 16, 0, 0);
}

// A hidden key's weight is 0, but 0 times an infinity or NaN of its value is
// not.  Where a row tile had hidden keys and a sum is not finite, the tile is
// computed again with the infinities and NaN of V set to 0 in the steps with
// hidden keys (zero_nonfinite, in LDS), and those of the keys that a row sees
// are added to its sums afterwards (nonfinite_of, from global memory).
template <class T>
__device__ __forceinline__ bool nonfinite_bits(unsigned x) {
  constexpr unsigned kExp = __is_same(T, half_t) ? 0x7C00u : 0x7F80u;
  return (x & kExp) == kExp;
}
// 16 bytes of V in LDS.
template <class T>
__device__ __forceinline__ void zero_nonfinite(T* v) {
  uint4_t u = *reinterpret_cast<const uint4_t*>(v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned lo = u[i] & 0xFFFFu, hi = u[i] >> 16;
    u[i] = (nonfinite_bits<T>(lo) ? 0u : lo) | ((nonfinite_bits<T>(hi) ? 0u : hi) << 16);
  }
  *reinterpret_cast<uint4_t*>(v) = u;
}
// What a value of a seen key adds to its sum if it is not finite.
template <class T>
__device__ __forceinline__ float nonfinite_of(T v) {
  return nonfinite_bits<T>(__builtin_bit_cast(unsigned short, v)) ? (float)v : 0.f;
}

// Max over a lane and its partner l ^ 32, and their sum.
__device__ __forceinline__ float pair_max(float v) {
  const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v),
                                                  false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v),
                                                  false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return __builtin_bit_cast(float, b0) + __builtin_bit_cast(float, b1);
}

// The scale as |c| log2(e); its sign and a scale of 0 are put into Q.
struct Scale {
  float c;
  unsigned flip, keep;  // per 16-bit element: XOR, AND
};
__device__ __forceinline__ Scale scale_of(float scale) {
  Scale s;
  s.c = scale == 0.f ? kLog2e : fabsf(scale) * kLog2e;
  s.flip = scale < 0.f ? 0x80008000u : 0u;
  s.keep = scale == 0.f ? 0u : 0xFFFFFFFFu;
  return s;
}
template <class V8>
__device__ __forceinline__ V8 load_q(const void* p, const Scale& s) {
  uint4_t u = *reinterpret_cast<const uint4_t*>(p);
  u = (u ^ s.flip) & s.keep;
  return __builtin_bit_cast(V8, u);
}

// Rows of no sequence [lo, hi) of one key head's group, set to 0.
template <class T>
__device__ __forceinline__ void zero_rows(const PackedAttentionArgs& a, int hk, int G, int64_t r0, int64_t r1, int tok0,
                                          int tid, int nt) {
  const int D = (int)a.D, units = D / 8;
  for (int64_t i = r0 * units + tid; i < r1 * units; i += nt) {
    const int64_t r = i / units;
    T* dst = (T*)a.out + (tok0 + r / G) * a.ldo + (hk * G + r % G) * D + (i % units) * 8;
    *reinterpret_cast<uint4_t*>(dst) = (uint4_t){0, 0, 0, 0};
  }
}

// First place for the parts of a sequence of more than one chunk whose keys start
// at k0: 2 floor(k0 / chunk).  It has ceil(n / chunk) parts, at most floor(n /
// chunk) + 1 <= 2 floor(n / chunk), so the next such sequence starts behind them,
// and 2 floor(tokens / chunk) + 2 places hold all, however many sequences there are.
__device__ __forceinline__ int64_t part_slot(int k0, int chunk) { return 2 * (int64_t)(k0 / chunk); }

// Keys of a part where a tile of the prompt kernel sees `seen` keys and has
// room for `split` parts: whole steps, at least four.
__device__ __forceinline__ int part_keys(int seen, int split) {
  return split == 1 ? INT_MAX / 64 * 64 : max(((seen + split - 1) / split + 63) / 64 * 64, 256);
}

// ---------------------------------------------------------------------------
// Many rows a sequence.
// ---------------------------------------------------------------------------
template <class T, int D, int NW, bool CAUSAL>
__global__ __launch_bounds__(64 * NW, D <= 128 ? 2 : 1) void prompt_kernel(PackedAttentionArgs a, int G, int Hk,
                                                                            int slots, int split, float* parts) {
  typedef typename Elem<T>::v8 v8;
  typedef typename Elem<T>::v4 v4;
  typedef typename Elem<T>::v2 v2;
  constexpr int BM = 32 * NW, KT = 64, DP = padded(D);
  constexpr int KS = D / 16, DB = D / 32;       // K slices of a score, 32-wide blocks of d
  constexpr int CPR = DP / 8;                   // 16-byte chunks of an LDS row
  constexpr int RPB = 64 / CPR;                 // rows that one DMA instruction of a wave brings
  constexpr int IT = KT * CPR / 64 / NW;        // DMA instructions a wave and tile for K, as many for V
  static_assert(KT * CPR % (64 * NW) == 0, "whole DMA instructions");
  constexpr int STAGE = KT * DP;
  // (an array a stage, named at compile time: the compiler then waits for the DMA
  // into the stage being read and leaves that into the other in flight)
  __shared__ __attribute__((aligned(1024))) T k_lds0[STAGE];
  __shared__ __attribute__((aligned(1024))) T k_lds1[STAGE];
  __shared__ __attribute__((aligned(1024))) T v_lds0[STAGE];
  __shared__ __attribute__((aligned(1024))) T v_lds1[STAGE];

  int idx = blockIdx.x;
  const int hk = idx % Hk;
  idx /= Hk;
  const int part = idx % split;
  // the last tiles of a causal sequence see the most keys: they start first
  const int64_t slot = slots - 1 - idx / split;
  int64_t first;
  // (one more slot in front: rows before the first sequence)
  Sequence sq;
  const int s = slot == 0 ? -1
                          : sequence_of_slot<false>(a, slot - 1, [&](int o) { return (int64_t)o * G / BM; }, first, sq);
  const int tid = threadIdx.x;
  if (s < 0 || s >= a.B) {
    if (a.zero_rest && part == 0) {
      // slots of no sequence share its rows evenly: rows [tile BM, tile BM + BM) of it
      const int tok0 = s < 0 ? 0 : clamp_to(a.q_off[a.B], (int)a.Tq);
      const int tok1 = s < 0 ? clamp_to(a.q_off[0], (int)a.Tq) : (int)a.Tq;
      const int64_t rows = (int64_t)(tok1 - tok0) * G;
      const int64_t tile = s < 0 ? slot : slot - 1 - first;
      const int64_t r0 = tile * BM;
      if (r0 < rows) zero_rows<T>(a, hk, G, r0, r0 + BM < rows ? r0 + BM : rows, tok0, tid, 64 * NW);
    }
    return;
  }
  const int64_t rows = (int64_t)sq.nq * G;
  const int64_t row0 = (slot - 1 - first) * BM;
  if (row0 >= rows) return;

  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, lh = lane >> 5;
  // token and head of this lane's row, held to the sequence's last
  const int64_t tok_first = row0 / G;
  const int rem = (int)(row0 - tok_first * G);
  const int64_t left = rows - row0;
  const int local = wave * 32 + lr;
  const bool live = local < left;
  const int lrow = rem + (live ? local : (int)left - 1);
  const int tok = (int)tok_first + lrow / G, head = hk * G + lrow % G;
  const int shift = sq.nk - sq.nq;
  const int last = CAUSAL ? min(shift + tok, sq.nk - 1) : sq.nk - 1;  // last key this row sees
  // the tile's rows in order: the first sees the fewest keys, the last the most
  const int tile_rows = left < BM ? (int)left : BM;
  const int tok_end = (int)tok_first + (rem + tile_rows - 1) / G;
  const int seen_min = CAUSAL ? max(min(shift + (int)tok_first + 1, sq.nk), 0) : sq.nk;
  const int seen_max = CAUSAL ? max(min(shift + tok_end + 1, sq.nk), 0) : sq.nk;
  const int tiles_all = (seen_max + KT - 1) / KT;
  const int per = part_keys(seen_max, split), parts_used = seen_max > per ? (seen_max + per - 1) / per : 1;
  if (part >= parts_used) return;
  const int t0 = part * (per / KT), t1 = min(t0 + per / KT, tiles_all);
  const int full = seen_min / KT;  // tiles that every row sees whole
  // the same for this wave's rows: tiles that it sees whole, and the first that it does not see at all
  const int wave_tok0 = (int)tok_first + (rem + min(wave * 32, tile_rows - 1)) / G;
  const int wave_tok1 = (int)tok_first + (rem + min(wave * 32 + 31, tile_rows - 1)) / G;
  const int wave_full = CAUSAL ? max(min(shift + wave_tok0 + 1, sq.nk), 0) / KT : sq.nk / KT;
  const int wave_end = wave * 32 >= tile_rows ? 0 : CAUSAL ? max(min(shift + wave_tok1 + 1, sq.nk) + KT - 1, 0) / KT
                                                           : tiles_all;

  const Scale sc = scale_of(a.scale);
  v8 qf[KS];
  {
    const T* q = (const T*)a.q + (int64_t)(sq.q0 + tok) * a.qst + head * a.qsh + 8 * lh;
#pragma unroll
    for (int i = 0; i < KS; ++i) qf[i] = load_q<v8>(q + 16 * i, sc);
  }

  // DMA: instruction i of this wave brings rows 16 wave + i RPB and on of a tile,
  // lane l of it 16 bytes of row l / CPR.  The swizzle of those rows is the
  // lane's own XOR a constant, so that an address is a uniform base and a few
  // bits; offsets within a tile are 32-bit (token strides are below 2^24
  // elements).  Rows past the last key repeat it.
  static_assert(IT * RPB == 16, "a wave brings 16 rows");
  const T* kbase = (const T*)a.k + (int64_t)sq.k0 * a.kst + hk * a.ksh;
  const T* vbase = (const T*)a.v + (int64_t)sq.k0 * a.vst + hk * a.vsh;
  const int dr = lane / CPR, dc = lane % CPR;
  auto issue = [&](const T* base, int64_t stride, int lane_row, int lane_chunk, int tile, T* stage, auto swizzle) {
    const int key0 = tile * KT + 16 * wave, left = sq.nk - key0;
    T* dst = stage + wave * IT * 512;
    if (tile * KT + KT <= sq.nk) {
      const T* src = base + (int64_t)key0 * stride;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = lane_chunk ^ swizzle(i * RPB);
        load_lds16t(src + (uint32_t)(lane_row + (D == DP ? c : min(c, D / 8 - 1)) * 8), dst + i * 512);
        src += RPB * stride;
      }
    } else {
      const T* src = base + (int64_t)min(key0, sq.nk - 1) * stride;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = lane_chunk ^ swizzle(i * RPB), r = max(min(dr + i * RPB, left - 1), 0);
        load_lds16t(src + (uint32_t)(r * (int)stride + (D == DP ? c : min(c, D / 8 - 1)) * 8), dst + i * 512);
      }
    }
  };
  const int k_row = dr * (int)a.kst, v_row = dr * (int)a.vst;
  const int k_chunk = dc ^ k_swizzle<DP>(dr), v_chunk = dc ^ (v_swizzle<DP, true>(dr) << 1);
  auto issue_k = [&](int tile, T* ks) {
    issue(kbase, a.kst, k_row, k_chunk, tile, ks, [](int r) { return k_swizzle<DP>(r); });
  };
  auto issue_v = [&](int tile, T* vs) {
    issue(vbase, a.vst, v_row, v_chunk, tile, vs, [](int r) { return v_swizzle<DP, true>(r) << 1; });
  };

  float16_t o[DB];
  float m, l;  // reference point of the row's exponentials in log2, sum of its weights
  // lanes' places in the LDS rows
  const int tr_row = 4 * lh + ((lane & 15) >> 2), tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  auto v_at = [&](const T* vs, int row, int db) {
    const int d = db * 32 + tr_col;
    return vs + row * DP + (((d >> 4) ^ v_swizzle<DP, true>(row)) << 4) + (d & 15);
  };

  for (bool careful = false;; careful = true) {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    if (t0 < t1) {
      issue_k(t0, k_lds0);
      issue_v(t0, v_lds0);
    }
    auto step = [&](int t, const T* ks, T* vs, T* next_k, T* next_v) {
      wait_vmcnt<0>();
      stage_barrier();  // tile t has landed; every wave is done with the other stage
      if (t + 1 < t1) {
        issue_k(t + 1, next_k);
        issue_v(t + 1, next_v);
      }
      if (careful && t >= full) {
        for (int i = tid; i < STAGE / 8; i += 64 * NW) zero_nonfinite(vs + 8 * i);
        stage_barrier();
      }
      if (t >= wave_end) return;
      // K fragments are read three slices ahead of their MFMAs and V's four MFMAs
      // ahead, the first of them before the softmax, in the order that the group
      // barriers give: left to itself, the compiler reads each just before its MFMA
      // and waits.  (16,384 tokens of 32 / 8 heads of 128 2,115 -> 2,052 us against
      // batches of eight reads, 8,192 of 16 / 4 heads of 256 692 -> 638 us.)
      float16_t x[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[kb][e] = 0.f;
      {
        v8 kf[KS][2];
        auto read_k = [&](int i) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            const int row = kb * 32 + lr;
            kf[i][kb] = *reinterpret_cast<const v8*>(ks + row * DP + (((2 * i + lh) ^ k_swizzle<DP>(row)) << 3));
          }
        };
        constexpr int AH = KS < 3 ? KS : 3;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < AH; ++i) read_k(i);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          if (i + AH < KS) read_k(i + AH);
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) x[kb] = Elem<T>::mfma32(kf[i][kb], qf[i], x[kb]);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * AH, 0);
#pragma unroll
        for (int i = 0; i < KS - AH; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * AH, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
      v8 vf[4 * DB];
      auto read_v_at = [&](int i) {
        const int row = 16 * (i / DB) + tr_row;
        vf[i] = read_v<T>(v_at(vs, row, i % DB), v_at(vs, row + 8, i % DB));
      };
      constexpr int VA = DB < 4 ? DB : 4;
#pragma unroll
      for (int i = 0; i < VA; ++i) read_v_at(i);
      __builtin_amdgcn_sched_barrier(0);
      if (t >= wave_full) {
        const int end = last - t * KT - 4 * lh;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) x[kb][e] = end < kb * 32 + 8 * (e >> 2) + (e & 3) ? -INFINITY : x[kb][e];
      }
      float top = x[0][0];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, x[kb][e]);
      top = pair_max(top) * sc.c;
      // The reference point of a row's exponentials follows its maximum only where
      // that has grown by more than 2^8: weights up to 256 are as exact as those
      // up to 1, and most tiles then leave the sums as they are.  (Each row by its
      // own scores; rows that do not move are multiplied by 1.)
      const bool grow = top > m + 8.0f;
      if (__ballot(grow) != 0) {
        const float next = grow ? top : m;
        const float shrink = next == m ? 1.0f : __builtin_amdgcn_exp2f(m - next);
        m = next;
        l *= shrink;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[i][e] *= shrink;
      }
      const float base = m == -INFINITY ? 0.f : m;
      v8 p[4];
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const v2 w = {(T)__builtin_amdgcn_exp2f(x[i >> 4][i & 15] * sc.c - base),
                      (T)__builtin_amdgcn_exp2f(x[i >> 4][(i & 15) + 1] * sc.c - base)};
        sum[(i >> 1) & 1] = Elem<T>::add2(w, sum[(i >> 1) & 1]);
        p[i >> 3][i & 7] = w[0];
        p[i >> 3][(i & 7) + 1] = w[1];
      }
      l += sum[0] + sum[1];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 4 * DB; ++i) {
        if (i + VA < 4 * DB) read_v_at(i + VA);
        o[i % DB] = Elem<T>::mfma32(vf[i], p[i / DB], o[i % DB]);
      }
#pragma unroll
      for (int i = 0; i < 4 * DB - VA; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, VA, 0);
      __builtin_amdgcn_sched_barrier(0);
    };
    for (int t = t0; t < t1; t += 2) {
      step(t, k_lds0, v_lds0, k_lds1, v_lds1);
      if (t + 1 < t1) step(t + 1, k_lds1, v_lds1, k_lds0, v_lds0);
    }
    if (careful) {
      for (int key = max(full, t0) * KT; key <= min(last, t1 * KT - 1); ++key) {
        const T* v = vbase + (int64_t)key * a.vst + 4 * lh;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[db][e] += nonfinite_of<T>(v[db * 32 + 8 * (e >> 2) + (e & 3)]);
      }
      break;
    }
    if (full >= t1) break;
    float probe = 0.f;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) probe += o[i][e] * 0.f;
    if (!__syncthreads_or(!(probe == 0.f))) break;
  }

  l = pair_sum(l);
  if (!live) return;
  const bool none = last < 0;
  if (parts_used > 1) {
    float* dst = parts + (((int64_t)(sq.q0 + tok) * a.Hq + head) * split + part) * part_stride(D);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4_t*>(dst + db * 32 + 8 * g + 4 * lh) =
            (float4_t){o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
    if (lh == 0) {
      dst[D] = m;
      dst[D + 1] = l;
    }
    return;
  }
  const float inv = none ? 0.f : 1.0f / l;
  T* dst = (T*)a.out + (int64_t)(sq.q0 + tok) * a.ldo + head * D + 4 * lh;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      v4 r;
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = (T)(none ? 0.f : o[db][4 * g + e] * inv);
      *reinterpret_cast<v4*>(dst + db * 32 + 8 * g) = r;
    }
}

// ---------------------------------------------------------------------------
// Few rows a sequence.
// ---------------------------------------------------------------------------
template <class T, int D, int RB, int NW>
__global__ __launch_bounds__(64 * NW) void token_kernel(PackedAttentionArgs a, int G, int Hk, int k_slots, int chunk,
                                                        float* parts) {
  typedef typename Elem<T>::v8 v8;
  constexpr int DP = padded(D), KB = 32, R = 16 * RB;
  constexpr int KS = D / 32, DT = D / 16;
  constexpr int CPR = DP / 8, RPB = 64 / CPR, IT = KB * CPR / 64;
  constexpr int VST = KB * DP;  // elements of a wave's V stage
  constexpr int JR = D + 2;               // a joined row: sums, maximum, sum of weights
  constexpr int JOIN = NW * 16 * JR * 2;  // elements of T that 16 rows of every wave take
  constexpr int V0 = NW * VST > JOIN ? NW * VST : JOIN;
  static_assert((V0 + NW * VST) * 2 <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(1024))) T v_lds0[V0];  // (the joined rows overlay it)
  __shared__ __attribute__((aligned(1024))) T v_lds1[NW * VST];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hk = blockIdx.x % Hk;
  const int64_t slot = blockIdx.x / Hk;
  if (slot >= k_slots) {
    // workgroups behind the last slot: rows of no sequence
    const int extra = (int)(slot - k_slots), n = gridDim.x / Hk - k_slots;
    const int head_end = clamp_to(a.q_off[0], (int)a.Tq), rest = clamp_to(a.q_off[a.B], (int)a.Tq);
    const int64_t per0 = ((int64_t)head_end * G + n - 1) / n, per1 = ((int64_t)(a.Tq - rest) * G + n - 1) / n;
    zero_rows<T>(a, hk, G, extra * per0, min((extra + 1) * per0, (int64_t)head_end * G), 0, tid, 64 * NW);
    zero_rows<T>(a, hk, G, extra * per1, min((extra + 1) * per1, (int64_t)(a.Tq - rest) * G), rest, tid, 64 * NW);
    return;
  }
  int64_t first;
  Sequence sq;
  const int s = sequence_of_slot<true>(a, slot, [&](int o) { return (int64_t)((unsigned)o / (unsigned)chunk); }, first, sq);
  if (s < 0 || s >= a.B) return;
  const int64_t rows = (int64_t)sq.nq * G;
  const int c = (int)(slot - first);
  const bool small = rows <= R;
  if (rows == 0) return;
  // More rows than a tile (a batch of as many queries as sequences, one of which
  // has several): the chunks' workgroups share the row tiles, each over all keys.
  const int slots_used = max((sq.nk + chunk - 1) / chunk, 1);
  if (c >= slots_used) return;
  const int chunks = small ? slots_used : 1;
  const int key_lo = small ? c * chunk : 0, key_hi = chunks > 1 ? min(key_lo + chunk, sq.nk) : sq.nk;
  const int64_t row_step = small ? R : (int64_t)slots_used * R;

  const int lc = lane & 15, lg = lane >> 4;
  const Scale sc = scale_of(a.scale);
  const int shift = sq.nk - sq.nq;
  const T* kbase = (const T*)a.k + (int64_t)sq.k0 * a.kst + hk * a.ksh;
  const T* vbase = (const T*)a.v + (int64_t)sq.k0 * a.vst + hk * a.vsh;
  const int kst = (int)a.kst, vst = (int)a.vst;
  T* const vst0 = v_lds0 + wave * VST;
  T* const vst1 = v_lds1 + wave * VST;
  const int dr = lane / CPR, dc = lane % CPR;
  const int tr_row = 4 * lg + (lc >> 2), tr_col = 4 * (lc & 3);
  auto v_at = [&](const T* vs, int row, int dt) {
    return vs + row * DP + ((dt ^ v_swizzle<DP, false>(row)) << 4) + tr_col;
  };

  for (int64_t row0 = small ? 0 : (int64_t)c * R; row0 < rows; row0 += row_step) {
    int last[RB];
    int last_min = INT_MAX, last_max = -1;
    v8 qf[RB][KS];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const int64_t r = min(row0 + b * 16 + lc, rows - 1);
      const int tok = (int)(r / G), head = hk * G + (int)(r % G);
      last[b] = a.causal ? min(shift + tok, sq.nk - 1) : sq.nk - 1;
      const T* q = (const T*)a.q + (int64_t)(sq.q0 + tok) * a.qst + head * a.qsh + 8 * lg;
#pragma unroll
      for (int i = 0; i < KS; ++i) qf[b][i] = load_q<v8>(q + 32 * i, sc);
    }
    {  // the first row of the tile sees the fewest keys, the last the most
      const int ta = (int)(row0 / G), tb = (int)((min(row0 + R, rows) - 1) / G);
      last_min = a.causal ? min(shift + ta, sq.nk - 1) : sq.nk - 1;
      last_max = a.causal ? min(shift + tb, sq.nk - 1) : sq.nk - 1;
    }
    const int hi = min(key_hi, last_max + 1);
    const int blocks = hi > key_lo ? (hi - key_lo + KB - 1) / KB : 0;

    float4_t o[RB][DT];
    float m[RB], l[RB];
    v8 kf[2][2][KS];  // [stage][16 keys][32 of d]
    auto issue = [&](int blk, auto stage) {
      constexpr int S = decltype(stage)::value;
      const int key0 = key_lo + blk * KB, end = sq.nk - 1 - key0;  // (rows past the last key repeat it)
      const T* kt = kbase + (int64_t)key0 * a.kst;
      const T* vt = vbase + (int64_t)key0 * a.vst;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const T* row = kt + (min(16 * b + lc, end) * kst + 8 * lg);
#pragma unroll
        for (int i = 0; i < KS; ++i) kf[S][b][i] = *reinterpret_cast<const v8*>(row + 32 * i);
      }
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int r = i * RPB + dr;
        const int vc = dc ^ (v_swizzle<DP, false>(r) << 1);
        load_lds16t(vt + (min(r, end) * vst + (D == DP ? vc : min(vc, D / 8 - 1)) * 8),
                    (S == 0 ? vst0 : vst1) + i * 512);
      }
    };
    const int full = (min(last_min + 1, key_hi) - key_lo) / KB;  // blocks that every row sees whole
    for (bool careful = false;; careful = true) {
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        m[b] = -INFINITY;
        l[b] = 0.f;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[b][i] = (float4_t){0.f, 0.f, 0.f, 0.f};
      }
      auto step = [&](int blk, auto stage) {
        constexpr int S = decltype(stage)::value;
        float4_t x[RB][2];
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            x[b][kb] = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < KS; ++i) x[b][kb] = Elem<T>::mfma16(kf[S][kb][i], qf[b][i], x[b][kb]);
          }
        const int key0 = key_lo + blk * KB;
        const bool hidden = blk >= full;
        T* const vs = S == 0 ? vst0 : vst1;
        if (careful && hidden) {
          for (int i = lane; i < VST / 8; i += 64) zero_nonfinite(vs + 8 * i);
          wave_lds_sync();
        }
        v8 p[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          if (hidden) {
            const int end = min(last[b], key_hi - 1);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                x[b][kb][e] = key0 + kb * 16 + 4 * lg + e > end ? -INFINITY : x[b][kb][e];
          }
          float top = x[b][0][0];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, x[b][kb][e]);
          top = fmaxf(m[b], rows_max(top));
          const float base = (top == -INFINITY ? 0.f : top) * sc.c;
          const float shrink = __builtin_amdgcn_exp2f(m[b] * sc.c - base);
          m[b] = top;
          float sum = 0.f;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const typename Elem<T>::v2 w = {(T)__builtin_amdgcn_exp2f(x[b][kb][e] * sc.c - base),
                                              (T)__builtin_amdgcn_exp2f(x[b][kb][e + 1] * sc.c - base)};
              sum = Elem<T>::add2(w, sum);
              p[b][4 * kb + e] = w[0];
              p[b][4 * kb + e + 1] = w[1];
            }
          l[b] = l[b] * shrink + sum;
#pragma unroll
          for (int i = 0; i < DT; ++i) o[b][i] *= shrink;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const v8 vf = read_v<T>(v_at(vs, tr_row, dt), v_at(vs, 16 + tr_row, dt));
#pragma unroll
          for (int b = 0; b < RB; ++b) o[b][dt] = Elem<T>::mfma16(vf, p[b], o[b][dt]);
        }
      };
      // blocks wave, wave + NW, ... of the chunk, one ahead in flight
      std::integral_constant<int, 0> s0;
      std::integral_constant<int, 1> s1;
      int blk = wave;
      if (blk < blocks) issue(blk, s0);
      while (blk < blocks) {
        wait_vmcnt<0>();
        wave_lds_sync();
        if (blk + NW < blocks) issue(blk + NW, s1);
        step(blk, s0);
        blk += NW;
        if (blk >= blocks) break;
        wait_vmcnt<0>();
        wave_lds_sync();
        if (blk + NW < blocks) issue(blk + NW, s0);
        step(blk, s1);
        blk += NW;
      }
      if (careful) {
        for (blk = wave; blk < blocks; blk += NW) {
          if (blk < full) continue;
          for (int key = key_lo + blk * KB; key < min(key_lo + (blk + 1) * KB, key_hi); ++key) {
            const T* v = vbase + (int64_t)key * a.vst + 4 * lg;
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
              for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (key <= last[b]) o[b][i][e] += nonfinite_of<T>(v[16 * i + e]);
          }
        }
        break;
      }
      float probe = 0.f;
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) probe += o[b][i][e] * 0.f;
      if (__ballot(!(probe == 0.f)) == 0) break;
    }

    // ---- join the waves, 16 rows at a time: each writes its rows, then a
    // thread sums four elements of a row over the waves ----
    float* js = reinterpret_cast<float*>(v_lds0);  // [NW][16][JR]
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      __syncthreads();  // every wave is done with its V stages, or with the rows before
      l[b] = rows_sum(l[b]);
      float* dst = js + (wave * 16 + lc) * JR;
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) dst[i * 16 + 4 * lg + e] = o[b][i][e];
      if (lg == 0) {
        dst[D] = m[b] * sc.c;
        dst[D + 1] = l[b];
      }
      __syncthreads();
      const int64_t rb0 = row0 + 16 * b;
      const int n = (int)max(min((int64_t)16, rows - rb0), (int64_t)0);
      for (int i = tid; i < n * (D / 4); i += 64 * NW) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float top = -INFINITY;
        for (int w = 0; w < NW; ++w) top = fmaxf(top, js[(w * 16 + r) * JR + D]);
        const float base = top == -INFINITY ? 0.f : top;
        float4_t v = {0.f, 0.f, 0.f, 0.f};
        float sum = 0.f;
        for (int w = 0; w < NW; ++w) {
          const float* src = js + (w * 16 + r) * JR;
          if (src[D] == -INFINITY) continue;  // (this wave saw no key)
          const float f = __builtin_amdgcn_exp2f(src[D] - base);
          sum += src[D + 1] * f;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] += src[d + e] * f;
        }
        const int64_t row = rb0 + r;
        const int tok = (int)(row / G), head = hk * G + (int)(row % G);
        if (chunks > 1) {
          float* part = parts + (((part_slot(sq.k0, chunk) + c) * Hk + hk) * R + 16 * b + r) * part_stride(D);
          *reinterpret_cast<float4_t*>(part + d) = v;
          if (d == 0) {
            part[D] = top;
            part[D + 1] = sum;
          }
        } else {
          const bool none = sq.nk == 0 || (a.causal && shift + tok < 0);
          typename Elem<T>::v4 out;
#pragma unroll
          for (int e = 0; e < 4; ++e) out[e] = (T)(none ? 0.f : v[e] / sum);
          *reinterpret_cast<typename Elem<T>::v4*>((T*)a.out + (int64_t)(sq.q0 + tok) * a.ldo + head * D + d) = out;
        }
      }
    }
    __syncthreads();  // (the next rows' V stages overlay the sums)
  }
}

// ---------------------------------------------------------------------------
// Joins the parts of a row: a workgroup a query row, whose groups of L lanes
// (four columns a lane) take every (256 / L)-th part.
// ---------------------------------------------------------------------------
constexpr int kPromptWaves = 4;
constexpr int kPromptRows = 32 * kPromptWaves;

// token_rows: rows of the token kernel's tile (it has written the parts of
// sequences that fit one), or 0 where the prompt kernel has.
template <class T, int D>
__global__ __launch_bounds__(256) void join_kernel(PackedAttentionArgs a, int G, int Hk, int token_rows, int chunk,
                                                   int split, const float* parts) {
  constexpr int L = padded(D) / 4, NG = 256 / L, stride = part_stride(D);
  __shared__ float js[NG][D + 4];
  const int item = blockIdx.x, Hq = (int)a.Hq;
  const int t = item / Hq, h = item % Hq;
  const int s = sequence_of_token(a.q_off, (int)a.B, t);
  if (s < 0 || s >= a.B) return;
  const Sequence sq = sequence_at(a, s);
  const int tok = t - sq.q0;
  if (tok < 0 || tok >= sq.nq) return;
  const int64_t rows = (int64_t)sq.nq * G, r = (int64_t)tok * G + h % G;
  int64_t step;
  int n;
  if (token_rows > 0) {
    n = (sq.nk + chunk - 1) / chunk;
    if (n <= 1 || rows > token_rows) return;
    step = (int64_t)Hk * token_rows * stride;
    parts += ((part_slot(sq.k0, chunk) * Hk + h / G) * token_rows + r) * stride;
  } else {
    // (as the prompt kernel counts them for this row's tile)
    const int64_t tile_end = min((r / kPromptRows + 1) * kPromptRows, rows) - 1;
    const int seen = a.causal ? max(min(sq.nk - sq.nq + (int)(tile_end / G) + 1, sq.nk), 0) : sq.nk;
    const int per = part_keys(seen, split);
    if (seen <= per) return;
    n = (seen + per - 1) / per;
    step = stride;
    parts += (int64_t)item * split * stride;
  }
  const int g = threadIdx.x / L, d = threadIdx.x % L * 4;
  float top = -INFINITY, sum = 0.f;
  float4_t v = {0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;  // parts in flight
  for (int i0 = g; i0 < n; i0 += U * NG) {
    float m[U], l[U];
    float4_t x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * NG;
      const float* p = parts + min(i, n - 1) * step;
      m[u] = i < n ? p[D] : -INFINITY;
      l[u] = p[D + 1];
      x[u] = *reinterpret_cast<const float4_t*>(p + (d < D ? d : 0));
    }
    float next = top;
#pragma unroll
    for (int u = 0; u < U; ++u) next = fmaxf(next, m[u]);
    const float base = next == -INFINITY ? 0.f : next;
    const float shrink = __builtin_amdgcn_exp2f(top - base);
    top = next;
    sum *= shrink;
    v *= shrink;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float f = __builtin_amdgcn_exp2f(m[u] - base);  // (0 where a part has no key that this row sees)
      sum = fmaf(l[u], f, sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(x[u][e], f, v[e]);
    }
  }
  if (d < D) *reinterpret_cast<float4_t*>(&js[g][d]) = v;
  if (d == 0) {
    js[g][D] = top;
    js[g][D + 1] = sum;
  }
  __syncthreads();
  if (threadIdx.x >= D / 4) return;
  const int c = threadIdx.x * 4;
  top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NG; ++i) top = fmaxf(top, js[i][D]);
  const float base = top == -INFINITY ? 0.f : top;
  sum = 0.f;
  v = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const float f = __builtin_amdgcn_exp2f(js[i][D] - base);
    const float4_t x = *reinterpret_cast<const float4_t*>(&js[i][c]);
    sum = fmaf(js[i][D + 1], f, sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fmaf(x[e], f, v[e]);
  }
  const bool none = sq.nk == 0 || (a.causal && sq.nk - sq.nq + tok < 0);
  typename Elem<T>::v4 out;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)(none ? 0.f : v[e] / sum);
  *reinterpret_cast<typename Elem<T>::v4*>((T*)a.out + t * a.ldo + h * D + c) = out;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// (pieces of 257, 1 and 64 tokens against 8,448, 4,099 and 64 keys: 39.4, 40.1, 42.2, 41.8 us
// with 8, 12, 16, 32 parts; 8 times 4 tokens against 8,192 keys: 44.4, 38.1, 38.6, 38.2)
constexpr int kMaxSplit = 12;
constexpr int kTokenExtra = 4;  // workgroups a key head for the rows of no sequence

Plan plan_of(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D) {
  Plan p;
  const int64_t G = Hq / Hk;
  const int64_t cus = device_cu_count();
  // The token kernel where no sequence can have more rows than its tile, or
  // where there are as many queries as sequences: one each (should one have
  // more, its tiles take all of its keys).
  const int64_t room = D <= 128 ? 64 : 32;
  if (B > 0 && (Tq * G <= room || (Tq == B && G <= room))) {
    const int64_t rows = Tq == B ? G : Tq * G;
    p.rb = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    // four workgroups a CU over all keys, at least 512 keys each
    const int64_t want = (Tk * Hk + 4 * cus - 1) / (4 * cus);
    p.chunk = (int)std::min<int64_t>(std::max<int64_t>((want + 127) / 128 * 128, 512), 1 << 30);
    p.k_slots = Tk / p.chunk + B + 1;
    if (Tk > p.chunk) p.floats = (2 * (Tk / p.chunk) + 2) * Hk * 16 * p.rb * part_stride((int)D);
    return p;
  }
  // Fewer tiles than two a CU and long keys: each tile's keys are split.
  const int64_t tiles = std::max((Tq * G + kPromptRows - 1) / kPromptRows, std::min(B, Tq)) * Hk;
  if (B > 0 && Tk / B >= 1024 && tiles > 0 && tiles < 2 * cus) {
    p.split = (int)std::max<int64_t>(1, std::min<int64_t>(2 * cus / tiles, kMaxSplit));
    if (p.split > 1) p.floats = Tq * Hq * p.split * part_stride((int)D);
  }
  return p;
}

template <class T, int D>
int launch_prompt(const PackedAttentionArgs& a, const Plan& p, int G, hipStream_t stream) {
  const int64_t slots = a.Tq * G / kPromptRows + a.B + 2;
  const int64_t blocks = slots * a.Hk * p.split;
  if (blocks > 0x7fffffff) return fail(GD_ERR_SHAPE, "packed_attention: too many tiles");
  const dim3 grid((unsigned)blocks), block(64 * kPromptWaves);
  float* parts = static_cast<float*>(a.workspace);
  if (a.causal)
    prompt_kernel<T, D, kPromptWaves, true><<<grid, block, 0, stream>>>(a, G, (int)a.Hk, (int)slots, p.split, parts);
  else
    prompt_kernel<T, D, kPromptWaves, false><<<grid, block, 0, stream>>>(a, G, (int)a.Hk, (int)slots, p.split, parts);
  GD_LAUNCH_CHECK();
  return GD_OK;
}

template <class T, int D, int RB>
int launch_token(const PackedAttentionArgs& a, const Plan& p, int G, hipStream_t stream) {
  constexpr int NW = D <= 128 && RB <= 2 ? 8 : 4;
  const int64_t blocks = (p.k_slots + (a.zero_rest ? kTokenExtra : 0)) * a.Hk;
  if (blocks > 0x7fffffff) return fail(GD_ERR_SHAPE, "packed_attention: too many key chunks");
  token_kernel<T, D, RB, NW><<<dim3((unsigned)blocks), dim3(64 * NW), 0, stream>>>(
      a, G, (int)a.Hk, (int)p.k_slots, p.chunk, static_cast<float*>(a.workspace));
  GD_LAUNCH_CHECK();
  return GD_OK;
}

template <class T, int D>
int launch_sized(const PackedAttentionArgs& a, const Plan& p, hipStream_t stream) {
  const int G = (int)(a.Hq / a.Hk);
  if (p.floats > 0 && a.Tq * a.Hq > 0x7fffffff) return fail(GD_ERR_SHAPE, "packed_attention: too many rows to join");
  if (p.rb == 0) GD_RETURN_IF_ERROR((launch_prompt<T, D>(a, p, G, stream)));
  if (p.rb == 1) GD_RETURN_IF_ERROR((launch_token<T, D, 1>(a, p, G, stream)));
  if (p.rb == 2) GD_RETURN_IF_ERROR((launch_token<T, D, 2>(a, p, G, stream)));
  if constexpr (D <= 128)
    if (p.rb == 4) GD_RETURN_IF_ERROR((launch_token<T, D, 4>(a, p, G, stream)));
  if (p.floats > 0) {
    join_kernel<T, D><<<dim3((unsigned)(a.Tq * a.Hq)), dim3(256), 0, stream>>>(a, G, (int)a.Hk, 16 * p.rb, p.chunk, p.split,
                                                                     static_cast<const float*>(a.workspace));
    GD_LAUNCH_CHECK();
  }
  return GD_OK;
}

template <class T>
int launch(const PackedAttentionArgs& a, const Plan& p, hipStream_t stream) {
  switch (a.D) {
    case 32: return launch_sized<T, 32>(a, p, stream);
    case 64: return launch_sized<T, 64>(a, p, stream);
    case 96: return launch_sized<T, 96>(a, p, stream);
    case 128: return launch_sized<T, 128>(a, p, stream);
    case 192: return launch_sized<T, 192>(a, p, stream);
    default: return launch_sized<T, 256>(a, p, stream);
  }
}

}  // namespace

int64_t packed_attention_workspace(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D) {
  return plan_of(B, Tq, Tk, Hq, Hk, D).floats * (int64_t)sizeof(float);
}

int launch_packed_attention(const PackedAttentionArgs& a, hipStream_t stream) {
  Plan p = plan_of(a.B, a.Tq, a.Tk, a.Hq, a.Hk, a.D);
  if (a.workspace_bytes < p.floats * (int64_t)sizeof(float)) {
    // no room for parts: whole sequences
    p.chunk = 1 << 30;
    p.k_slots = a.Tk / p.chunk + a.B + 1;
    p.split = 1;
    p.floats = 0;
  }
  return a.bf16 ? launch<bf16_t>(a, p, stream) : launch<half_t>(a, p, stream);
}

}  // namespace gd
