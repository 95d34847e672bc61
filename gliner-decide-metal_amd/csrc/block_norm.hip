// Between two blocks over rows of a residual stream:
//   h = residual + scale * gate * post(y),   n = pre(h)
// with post() and pre() LayerNorms (biased variance) or RMS norms.
//
// The operator moves y, the residual, h and n once (and a gate row where rows
// have their own) for a dozen operations an element, so HBM bounds it: a row is
// read once into registers, both norms' statistics are sums over those
// registers (the variance of the differences from the mean, not of squares),
// and pre() norms h from its fp32 value.  A row is held by one wave (up to 1,024
// columns: no barrier) or by a workgroup; weights are loaded once by a
// workgroup, which takes every gridDim-th row or group of four rows.  16,384 x
// 4,096 bf16 with an fp32 stream: 805 MB in 154 us, 5.24 TB/s, the rate of a large
// copy; 4,103 x 1,024 fp16 with a gate a row takes less than the host's 10 us for
// the call.
#include <algorithm>

#include "elem16.hpp"
#include "gd_kernels.hpp"

namespace gd {
namespace {

// Sum over the TPR threads of a row.  Two buffers in turn: a buffer is written
// again only after the barrier of the sum between.
template <int TPR>
struct RowSum {
  float* red;
  int turn = 0;
  __device__ __forceinline__ float operator()(float v) {
    v = wave_sum_dpp(v);
    if constexpr (TPR == 64) {
      return v;
    } else {
      constexpr int W = TPR / 64;
      float* buf = red + turn * W;
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
      __syncthreads();
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) s += buf[i];
      return s;
    }
  }
};

// V consecutive elements (8, or 1 for rows of no 16-byte pieces) as fp32.
template <class T, int V>
struct Piece {
  typedef T vec __attribute__((ext_vector_type(V)));
  vec v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const vec*>(p); }
  __device__ __forceinline__ float get(int e) const { return (float)v[e]; }
};
template <class T>
struct Piece<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ float get(int) const { return (float)v; }
};
template <class T, int V>
__device__ __forceinline__ void store_piece(T* p, const float* x) {
  if constexpr (V == 1) {
    *p = (T)x[0];
  } else {
    typedef T vec __attribute__((ext_vector_type(V)));
    vec v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (T)x[e];
    *reinterpret_cast<vec*>(p) = v;
  }
}

// Thread t of a row's TPR holds pieces t, t + TPR, ... (N of them at most).
template <class T, class S, int V, int N, int TPR, bool RMS>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void block_norm_kernel(BlockNormArgs a) {
  constexpr int RPW = TPR < 256 ? 256 / TPR : 1;  // rows at a time
  __shared__ float red[2 * (TPR / 64)];
  RowSum<TPR> row_sum{red};
  const int t = threadIdx.x % TPR;
  const int cols = (int)a.cols;
  const float inv = 1.0f / (float)cols;
  const bool post = a.post_w != nullptr, gated = a.gate != nullptr;
  bool in[N];
#pragma unroll
  for (int i = 0; i < N; ++i) in[i] = (t + i * TPR) * V < cols;

  // weights, kept for all rows
  Piece<T, V> post_w[N], post_b[N], pre_w[N], pre_b[N], gate[N];
  const bool one_gate = gated && a.rows_per_gate >= a.rows;
  auto keep = [&](Piece<T, V>* w, const void* p) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (p && in[i]) w[i].load((const T*)p + (t + i * TPR) * V);
  };
  keep(post_w, a.post_w);
  keep(post_b, a.post_b);
  keep(pre_w, a.pre_w);
  keep(pre_b, a.pre_b);
  if (one_gate) keep(gate, a.gate);

  const int64_t step = (int64_t)gridDim.x * RPW;
  for (int64_t row = blockIdx.x * (int64_t)RPW + threadIdx.x / TPR; row < a.rows; row += step) {
    const T* y = (const T*)a.y + row * a.ldy;
    const S* res = (const S*)a.residual + row * a.ldr;
    float x[N][V];
    Piece<T, V> yv[N];
    Piece<S, V> rv[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (in[i]) {
        yv[i].load(y + (t + i * TPR) * V);
        rv[i].load(res + (t + i * TPR) * V);
      }
    if (gated && !one_gate) {
      const T* g = (const T*)a.gate + (a.rows_per_gate == 1 ? row : row / a.rows_per_gate) * a.ldg;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (in[i]) gate[i].load(g + (t + i * TPR) * V);
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) x[i][e] = in[i] ? yv[i].get(e) : 0.f;

    auto norm = [&](const Piece<T, V>* w, const Piece<T, V>* b, bool biased) {
      float mean = 0.f, s = 0.f;
      if constexpr (!RMS) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int e = 0; e < V; ++e) s += x[i][e];
        mean = row_sum(s) * inv;
        s = 0.f;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if constexpr (!RMS) {
#pragma unroll
          for (int e = 0; e < V; ++e) x[i][e] = in[i] ? x[i][e] - mean : 0.f;
        }
#pragma unroll
        for (int e = 0; e < V; ++e) s = fmaf(x[i][e], x[i][e], s);
      }
      const float rs = rsqrtf(row_sum(s) * inv + a.eps);
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          x[i][e] *= rs * w[i].get(e);
          if (biased) x[i][e] += b[i].get(e);
        }
    };
    if (post) norm(post_w, post_b, a.post_b != nullptr);
    S* h = (S*)a.h + row * a.ldh;
    T* n = (T*)a.n + row * a.ldn;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float z = gated ? x[i][e] * gate[i].get(e) : x[i][e];
        x[i][e] = in[i] ? rv[i].get(e) + a.scale * z : 0.f;
      }
      if (in[i]) store_piece<S, V>(h + (t + i * TPR) * V, x[i]);
    }
    norm(pre_w, pre_b, a.pre_b != nullptr);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (in[i]) store_piece<T, V>(n + (t + i * TPR) * V, x[i]);
  }
}

template <class T, class S, bool RMS, int V, int N, int TPR>
int launch_shape(const BlockNormArgs& a, hipStream_t stream) {
  constexpr int RPW = TPR < 256 ? 256 / TPR : 1, NT = TPR < 256 ? 256 : TPR;
  // workgroups for 32 waves a CU; more rows come in turn
  const int64_t blocks = std::min<int64_t>((a.rows + RPW - 1) / RPW, (int64_t)device_cu_count() * (2048 / NT));
  block_norm_kernel<T, S, V, N, TPR, RMS><<<dim3((unsigned)blocks), dim3(NT), 0, stream>>>(a);
  GD_LAUNCH_CHECK();
  return GD_OK;
}

template <class T, class S, bool RMS>
int launch(const BlockNormArgs& a, hipStream_t stream) {
  auto p16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const bool pieces = a.cols % 8 == 0 && p16(a.y) && p16(a.residual) && p16(a.gate) && p16(a.post_w) &&
                      p16(a.post_b) && p16(a.pre_w) && p16(a.pre_b) && p16(a.h) && p16(a.n) && a.ldy % 8 == 0 &&
                      a.ldr % 8 == 0 && a.ldg % 8 == 0 && a.ldh % 8 == 0 && a.ldn % 8 == 0;
  if (pieces) {
    if (a.cols <= 512) return launch_shape<T, S, RMS, 8, 1, 64>(a, stream);
    if (a.cols <= 1024) return launch_shape<T, S, RMS, 8, 2, 64>(a, stream);
    if (a.cols <= 2048) return launch_shape<T, S, RMS, 8, 1, 256>(a, stream);
    if (a.cols <= 4096) return launch_shape<T, S, RMS, 8, 2, 256>(a, stream);
    if (a.cols <= 8192) return launch_shape<T, S, RMS, 8, 2, 512>(a, stream);
    if (a.cols <= 16384) return launch_shape<T, S, RMS, 8, 2, 1024>(a, stream);
    return launch_shape<T, S, RMS, 8, 4, 1024>(a, stream);
  }
  if (a.cols <= 256) return launch_shape<T, S, RMS, 1, 4, 64>(a, stream);
  if (a.cols <= 1024) return launch_shape<T, S, RMS, 1, 4, 256>(a, stream);
  if (a.cols <= 4096) return launch_shape<T, S, RMS, 1, 8, 512>(a, stream);
  if (a.cols <= 8192) return launch_shape<T, S, RMS, 1, 8, 1024>(a, stream);
  return launch_shape<T, S, RMS, 1, 32, 1024>(a, stream);
}

template <class T>
int launch_typed(const BlockNormArgs& a, hipStream_t stream) {
  if (a.stream_f32) return a.rms ? launch<T, float, true>(a, stream) : launch<T, float, false>(a, stream);
  return a.rms ? launch<T, T, true>(a, stream) : launch<T, T, false>(a, stream);
}

}  // namespace

int launch_block_norm(const BlockNormArgs& a, hipStream_t stream) {
  return a.bf16 ? launch_typed<bf16_t>(a, stream) : launch_typed<half_t>(a, stream);
}

}  // namespace gd
