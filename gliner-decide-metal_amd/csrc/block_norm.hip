// Between two blocks over rows of a residual stream:
//   h = residual + scale * gate * post(y),   n = pre(h)
// with post() and pre() LayerNorms (biased variance) or RMS norms.
//
// The operator moves y, the residual, h and n once (and a gate row where rows
// have their own) and computes a dozen operations an element, so HBM bounds
// it: a row is read into registers once, both norms' statistics are sums over
// those registers, and h is normed from its fp32 value before either is
// rounded.
#include "elem16.hpp"
#include "gd_kernels.hpp"

namespace gd {
namespace {

// One workgroup of 256 threads a row, elements t, t + 256, ... of the row in
// thread t's registers.
constexpr int kThreads = 256;

__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < kThreads / 64; ++i) s += red[i];
  return s;
}

template <class T, class S, int N, bool RMS>
__global__ __launch_bounds__(kThreads) void block_norm_kernel(BlockNormArgs a) {
  __shared__ float red[kThreads / 64];
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x, cols = (int)a.cols;
  const T* y = (const T*)a.y + row * a.ldy;
  const S* res = (const S*)a.residual + row * a.ldr;
  const T* gate = a.gate ? (const T*)a.gate + row / a.rows_per_gate * a.ldg : nullptr;
  const float inv = 1.0f / (float)cols;
  float x[N];
  // statistics of x over the row: the mean (0 for RMS) and 1 / spread
  auto norm = [&](const T* w, const T* b) {
    float s = 0.f, mean = 0.f;
    if (!RMS) {
#pragma unroll
      for (int i = 0; i < N; ++i) s += t + i * kThreads < cols ? x[i] : 0.f;
      mean = block_sum(s, red) * inv;
    }
    s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += t + i * kThreads < cols ? (x[i] - mean) * (x[i] - mean) : 0.f;
    const float rs = rsqrtf(block_sum(s, red) * inv + a.eps);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = t + i * kThreads;
      if (c < cols) x[i] = (x[i] - mean) * rs * (float)w[c] + (b ? (float)b[c] : 0.f);
    }
  };
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = t + i * kThreads < cols ? (float)y[t + i * kThreads] : 0.f;
  if (a.post_w) norm((const T*)a.post_w, (const T*)a.post_b);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = t + i * kThreads;
    if (c < cols) x[i] = (float)res[c] + a.scale * (gate ? x[i] * (float)gate[c] : x[i]);
  }
  float hv[N];
#pragma unroll
  for (int i = 0; i < N; ++i) hv[i] = x[i];
  norm((const T*)a.pre_w, (const T*)a.pre_b);
  S* h = (S*)a.h + row * a.ldh;
  T* n = (T*)a.n + row * a.ldn;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = t + i * kThreads;
    if (c < cols) {
      h[c] = (S)hv[i];
      n[c] = (T)x[i];
    }
  }
}

template <class T, class S, bool RMS>
int launch(const BlockNormArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)a.rows);
  if (a.cols <= 4 * kThreads)
    block_norm_kernel<T, S, 4, RMS><<<grid, kThreads, 0, stream>>>(a);
  else if (a.cols <= 32 * kThreads)
    block_norm_kernel<T, S, 32, RMS><<<grid, kThreads, 0, stream>>>(a);
  else
    block_norm_kernel<T, S, 128, RMS><<<grid, kThreads, 0, stream>>>(a);
  GD_LAUNCH_CHECK();
  return GD_OK;
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
