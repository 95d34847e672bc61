// Softmax attention over packed sequences with grouped heads:
//   out[t, h] = sum_j exp(scale q_t,h . k_j) v_j / sum_j exp(scale q_t,h . k_j)
// over the keys j of t's sequence that it sees.
#include "elem16.hpp"
#include "gd_kernels.hpp"

namespace gd {
namespace {

// Sequence of token t: the last i with off[i] <= t, in [-1, B] (-1: before the
// first, B: behind the last).  One ballot over 64 offsets a round.
__device__ __forceinline__ int sequence_of(const int32_t* off, int B, int t) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int i0 = 0; i0 <= B; i0 += 64) {
    const int c = __popcll(__ballot(i0 + lane <= B && off[i0 + lane] <= t));
    n += c;
    if (c < 64) break;
  }
  return n - 1;
}

__device__ __forceinline__ int clamp_to(int v, int64_t hi) { return v < 0 ? 0 : (v > hi ? (int)hi : v); }

// One wave a query row (token, head): lane l holds elements l, l + 64, ... of
// the row, a running maximum and sum over the keys one after the other.
template <class T, int N>
__global__ __launch_bounds__(256) void packed_attention_kernel(PackedAttentionArgs a) {
  const int64_t item = blockIdx.x * (int64_t)4 + (threadIdx.x >> 6);
  if (item >= a.Tq * a.Hq) return;
  const int lane = threadIdx.x & 63;
  const int t = (int)(item / a.Hq), h = (int)(item % a.Hq), D = (int)a.D;
  T* out = (T*)a.out + t * a.ldo + h * D;
  const int s = sequence_of(a.q_off, (int)a.B, t);
  if (s < 0 || s >= a.B) {
    if (a.zero_rest)
      for (int d = lane; d < D; d += 64) out[d] = (T)0.f;
    return;
  }
  const int q0 = clamp_to(a.q_off[s], a.Tq), q1 = clamp_to(a.q_off[s + 1], a.Tq);
  const int k0 = clamp_to(a.k_off[s], a.Tk), k1 = clamp_to(a.k_off[s + 1], a.Tk);
  const int nk = k1 > k0 ? k1 - k0 : 0;
  int seen = nk;
  if (a.causal) seen = min(nk, nk - (q1 - q0) + (t - q0) + 1);
  const T* q = (const T*)a.q + t * a.qst + h * a.qsh;
  const T* k = (const T*)a.k + k0 * a.kst + h / (a.Hq / a.Hk) * a.ksh;
  const T* v = (const T*)a.v + k0 * a.vst + h / (a.Hq / a.Hk) * a.vsh;
  float qf[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    qf[i] = lane + 64 * i < D ? (float)q[lane + 64 * i] * a.scale : 0.f;
    o[i] = 0.f;
  }
  for (int j = 0; j < seen; ++j) {
    float p = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 64 * i < D) p += qf[i] * (float)k[j * a.kst + lane + 64 * i];
    p = wave_sum(p);
    const float m2 = fmaxf(m, p), base = m2 == -INFINITY ? 0.f : m2;
    const float c = expf(m - base), w = expf(p - base);
    m = m2;
    l = l * c + w;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 64 * i < D) o[i] = o[i] * c + w * (float)v[j * a.vst + lane + 64 * i];
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lane + 64 * i < D) out[lane + 64 * i] = (T)(seen > 0 ? o[i] / l : 0.f);
}

template <class T>
int launch(const PackedAttentionArgs& a, hipStream_t stream) {
  const int64_t blocks = (a.Tq * a.Hq + 3) / 4;
  if (blocks > 0x7fffffff) return fail(GD_ERR_SHAPE, "packed_attention: too many rows");
  const dim3 grid((unsigned)blocks), block(256);
  if (a.D <= 64)
    packed_attention_kernel<T, 1><<<grid, block, 0, stream>>>(a);
  else if (a.D <= 128)
    packed_attention_kernel<T, 2><<<grid, block, 0, stream>>>(a);
  else
    packed_attention_kernel<T, 4><<<grid, block, 0, stream>>>(a);
  GD_LAUNCH_CHECK();
  return GD_OK;
}

}  // namespace

int64_t packed_attention_workspace(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

int launch_packed_attention(const PackedAttentionArgs& a, hipStream_t stream) {
  return a.bf16 ? launch<bf16_t>(a, stream) : launch<half_t>(a, stream);
}

}  // namespace gd
