// out = residual + scale * act(x w^T + bias), fp16 and bf16, any sizes.
#include "elem16.hpp"
#include "gd_kernels.hpp"

namespace gd {
namespace {

constexpr int kBM = 64, kBN = 64, kBK = 32;

template <int ACT>
__device__ __forceinline__ float activate(float y) {
  if (ACT == GD_ACT_RELU) return y > 0.f ? y : (y <= 0.f ? 0.f : y);
  if (ACT == GD_ACT_GELU) return 0.5f * y * erfcf(-0.70710678f * y);
  if (ACT == GD_ACT_GELU_TANH) return y / (1.0f + expf(-1.5957691216f * (y + 0.044715f * y * y * y)));
  if (ACT == GD_ACT_SILU) return y / (1.0f + expf(-y));
  return y;
}

// A 64 x 64 tile a workgroup of four waves, operands through LDS in steps of
// 32 columns, each element loaded by itself.
template <class T, int ACT>
__global__ __launch_bounds__(256) void projection_kernel(ProjectionArgs a) {
  __shared__ __attribute__((aligned(16))) T xs[kBM][kBK + 8];
  __shared__ __attribute__((aligned(16))) T ws[kBN][kBK + 8];
  typedef typename Elem<T>::v8 v8;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t tiles_n = (a.n + kBN - 1) / kBN;
  const int64_t m0 = blockIdx.x / tiles_n * kBM, n0 = blockIdx.x % tiles_n * kBN;
  float4_t acc[4] = {};
  for (int64_t k0 = 0; k0 < a.k; k0 += kBK) {
    for (int i = t; i < kBM * kBK; i += 256) {
      const int r = i / kBK, c = i % kBK;
      xs[r][c] = m0 + r < a.m && k0 + c < a.k ? ((const T*)a.x)[(m0 + r) * a.ldx + k0 + c] : (T)0.f;
      ws[r][c] = n0 + r < a.n && k0 + c < a.k ? ((const T*)a.w)[(n0 + r) * a.ldw + k0 + c] : (T)0.f;
    }
    __syncthreads();
    const v8 fx = *(const v8*)&xs[16 * wave + (lane & 15)][8 * (lane >> 4)];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const v8 fw = *(const v8*)&ws[16 * j + (lane & 15)][8 * (lane >> 4)];
      acc[j] = Elem<T>::mfma16(fw, fx, acc[j]);  // column of C: x row; rows of C: w rows
    }
    __syncthreads();
  }
  const int64_t row = m0 + 16 * wave + (lane & 15);
  if (row >= a.m) return;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t col = n0 + 16 * j + 4 * (lane >> 4) + e;
      if (col >= a.n) continue;
      float y = acc[j][e];
      if (a.bias) y += (float)((const T*)a.bias)[col];
      y = a.scale * activate<ACT>(y);
      if (a.residual) y += (float)((const T*)a.residual)[row * a.ldr + col];
      ((T*)a.out)[row * a.ldo + col] = (T)y;
    }
}

template <class T>
int launch(const ProjectionArgs& a, hipStream_t stream) {
  const int64_t tiles = (a.m + kBM - 1) / kBM * ((a.n + kBN - 1) / kBN);
  if (tiles > 0x7fffffff) return fail(GD_ERR_SHAPE, "projection: too many tiles");
  const dim3 grid((unsigned)tiles), block(256);
  switch (a.activation) {
    case GD_ACT_RELU: projection_kernel<T, GD_ACT_RELU><<<grid, block, 0, stream>>>(a); break;
    case GD_ACT_GELU: projection_kernel<T, GD_ACT_GELU><<<grid, block, 0, stream>>>(a); break;
    case GD_ACT_GELU_TANH: projection_kernel<T, GD_ACT_GELU_TANH><<<grid, block, 0, stream>>>(a); break;
    case GD_ACT_SILU: projection_kernel<T, GD_ACT_SILU><<<grid, block, 0, stream>>>(a); break;
    default: projection_kernel<T, GD_ACT_NONE><<<grid, block, 0, stream>>>(a);
  }
  GD_LAUNCH_CHECK();
  return GD_OK;
}

}  // namespace

int launch_projection(const ProjectionArgs& a, hipStream_t stream) {
  return a.bf16 ? launch<bf16_t>(a, stream) : launch<half_t>(a, stream);
}

}  // namespace gd
