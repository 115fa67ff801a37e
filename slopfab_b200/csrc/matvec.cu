// y = act(W x + b) for few rows of x, W as stored in 4 bits with group scales (NVFP4, NF4).
//
// Bound by the weight's bytes: N K / 2 codes and N K / 16 (NVFP4) or about N K / 64 (NF4) scale bytes are read once, whatever the
// number of rows. Weight values are used as the bytes define them (code x group scale x tensor scale, without the rounding to
// bf16 that the dense form has), sums are fp32, and the result is rounded once, behind bias and activation.
#include <cuda_bf16.h>

#include <stdexcept>
#include <string>

#include "codec.cuh"
#include "kernels.cuh"
#include "ptx.cuh"
#include "runtime.h"

namespace sfq {
namespace {

using namespace ptx;

constexpr int kWarps = 8;
constexpr int kMostRows = 16;  // rows of x in one launch

__device__ __forceinline__ float activated(float z, float up, int act) {
  if (act == SFQ_ACT_GELU_TANH) return 0.5f * z * (1.0f + tanhf(0.7978845608028654f * (z + 0.044715f * z * z * z)));
  if (act == SFQ_ACT_SWIGLU) return z / (1.0f + __expf(-z)) * up;
  return z;
}

// One warp per output column (a pair of weight rows for SwiGLU), lanes along K.
template <bool NF4>
__global__ void __launch_bounds__(kWarps * 32) matvec_kernel(MatvecArgs g) {
  grid_dependency_release();
  grid_dependency_wait();
  __shared__ float map[16];
  if (threadIdx.x < 16) map[threadIdx.x] = NF4 ? g.map[threadIdx.x] : e2m1_decode(threadIdx.x);
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int col = blockIdx.x * kWarps + int(threadIdx.x >> 5);
  const int cols = g.act == SFQ_ACT_SWIGLU ? g.out / 2 : g.out;
  if (col >= cols) return;
  const int halves = g.act == SFQ_ACT_SWIGLU ? 2 : 1;
  float sum[2][kMostRows];
  for (int h = 0; h < 2; ++h)
    for (int r = 0; r < kMostRows; ++r) sum[h][r] = 0.0f;
  for (int h = 0; h < halves; ++h) {
    const int n = col + h * cols;
    const uint8_t* w = g.data + size_t(n) * (g.in / 2);
    for (int k = lane * 16; k < g.in; k += 512) {
      float scale;
      if (NF4) {
        const size_t block = (size_t(n) * g.in + k) >> g.block_shift;
        scale = fmaf(g.nested_map[g.scale[block]], g.nested_absmax[block >> g.nested_shift], g.offset);
      } else {
        scale = e4m3_decode(g.scale[nvfp4_scale_offset(n, k / 16, g.in / 16)]);
      }
      const uint2 raw = *reinterpret_cast<const uint2*>(w + k / 2);
      float v[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t byte = ((i < 4 ? raw.x : raw.y) >> (8 * (i & 3))) & 0xFFu;
        v[2 * i] = map[byte >> 4] * scale;
        v[2 * i + 1] = map[byte & 15u] * scale;
      }
#pragma unroll
      for (int r = 0; r < kMostRows; ++r) {
        if (r >= g.rows) break;
        const __nv_bfloat16* x = g.x + size_t(r) * g.in + k;
        for (int i = 0; i < 16; ++i) sum[h][r] = fmaf(v[i], __bfloat162float(x[i]), sum[h][r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kMostRows; ++r) {
    if (r >= g.rows) break;
    float z[2];
    for (int h = 0; h < halves; ++h) {
      float s = sum[h][r];
      for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      const int n = col + h * cols;
      const float b = g.bias == nullptr ? 0.0f : g.bias_is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(g.bias)[n]) : static_cast<const float*>(g.bias)[n];
      z[h] = fmaf(s, g.global_scale, b);
    }
    if (lane == 0) g.y[size_t(r) * cols + col] = __float2bfloat16(activated(z[0], z[halves - 1], g.act));
  }
}

int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}
bool power_of_two(int v) { return v > 0 && (v & (v - 1)) == 0; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace

void linear_matvec(MatvecArgs g, int nf4_block, int nf4_nested_block, cudaStream_t stream) {
  if (g.rows <= 0) return;
  if (g.out <= 0 || g.in <= 0) throw std::invalid_argument("matvec: features must be positive");
  if (!g.x || !g.y || !g.data) throw std::invalid_argument("matvec: null operand");
  if (g.nf4) {
    if (!g.scale || !g.map || !g.nested_map || !g.nested_absmax) throw std::invalid_argument("matvec: nf4 weight without complete double-quant state");
    if (!power_of_two(nf4_block) || nf4_block < 32 || !power_of_two(nf4_nested_block)) throw std::invalid_argument("matvec: nf4 blocks must be powers of two, of 32 elements at least");
    if (g.in % 32 != 0) throw std::invalid_argument("matvec: nf4 needs in_features % 32 == 0");
    g.block_shift = log2_of(nf4_block), g.nested_shift = log2_of(nf4_nested_block);
    g.global_scale = 1.0f;
  } else {
    if (!g.scale) throw std::invalid_argument("matvec: block_scale is null");
    if (g.out % 128 != 0 || g.in % 64 != 0) throw std::invalid_argument("matvec: nvfp4 needs out_features % 128 == 0 and in_features % 64 == 0");
    if (!aligned(g.scale, 4)) throw std::invalid_argument("matvec: block_scale must be 4-byte aligned");
  }
  if (g.act == SFQ_ACT_SWIGLU && g.out % 2 != 0) throw std::invalid_argument("matvec: SwiGLU needs an even out_features");
  if (!aligned(g.data, 16) || !aligned(g.x, 16) || !aligned(g.y, 2)) throw std::invalid_argument("matvec: x and the weight must be 16-byte aligned");
  const int cols = g.act == SFQ_ACT_SWIGLU ? g.out / 2 : g.out;
  {
    const auto x0 = reinterpret_cast<uintptr_t>(g.x), x1 = x0 + size_t(g.rows) * g.in * 2, y0 = reinterpret_cast<uintptr_t>(g.y), y1 = y0 + size_t(g.rows) * cols * 2;
    if (x0 < y1 && y0 < x1) throw std::invalid_argument("matvec: x and y may not overlap");
  }
  const int rows = g.rows;
  for (int r = 0; r < rows; r += kMostRows) {
    MatvecArgs part = g;
    part.rows = rows - r < kMostRows ? rows - r : kMostRows;
    part.x = g.x + size_t(r) * g.in;
    part.y = g.y + size_t(r) * cols;
    const cudaError_t e = launch_overlapped(size_t(g.out) * g.in / 2, g.nf4 ? matvec_kernel<true> : matvec_kernel<false>, dim3((cols + kWarps - 1) / kWarps),
                                            dim3(kWarps * 32), 0, stream, part);
    if (e != cudaSuccess) throw std::runtime_error(std::string("matvec: launch failed: ") + cudaGetErrorString(e));
  }
}

}  // namespace sfq
