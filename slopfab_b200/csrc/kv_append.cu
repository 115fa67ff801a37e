// New tokens' keys and values into the paged 8-bit cache, with head norm and rotation of q and k on the way.
//
// Bound by memory: q, k and v rows are read once, q is written as bf16, k and v as e4m3. A (page, head) has one scale, the smallest
// power of two s with |x| <= 448 s for all its tokens so far; a power of two, because a page that is filled token by token has its scale
// raised now and then, and the codes that are there then only move by whole exponents (rounded again where they become subnormal).
#include <cuda_fp8.h>

#include <stdexcept>
#include <string>

#include "codec.cuh"
#include "kv_cache.cuh"
#include "ptx.cuh"
#include "runtime.h"

namespace sfq {
namespace {

using namespace ptx;

constexpr int kThreads = 256;
constexpr int kLanes = 16;                     // threads of one head's vector, 8 channels each
constexpr int kAtOnce = kThreads / kLanes;     // vectors a block works on at once
constexpr int kQueryHeads = 8;                 // query heads a block rotates

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
}

// The smallest power of two s, 2^-100 at least, with amax <= 448 s.
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = int(u >> 23) - 135 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);  // 448 = 1.75 x 2^8
  return __uint_as_float(uint32_t(max(e, -100) + 127) << 23);
}

__device__ __forceinline__ uint8_t encode(float v) { return uint8_t(__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3)); }

__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.0f;
}

// Norm (weight may be null) and rotation of one head vector spread over 16 lanes, in fp32. All 32 lanes of a warp take part.
__device__ __forceinline__ void norm_rope(float (&v)[8], const __nv_bfloat16* weight, float eps, const RotaryArgs& r, long long position) {
  const int l = threadIdx.x & 15;
  if (weight != nullptr) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(v[i], v[i], sum);
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    const float inv = rsqrtf(fmaf(sum, 1.0f / kKvHeadDim, eps));
    float w[8];
    load8(weight + l * 8, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * w[i];
  }
  if (r.cos != nullptr) {
    const int half = r.rotary_dim / 16;  // lanes of one half
    const bool low = l < half, turns = l < 2 * half;
    const int partner = (threadIdx.x & 16) | (low ? l + half : turns ? l - half : l);
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(0xffffffffu, v[i], partner);
    if (turns) {
      const size_t at = size_t(position) * (half * 8) + (low ? l : l - half) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float c = r.cos[at + i], s = r.sin[at + i];
        v[i] = low ? fmaf(v[i], c, -(o[i] * s)) : fmaf(v[i], c, o[i] * s);
      }
    }
  }
}

// blockIdx.x: page of the sequence's new tokens; y: sequence; z: a kv head, behind them groups of query heads.
__global__ void __launch_bounds__(kThreads) kv_append_kernel(KvCacheView c, RotaryArgs rot, AppendArgs g) {
  grid_dependency_release();
  grid_dependency_wait();
  __shared__ float peak[2][kThreads / 32];
  const int page_size = 1 << c.page_shift;
  const int vector = threadIdx.x / kLanes, l = threadIdx.x & 15;
  for (int b = blockIdx.y; b < c.batch; b += gridDim.y) {
    const KvSequence s = kv_sequence(c, b);
    const long long past = s.length - s.rows;  // position of the first new token
    const long long first_page = (past > 0 ? past : 0) >> c.page_shift, last_page = (s.length - 1) >> c.page_shift;
    for (long long p = first_page + blockIdx.x; s.rows > 0 && p <= last_page; p += gridDim.x) {
      const long long begin = max(p << c.page_shift, past), end = min((p + 1) << c.page_shift, s.length);
      const int tokens = int(end - begin), row0 = s.row0 + int(begin - past);
      auto position = [&](int i) -> long long { return rot.position != nullptr ? rot.position[row0 + i] : begin + i; };
      auto turn = [&](float (&v)[8], const __nv_bfloat16* weight, int i) {
        long long at = rot.cos != nullptr ? position(i) : 0;
        if (rot.cos != nullptr && (at < 0 || at >= rot.table_rows)) {
          atomicCAS(c.status, 0, kKvBadPosition);
          at = 0;
        }
        norm_rope(v, weight, rot.eps, rot, at);
      };
      if (int(blockIdx.z) >= c.kv_heads) {
        const int head0 = (blockIdx.z - c.kv_heads) * kQueryHeads, heads = min(kQueryHeads, g.heads - head0);
        for (int j = vector; j - vector < tokens * heads; j += kAtOnce) {  // whole warps
          const bool live = j < tokens * heads;
          const int i = live ? j / heads : 0, h = live ? j % heads : 0;
          float v[8];
          load8(g.q + size_t(row0 + i) * g.ld_q + (head0 + h) * kKvHeadDim + l * 8, v);
          turn(v, rot.q_norm, i);
          if (live) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
              w[k] = *reinterpret_cast<const uint32_t*>(&t);
            }
            *reinterpret_cast<uint4*>(g.q_out + size_t(row0 + i) * g.ld_q_out + (head0 + h) * kKvHeadDim + l * 8) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        continue;
      }
      const int head = blockIdx.z;
      const int page = kv_page(c, b, p);
      if (page < 0) continue;
      const size_t block = size_t(page) * c.kv_heads + head;
      uint8_t* kc = c.k + block * page_size * kKvHeadDim;
      uint8_t* vc = c.v + block * page_size * kKvHeadDim;
      const int slot0 = int(begin & (page_size - 1));
      float k_peak = 0.0f, v_peak = 0.0f;
      auto load_k = [&](float (&v)[8], int i) {
        load8(g.k + size_t(row0 + i) * g.ld_kv + head * kKvHeadDim + l * 8, v);
        turn(v, rot.k_norm, i);
      };
      for (int j = vector; j - vector < tokens; j += kAtOnce) {
        const int i = min(j, tokens - 1);
        float k[8], v[8];
        load_k(k, i);
        load8(g.v + size_t(row0 + i) * g.ld_kv + head * kKvHeadDim + l * 8, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) k_peak = fmaxf(k_peak, finite_abs(k[e])), v_peak = fmaxf(v_peak, finite_abs(v[e]));
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) {
        k_peak = fmaxf(k_peak, __shfl_xor_sync(0xffffffffu, k_peak, off));
        v_peak = fmaxf(v_peak, __shfl_xor_sync(0xffffffffu, v_peak, off));
      }
      if ((threadIdx.x & 31) == 0) peak[0][threadIdx.x / 32] = k_peak, peak[1][threadIdx.x / 32] = v_peak;
      __syncthreads();
      for (int w = 0; w < kThreads / 32; ++w) k_peak = fmaxf(k_peak, peak[0][w]), v_peak = fmaxf(v_peak, peak[1][w]);
      const float old_k = slot0 > 0 ? c.k_scale[block] : 0.0f, old_v = slot0 > 0 ? c.v_scale[block] : 0.0f;
      const float new_k = fmaxf(old_k, scale_for(k_peak)), new_v = fmaxf(old_v, scale_for(v_peak));
      __syncthreads();
      if (threadIdx.x == 0) c.k_scale[block] = new_k, c.v_scale[block] = new_v;
      if (new_k != old_k)
        for (int i = threadIdx.x; i < slot0 * kKvHeadDim; i += kThreads) kc[i] = encode(e4m3_decode(kc[i]) * old_k / new_k);
      if (new_v != old_v)
        for (int i = threadIdx.x; i < slot0 * kKvHeadDim; i += kThreads) {
          uint8_t* at = vc + size_t(i / slot0) * page_size + i % slot0;
          *at = encode(e4m3_decode(*at) * old_v / new_v);
        }
      for (int j = vector; j - vector < tokens; j += kAtOnce) {
        const bool live = j < tokens;
        const int i = min(j, tokens - 1), slot = slot0 + i;
        float k[8], v[8];
        load_k(k, i);
        load8(g.v + size_t(row0 + i) * g.ld_kv + head * kKvHeadDim + l * 8, v);
        if (live) {
          uint32_t w[2] = {0, 0};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            w[e / 4] |= uint32_t(encode(k[e] / new_k)) << (8 * (e % 4));
            vc[size_t(l * 8 + e) * page_size + slot] = encode(v[e] / new_v);
          }
          *reinterpret_cast<uint2*>(kc + size_t(slot) * kKvHeadDim + l * 8) = make_uint2(w[0], w[1]);
        }
      }
    }
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

void kv_check(const KvCacheView& c, int head_dim) {
  if (head_dim != kKvHeadDim) throw std::invalid_argument("kv cache: only head_dim 128 is built");
  if (c.page_shift < 4 || c.page_shift > 8) throw std::invalid_argument("kv cache: page_size must be 16, 32, 64, 128 or 256");
  if (c.num_pages <= 0 || c.kv_heads <= 0 || c.batch <= 0 || c.max_pages <= 0 || c.max_new <= 0 || c.max_len <= 0)
    throw std::invalid_argument("kv cache: extents must be positive");
  if (c.kv_heads > 32768) throw std::invalid_argument("kv cache: too many heads");
  if (!c.k || !c.v || !c.k_scale || !c.v_scale || !c.table || !c.seq_len || !c.row_start) throw std::invalid_argument("kv cache: null buffer");
  if (!aligned16(c.k) || !aligned16(c.v)) throw std::invalid_argument("kv cache: the pools must be 16-byte aligned");
}

void kv_append(KvCacheView c, int head_dim, const RotaryArgs& rot, const AppendArgs& g, cudaStream_t stream) {
  kv_check(c, head_dim);
  if (c.rows <= 0) return;
  if (!g.k || !g.v || (g.heads > 0 && (!g.q || !g.q_out))) throw std::invalid_argument("kv append: null operand");
  if (g.heads < 0 || g.heads > 32768) throw std::invalid_argument("kv append: bad number of query heads");
  if (g.ld_kv < c.kv_heads * kKvHeadDim || g.ld_kv % 8 != 0 || !aligned16(g.k) || !aligned16(g.v) ||
      (g.heads > 0 && (g.ld_q < g.heads * kKvHeadDim || g.ld_q_out < g.heads * kKvHeadDim || g.ld_q % 8 != 0 || g.ld_q_out % 8 != 0 || !aligned16(g.q) || !aligned16(g.q_out))))
    throw std::invalid_argument("kv append: row pitches must cover heads * 128 columns and keep 16-byte alignment");
  if ((rot.cos == nullptr) != (rot.sin == nullptr)) throw std::invalid_argument("kv append: cos and sin come together");
  if (rot.cos != nullptr && (rot.rotary_dim <= 0 || rot.rotary_dim > kKvHeadDim || rot.rotary_dim % 16 != 0 || rot.table_rows <= 0))
    throw std::invalid_argument("kv append: rotary_dim must be a multiple of 16 up to 128, with at least one table row");
  if (!aligned16(rot.cos) || !aligned16(rot.sin) || !aligned16(rot.q_norm) || !aligned16(rot.k_norm)) throw std::invalid_argument("kv append: tables and norm weights must be 16-byte aligned");
  c.status = device_status_word();
  const int pages = (c.max_new + (1 << c.page_shift) - 2) / (1 << c.page_shift) + 1;
  const int groups = (g.heads + kQueryHeads - 1) / kQueryHeads;
  const size_t bytes = size_t(c.rows) * (g.heads * 4 + c.kv_heads * 6) * kKvHeadDim;
  const cudaError_t e = launch_overlapped(bytes, kv_append_kernel, dim3(pages, c.batch < 65535 ? c.batch : 65535, c.kv_heads + groups), dim3(kThreads), 0, stream, c, rot, g);
  if (e != cudaSuccess) throw std::runtime_error(std::string("kv append: launch failed: ") + cudaGetErrorString(e));
}

}  // namespace sfq
