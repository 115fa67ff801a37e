// New tokens' keys and values into the paged 8-bit cache, with head norm and rotation of q and k on the way.
//
// Bound by memory: q, k and v rows are read once, q is written as bf16, k and v as e4m3. A (page, head) has one scale, the smallest
// power of two s with |x| <= 448 s for all its tokens so far; a power of two, because a page that is filled token by token has its scale
// raised now and then, and the codes that are there then only move by whole exponents (rounded again where they become subnormal).
// Measured in a graph with 40 query heads: 1 token 3.1 us, 64 sequences of one token each 4.9 (a launch and four dependent loads), a prompt
// of 4747 tokens with norm and rotation 36.3 us (3.7 TB/s; norm, rotation and conversions take most of the issue slots).
#include <cuda_fp8.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "codec.cuh"
#include "kv_cache.cuh"
#include "ptx.cuh"
#include "runtime.h"

namespace sfq {
namespace {

using namespace ptx;

constexpr int kLanes = 16;                  // threads of one head's vector, 8 channels each
constexpr int kQueryHeads = 4;              // query heads a block of the page form rotates; 4747 tokens of 40 heads 36.3 us, 2 / 6 / 8: 40.8 / 36.9 / 37.9
// New tokens of a sequence up to which a warp takes a (page, head), and up to which a block of 128 threads does; for more, one of 512. 64
// sequences, 40 + 2 x 8 heads: 2 tokens 7.7 us by warps, 6.7 by small blocks; 5 tokens 15.1, 8.0 and 20.3 by large blocks; 16 tokens 43.7, 13.3
// and 26.5. More than 16 tokens a page would be computed twice in a small block.
constexpr int kFewTokens = 1, kSomeTokens = 16;
constexpr int kHeld = 2;                    // vectors a thread of the page form holds between its two passes

// A thread's eight channels of a head lie in two pieces of four: with rotation over 2 h channels, 4 l .. and h + 4 l .. for the first
// h / 4 threads, so that both halves of a pair are in one thread, and eight neighbours for the others.
struct Place {
  int a, b;    // first channels of the two pieces
  bool turns;
};
__device__ __forceinline__ Place place_of(const RotaryArgs& r, int l) {
  const int turning = r.cos != nullptr ? r.rotary_dim / 8 : 0;
  if (l < turning) return {4 * l, r.rotary_dim / 2 + 4 * l, true};
  return {8 * l, 8 * l + 4, false};
}

__device__ __forceinline__ void widen(uint2 w, float* v) {
  v[0] = __uint_as_float(w.x << 16), v[1] = __uint_as_float(w.x & 0xFFFF0000u);
  v[2] = __uint_as_float(w.y << 16), v[3] = __uint_as_float(w.y & 0xFFFF0000u);
}
__device__ __forceinline__ uint2 narrow(const float* v) {
  const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}
__device__ __forceinline__ uint2 load4(const __nv_bfloat16* p) { return *reinterpret_cast<const uint2*>(p); }

// The smallest power of two s, 2^-100 at least, with amax <= 448 s.
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = int(u >> 23) - 135 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);  // 448 = 1.75 x 2^8
  return __uint_as_float(uint32_t(max(e, -100) + 127) << 23);
}

__device__ __forceinline__ uint32_t encode2(float lo, float hi) { return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ uint32_t encode4(const float* v, float inv) {
  return encode2(v[0] * inv, v[1] * inv) | encode2(v[2] * inv, v[3] * inv) << 16;
}
// 1 / s: a power of two from 2^-126 up; s itself is 2^-100 .. 2^120 for what this kernel has scaled, and anything for what it has not.
__device__ __forceinline__ float inverse(float s) { return 1.0f / s; }

__device__ __forceinline__ float peak_of(const float (&v)[8], float peak) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(v[i]);
    if (a <= 3.402823466e38f) peak = fmaxf(peak, a);  // finite ones
  }
  return peak;
}

// Angles of a thread's four pairs; the row of the tables is checked.
struct Angles {
  float4 c, s;
};
__device__ __forceinline__ Angles angles_of(const KvCacheView& c, const RotaryArgs& r, const Place& at, int row, long long place) {
  Angles a = {make_float4(1, 1, 1, 1), make_float4(0, 0, 0, 0)};
  if (!at.turns) return a;
  long long position = r.position != nullptr ? r.position[row] : place;
  if (position < 0 || position >= r.table_rows) {
    atomicCAS(c.status, 0, kKvBadPosition);
    position = 0;
  }
  const size_t from = size_t(position) * (r.rotary_dim / 2) + at.a;
  a.c = *reinterpret_cast<const float4*>(r.cos + from), a.s = *reinterpret_cast<const float4*>(r.sin + from);
  return a;
}

// Norm (w: the weight's two pieces, or none) and rotation of one head vector spread over 16 lanes, in fp32, two channels an instruction.
// Whole warps.
__device__ __forceinline__ void norm_rope(float (&v)[8], bool norm, const float (&w)[8], float eps, bool turns, const Angles& t) {
  f32x2 x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = pack2(v[2 * i], v[2 * i + 1]);
  if (norm) {
    f32x2 sum2 = mul2(x[0], x[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) sum2 = fma2(x[i], x[i], sum2);
    float lo, hi;
    unpack2(sum2, lo, hi);
    float sum = lo + hi;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    const float inv = rsqrtf(fmaf(sum, 1.0f / kKvHeadDim, eps));
    const f32x2 inv2 = pack2(inv, inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = mul2(mul2(x[i], inv2), pack2(w[2 * i], w[2 * i + 1]));
  }
  if (turns) {
    const f32x2 c[2] = {pack2(t.c.x, t.c.y), pack2(t.c.z, t.c.w)}, s[2] = {pack2(t.s.x, t.s.y), pack2(t.s.z, t.s.w)};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x2 a = x[i], b = x[2 + i];
      x[i] = sub2(mul2(a, c[i]), mul2(b, s[i])), x[2 + i] = fma2(b, c[i], mul2(a, s[i]));
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2(x[i], v[2 * i], v[2 * i + 1]);
}

// Codes that are there, rounded again for a larger scale. V has `slots` of each channel's 2^page_shift.
__device__ __forceinline__ void scale_again(uint8_t* codes, int slots, int page_shift, bool v, float factor, int thread, int threads) {
  for (int i = thread; i < slots * kKvHeadDim; i += threads) {
    uint8_t* at = v ? codes + (size_t(i / slots) << page_shift) + i % slots : codes + i;
    *at = uint8_t(__nv_cvt_float_to_fp8(e4m3_decode(*at) * factor, __NV_SATFINITE, __NV_E4M3));
  }
}

struct Run {  // a sequence's new tokens in one page
  int row0, tokens, slot0;
  long long begin;  // place of the first in its sequence
};
__device__ __forceinline__ Run run_of(const KvCacheView& c, const KvSequence& s, long long page) {
  const long long past = s.length - s.rows, begin = max(page << c.page_shift, past), end = min((page + 1) << c.page_shift, s.length);
  return {s.row0 + int(begin - past), int(max(0ll, end - begin)), int(begin & ((1 << c.page_shift) - 1)), begin};
}

// One token a sequence: a warp for each (page of the new tokens, sequence, kv head), k in its lower half and v in its upper, and
// for each pair of query heads. What takes the time is the chain of dependent loads (sequence, page, scale), so nothing waits for
// anything else: no block-wide step, one piece of work a warp.
__global__ void __launch_bounds__(128) kv_append_few_kernel(KvCacheView c, RotaryArgs rot, AppendArgs g) {
  grid_dependency_release();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, half = lane >> 4, l = lane & 15;
  const int unit = blockIdx.x * 4 + int(threadIdx.x >> 5);
  if (unit >= c.kv_heads + (g.heads + 1) / 2) return;
  const Place at = place_of(rot, l);
  for (int b = blockIdx.z; b < c.batch; b += gridDim.z) {
    const KvSequence s = kv_sequence(c, b);
    if (s.rows <= 0) continue;
    const long long first_page = max(s.length - s.rows, 0ll) >> c.page_shift, last_page = (s.length - 1) >> c.page_shift;
    for (long long p = first_page + blockIdx.y; p <= last_page; p += gridDim.y) {
      const Run run = run_of(c, s, p);
      if (unit >= c.kv_heads) {
        const int head = (unit - c.kv_heads) * 2 + half;
        const bool live = head < g.heads, norm = rot.q_norm != nullptr;
        float w[8] = {1, 1, 1, 1, 1, 1, 1, 1};
        if (norm) widen(load4(rot.q_norm + at.a), w), widen(load4(rot.q_norm + at.b), w + 4);
        for (int i = 0; i < run.tokens; ++i) {
          const __nv_bfloat16* src = g.q + size_t(run.row0 + i) * g.ld_q + (live ? head : 0) * kKvHeadDim;
          const uint2 lo = load4(src + at.a), hi = load4(src + at.b);
          const Angles t = angles_of(c, rot, at, run.row0 + i, run.begin + i);
          float v[8];
          widen(lo, v), widen(hi, v + 4);
          norm_rope(v, norm, w, rot.eps, at.turns, t);
          if (live) {
            __nv_bfloat16* dst = g.q_out + size_t(run.row0 + i) * g.ld_q_out + head * kKvHeadDim;
            *reinterpret_cast<uint2*>(dst + at.a) = narrow(v), *reinterpret_cast<uint2*>(dst + at.b) = narrow(v + 4);
          }
        }
        continue;
      }
      if (run.tokens <= 0) continue;
      const int page = kv_page(c, b, p);
      const size_t block = size_t(max(page, 0)) * c.kv_heads + unit;
      const bool norm = rot.k_norm != nullptr;
      float w[8] = {1, 1, 1, 1, 1, 1, 1, 1};
      if (norm) widen(load4(rot.k_norm + at.a), w), widen(load4(rot.k_norm + at.b), w + 4);
      auto load = [&](int i, float (&x)[8]) {  // k in the lower half of the warp, v in the upper, whose pieces lie side by side
        const __nv_bfloat16* src = (half ? g.v : g.k) + size_t(run.row0 + i) * g.ld_kv + unit * kKvHeadDim;
        const uint2 lo = load4(src + (half ? l * 8 : at.a)), hi = load4(src + (half ? l * 8 + 4 : at.b));
        const Angles t = angles_of(c, rot, at, run.row0 + i, run.begin + i);
        widen(lo, x), widen(hi, x + 4);
        float k[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] = x[e];
        norm_rope(k, norm, w, rot.eps, at.turns, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = half ? x[e] : k[e];
      };
      float* const scales = half ? c.v_scale : c.k_scale;
      const float old = run.slot0 > 0 && page >= 0 ? scales[block] : 0.0f;
      float peak = 0.0f, x[8];
      for (int i = run.tokens - 1; i >= 0; --i) load(i, x), peak = peak_of(x, peak);  // ends with the first token's values in x
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, off));
      const float now = fmaxf(old, scale_for(peak)), inv = inverse(now);
      if (page < 0) continue;
      uint8_t* const codes = (half ? c.v : c.k) + ((block * kKvHeadDim) << c.page_shift);
      if (l == 0) scales[block] = now;
      if (now != old && run.slot0 > 0) scale_again(codes, run.slot0, c.page_shift, half != 0, old / now, l, kLanes);
      for (int i = 0; i < run.tokens; ++i) {
        if (i > 0) load(i, x);
        const uint32_t lo = encode4(x, inv), hi = encode4(x + 4, inv);
        const int slot = run.slot0 + i;
        if (half == 0) {
          *reinterpret_cast<uint32_t*>(codes + size_t(slot) * kKvHeadDim + at.a) = lo;
          *reinterpret_cast<uint32_t*>(codes + size_t(slot) * kKvHeadDim + at.b) = hi;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) codes[(size_t(l * 8 + e) << c.page_shift) + slot] = uint8_t((e < 4 ? lo : hi) >> (8 * (e & 3)));
        }
      }
    }
  }
}

// Several tokens, prompts. blockIdx.x: a kv head, behind them groups of query heads; y: sequence; z: page of the sequence's new tokens, so that what runs at
// a time reads rows of a fused projection whole (with the pages first 38.6 us in place of 36.3). A thread takes the
// same piece of up to kHeld tokens' vectors, which stay in registers while the block finds the page's scale (more than 64 tokens of a
// page, 16 with 128 threads, are computed twice); V goes through shared memory, so that a channel's tokens are stored side by side.
template <int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) kv_append_page_kernel(KvCacheView c, RotaryArgs rot, AppendArgs g) {
  constexpr int kAtOnce = kThreads / kLanes;  // vectors a block works on at once
  grid_dependency_release();
  grid_dependency_wait();
  __shared__ float peaks[2][kThreads / 32];
  // V's codes, a channel's tokens side by side. A word more than they take, and two more every 32 channels, puts the words that the
  // sixteen threads of a vector write to into different banks.
  extern __shared__ __align__(16) uint8_t sh_v[];
  const int page_size = 1 << c.page_shift;
  auto staged = [&](int channel) { return sh_v + channel * (page_size + 4) + (channel >> 5) * 8; };
  const int vector = threadIdx.x / kLanes, l = threadIdx.x & 15;
  const Place at = place_of(rot, l);
  const bool queries = int(blockIdx.x) >= c.kv_heads;
  const __nv_bfloat16* weight = queries ? rot.q_norm : rot.k_norm;
  const bool norm = weight != nullptr;
  float w[8] = {1, 1, 1, 1, 1, 1, 1, 1};
  if (norm) widen(load4(weight + at.a), w), widen(load4(weight + at.b), w + 4);
  for (int b = blockIdx.y; b < c.batch; b += gridDim.y) {
    const KvSequence s = kv_sequence(c, b);
    if (s.rows <= 0) continue;
    const long long first_page = max(s.length - s.rows, 0ll) >> c.page_shift, last_page = (s.length - 1) >> c.page_shift;
    for (long long p = first_page + blockIdx.z; p <= last_page; p += gridDim.z) {
      const Run run = run_of(c, s, p);
      if (queries) {
        const int head0 = (blockIdx.x - c.kv_heads) * kQueryHeads, heads = min(kQueryHeads, g.heads - head0);
        for (int j = vector; j - vector < run.tokens; j += kAtOnce) {  // whole warps
          const bool live = j < run.tokens;
          const int i = min(j, run.tokens - 1);
          const Angles t = angles_of(c, rot, at, run.row0 + i, run.begin + i);
          const __nv_bfloat16* src = g.q + size_t(run.row0 + i) * g.ld_q + head0 * kKvHeadDim;
          __nv_bfloat16* dst = g.q_out + size_t(run.row0 + i) * g.ld_q_out + head0 * kKvHeadDim;
          // two heads at a time, the next two on their way
          uint2 raw[2][2][2];
          auto fetch = [&](int h, uint2 (&to)[2][2]) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const __nv_bfloat16* from = src + min(h + k, heads - 1) * kKvHeadDim;
              to[k][0] = load4(from + at.a), to[k][1] = load4(from + at.b);
            }
          };
          fetch(0, raw[0]);
#pragma unroll
          for (int h = 0; h < kQueryHeads; h += 2) {
            if (h >= heads) break;
            if (h + 2 < kQueryHeads) fetch(h + 2, raw[(h / 2 + 1) & 1]);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float v[8];
              widen(raw[(h / 2) & 1][k][0], v), widen(raw[(h / 2) & 1][k][1], v + 4);
              norm_rope(v, norm, w, rot.eps, at.turns, t);
              if (live && h + k < heads) {
                *reinterpret_cast<uint2*>(dst + (h + k) * kKvHeadDim + at.a) = narrow(v);
                *reinterpret_cast<uint2*>(dst + (h + k) * kKvHeadDim + at.b) = narrow(v + 4);
              }
            }
          }
        }
        continue;
      }
      if (run.tokens <= 0) continue;
      const int head = blockIdx.x, page = kv_page(c, b, p);
      if (page < 0) continue;
      const size_t block = size_t(page) * c.kv_heads + head;
      uint8_t* const kc = c.k + ((block * kKvHeadDim) << c.page_shift);
      uint8_t* const vc = c.v + ((block * kKvHeadDim) << c.page_shift);
      float k_peak = 0.0f, v_peak = 0.0f;
      auto load = [&](int j, float (&k)[8], uint4& v) {
        const int i = min(j, run.tokens - 1);
        const size_t row = size_t(run.row0 + i) * g.ld_kv + head * kKvHeadDim;
        const uint2 lo = load4(g.k + row + at.a), hi = load4(g.k + row + at.b);
        v = *reinterpret_cast<const uint4*>(g.v + row + l * 8);
        const Angles t = angles_of(c, rot, at, run.row0 + i, run.begin + i);
        widen(lo, k), widen(hi, k + 4);
        norm_rope(k, norm, w, rot.eps, at.turns, t);
      };
      auto widen8 = [](const uint4& v, float (&x)[8]) { widen(make_uint2(v.x, v.y), x), widen(make_uint2(v.z, v.w), x + 4); };
      float k[kHeld][8];
      uint4 v[kHeld];
      const bool held = run.tokens <= kHeld * kAtOnce;
      for (int j0 = 0; j0 < run.tokens; j0 += kHeld * kAtOnce)
#pragma unroll
        for (int h = 0; h < kHeld; ++h) {
          const int j = j0 + h * kAtOnce + vector;
          if (j - vector >= run.tokens) break;
          load(j, k[h], v[h]);
          float x[8];
          widen8(v[h], x);
          k_peak = peak_of(k[h], k_peak), v_peak = peak_of(x, v_peak);
        }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) {
        k_peak = fmaxf(k_peak, __shfl_xor_sync(0xffffffffu, k_peak, off));
        v_peak = fmaxf(v_peak, __shfl_xor_sync(0xffffffffu, v_peak, off));
      }
      if ((threadIdx.x & 31) == 0) peaks[0][threadIdx.x / 32] = k_peak, peaks[1][threadIdx.x / 32] = v_peak;
      const float old_k = run.slot0 > 0 ? c.k_scale[block] : 0.0f, old_v = run.slot0 > 0 ? c.v_scale[block] : 0.0f;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) k_peak = fmaxf(k_peak, peaks[0][i]), v_peak = fmaxf(v_peak, peaks[1][i]);
      const float new_k = fmaxf(old_k, scale_for(k_peak)), new_v = fmaxf(old_v, scale_for(v_peak));
      const float inv_k = inverse(new_k), inv_v = inverse(new_v);
      if (run.slot0 > 0) {
        if (new_k != old_k) scale_again(kc, run.slot0, c.page_shift, false, old_k / new_k, threadIdx.x, kThreads);
        if (new_v != old_v) scale_again(vc, run.slot0, c.page_shift, true, old_v / new_v, threadIdx.x, kThreads);
      }
      for (int j0 = 0; j0 < run.tokens; j0 += kHeld * kAtOnce)
#pragma unroll
        for (int h = 0; h < kHeld; ++h) {
          const int j = j0 + h * kAtOnce + vector;
          if (j - vector >= run.tokens) break;
          if (!held) load(j, k[h], v[h]);
          float x[8];
          widen8(v[h], x);
          if (j < run.tokens) {
            *reinterpret_cast<uint32_t*>(kc + size_t(run.slot0 + j) * kKvHeadDim + at.a) = encode4(k[h], inv_k);
            *reinterpret_cast<uint32_t*>(kc + size_t(run.slot0 + j) * kKvHeadDim + at.b) = encode4(k[h] + 4, inv_k);
            const uint32_t lo = encode4(x, inv_v), hi = encode4(x + 4, inv_v);
#pragma unroll
            for (int e = 0; e < 8; ++e) staged(l * 8 + e)[run.slot0 + j] = uint8_t((e < 4 ? lo : hi) >> (8 * (e & 3)));
          }
        }
      __syncthreads();  // every thread has read the old scales, too
      if (threadIdx.x == 0) c.k_scale[block] = new_k, c.v_scale[block] = new_v;
      // whole groups of 16 tokens of a channel as one store, the ragged ends byte by byte
      const int first = run.slot0, end = run.slot0 + run.tokens, groups = page_size / 16;
      for (int i = threadIdx.x; i < kKvHeadDim * groups; i += kThreads) {
        const int channel = i / groups, t = i % groups * 16;
        const uint8_t* from = staged(channel) + t;
        uint8_t* to = vc + (size_t(channel) << c.page_shift) + t;
        if (t >= first && t + 16 <= end) {
          const uint32_t* f = reinterpret_cast<const uint32_t*>(from);
          *reinterpret_cast<uint4*>(to) = make_uint4(f[0], f[1], f[2], f[3]);
        } else {
          for (int k2 = max(first - t, 0); k2 < min(end - t, 16); ++k2) to[k2] = from[k2];
        }
      }
      __syncthreads();  // the next page's work may overwrite peaks and V
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
  for (const void* p : {static_cast<const void*>(c.k_scale), static_cast<const void*>(c.v_scale), static_cast<const void*>(c.table), static_cast<const void*>(c.seq_len),
                        static_cast<const void*>(c.row_start)})
    if (reinterpret_cast<uintptr_t>(p) % 4 != 0) throw std::invalid_argument("kv cache: scales, page table, lengths and row starts must be 4-byte aligned");
}

void kv_append(KvCacheView c, int head_dim, const RotaryArgs& rot, const AppendArgs& g, cudaStream_t stream) {
  kv_check(c, head_dim);
  if (c.rows <= 0) return;
  if (!g.k || !g.v || (g.heads > 0 && (!g.q || !g.q_out))) throw std::invalid_argument("kv append: null operand");
  if (g.heads < 0 || g.heads > 32768) throw std::invalid_argument("kv append: bad number of query heads");
  if (g.ld_kv < c.kv_heads * kKvHeadDim || g.ld_kv % 8 != 0 || !aligned16(g.k) || !aligned16(g.v) ||
      (g.heads > 0 && (g.ld_q < g.heads * kKvHeadDim || g.ld_q_out < g.heads * kKvHeadDim || g.ld_q % 8 != 0 || g.ld_q_out % 8 != 0 || !aligned16(g.q) || !aligned16(g.q_out))))
    throw std::invalid_argument("kv append: row pitches must cover heads * 128 columns and keep 16-byte alignment");
  const int q_cols = g.heads * kKvHeadDim, kv_cols = c.kv_heads * kKvHeadDim;
  if (g.heads > 0 && ((!(g.q == g.q_out && (g.ld_q == g.ld_q_out || c.rows == 1)) && rows_overlap(g.q, g.ld_q, q_cols, g.q_out, g.ld_q_out, q_cols, c.rows)) ||
                      rows_overlap(g.k, g.ld_kv, kv_cols, g.q_out, g.ld_q_out, q_cols, c.rows) || rows_overlap(g.v, g.ld_kv, kv_cols, g.q_out, g.ld_q_out, q_cols, c.rows)))
    throw std::invalid_argument("kv append: q_out is q itself, with its pitch, or lies apart from q, k and v");
  if ((rot.cos == nullptr) != (rot.sin == nullptr)) throw std::invalid_argument("kv append: cos and sin come together");
  if (rot.cos != nullptr && (rot.rotary_dim <= 0 || rot.rotary_dim > kKvHeadDim || rot.rotary_dim % 16 != 0 || rot.table_rows <= 0))
    throw std::invalid_argument("kv append: rotary_dim must be a multiple of 16 up to 128, with at least one table row");
  if (!aligned16(rot.cos) || !aligned16(rot.sin) || !aligned16(rot.q_norm) || !aligned16(rot.k_norm)) throw std::invalid_argument("kv append: tables and norm weights must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(rot.position) % 4 != 0) throw std::invalid_argument("kv append: positions must be 4-byte aligned");
  c.status = device_status_word();
  const int page_size = 1 << c.page_shift, pages = (std::min(c.max_new, c.rows) + page_size - 2) / page_size + 1;
  const size_t bytes = size_t(c.rows) * (g.heads * 4 + c.kv_heads * 6) * kKvHeadDim;
  cudaError_t e;
  if (c.max_new <= kFewTokens) {
    const int units = c.kv_heads + (g.heads + 1) / 2;
    e = launch_overlapped(bytes, kv_append_few_kernel, dim3((units + 3) / 4, pages, std::min(c.batch, 65535)), dim3(128), 0, stream, c, rot, g);
  } else {
    const size_t smem = size_t(kKvHeadDim) * (page_size + 4) + 32;
    const int groups = (g.heads + kQueryHeads - 1) / kQueryHeads;
    const int threads = c.max_new <= kSomeTokens ? 128 : 512;
    e = launch_overlapped(bytes, threads == 128 ? kv_append_page_kernel<128> : kv_append_page_kernel<512>,
                          dim3(c.kv_heads + groups, std::min(c.batch, 65535), std::min(pages, 65535)), dim3(threads), smem, stream, c, rot, g);
  }
  if (e != cudaSuccess) throw std::runtime_error(std::string("kv append: launch failed: ") + cudaGetErrorString(e));
}

}  // namespace sfq
