// Attention of a few new tokens per sequence over the paged 8-bit cache, grouped heads, causal among the new tokens.
//
// Bound by memory: every sequence's e4m3 codes of K and V are read once, 256 bytes for a token and kv head, and each is one conversion of
// half an instruction away from fp16. The products run on mma.sync m16n8k16, transposed, so that the query heads of a group (and the new
// tokens of a sequence), of which there are few, are its N of 8 and the cache its M of 16:
//   S^T [tokens, queries] = K Q^T    O^T [channels, queries] += V^T P^T
// A warp takes 64 tokens at a time, which asynchronous copies put into its own 16 KB of shared memory: the next K while this one's softmax
// and second product run, the next V under the scores. V lies with a channel's tokens side by side, so both operands are 16-byte reads, and
// the weights P go from the first product's result to the second one's operand by 8 x 8 transposes between lanes. Which
// token is which row of the first product is free: the order is chosen so that the transposed weights of four MMAs meet the 16
// neighbouring tokens of a lane's V. Softmax with running maximum and sum in fp32; the page's scale of K goes into the score, that of V into
// the weight.
// Long sequences are divided over CTAs (flash decoding); a second launch joins their parts in order.
// Measured in a graph, 40 query heads on 8 kv heads: one sequence of 333 tokens 8.7 us, of 131072 51.0 (5.3 TB/s), 32 of up to 4096
// 42.2 (4.1 TB/s). 16 of up to 3001 with five new tokens, 40 heads on 10, 52.0 us: three query tiles of
// eight, where scores, exponentials and products, not memory, take the time. Prompts go through 24 query columns at a time, which is right
// but not fast: 4747 new tokens, 40 heads on 10, 1.5 ms, behind as many cached ones 3.8.
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <stdexcept>
#include <string>

#include "kv_cache.cuh"
#include "ptx.cuh"
#include "runtime.h"

namespace sfq {
namespace {

using namespace ptx;

constexpr int kTile = 64;        // tokens a warp takes at a time
constexpr int kTileBytes = kTile * kKvHeadDim;  // of K, and of V
constexpr float kLift = 15.0f, kLower = 0x1p-15f;  // the largest weight of the second product is below 2^kLift, see there
constexpr int kPartFloats = 132; // of a divided row and head: O [128], maximum, sum, whether any key was seen, how many parts there are
constexpr int kMostSplits = 64;
constexpr int kNarrowSplits = 16;  // parts up to which a warp joins them
constexpr int kSms = 148;        // the launch is planned for; the workspace can be asked for without a device
constexpr int kResident[4] = {0, 3, 2, 2};  // CTAs of an SM, by the query tiles of eight

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// Four e4m3 of a word as two pairs of fp16.
__device__ __forceinline__ void e4m3_pairs(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {  // 16 bytes, or zeros for bytes == 0
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// 2^x to two units in the last place of fp32; results below 2^-126 are zero.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 0xFF in the bytes of w that are NaN (0x7F or 0xFF).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu); }

// Notes for one channel that the columns which see a token with a NaN value there are NaN: `bad` has the bytes of tokens at ..
// at + 3, column i sees the first `first + (col0 + i) / group` tokens.
__device__ __noinline__ void note_nan(uint32_t* columns, uint32_t bad, int at, int first, int col0, int cols, int group) {
  for (int i = 0; i < cols; ++i) {
    const int sees = first + (col0 + i) / group;
    for (int k = 0; k < 4; ++k)
      if ((bad >> (8 * k) & 1) != 0 && at + k < sees) atomicOr(columns, 1u << i);
  }
}

// Into how many parts of a sequence's tiles a launch goes. All parts have as many tiles, those of the longest sequence over `even` where the
// sequences are nearly as long as each other, else over `ragged`; short ones have fewer parts. So all CTAs take about as long, and their
// number suits the SMs whichever the lengths are.
struct Splits {
  int grid, even, ragged;  // grid: the larger one
};
__device__ __forceinline__ int length_of(const KvCacheView& c, long long length) {
  // lengths are 32-bit; the last few thousand of their range are not used, so that sums of places stay in it
  return int(max(0ll, min(min(length, (long long)c.max_pages << c.page_shift), 0x7FFF0000ll)));
}
__device__ __forceinline__ int tiles_of(int length) { return (length + kTile - 1) / kTile; }
// Tiles of a part. Whole warps.
__device__ __forceinline__ int tiles_of_part(const KvCacheView& c, const Splits& splits) {
  int longest = 0;
  float sum = 0.0f;
  for (int b = threadIdx.x & 31; b < c.batch; b += 32) {
    const int tiles = tiles_of(length_of(c, c.seq_len[b]));
    longest = max(longest, tiles), sum += float(tiles);
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  const int over = sum * 8.0f >= float(longest) * float(c.batch) * 7.0f ? splits.even : splits.ragged;
  return max(1, (longest + over - 1) / over);
}

template <int NT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kWarps == 4 ? kResident[NT] : 1) kv_attention_kernel(KvCacheView c, KvAttentionArgs g, float* parts, Splits splits) {
  constexpr int kCols = NT * 8, kThreads = kWarps * 32;
  // a tile of K [64 tokens][128] and of V [128][64 tokens] for each warp; when they are done, [kWarps][128][kCols + 1] sums
  extern __shared__ __align__(128) uint8_t smem[];
  float* const sh_o = reinterpret_cast<float*>(smem);
  static_assert(kWarps * kKvHeadDim * (kCols + 1) * 4 <= kWarps * 2 * kTileBytes, "the sums fit");
  __shared__ float sh_m[kWarps][kCols], sh_mv[kWarps][kCols], sh_l[kWarps][kCols];
  __shared__ int sh_seen[kWarps][kCols];
  __shared__ uint2 sh_q[8][NT][32];
  __shared__ uint32_t sh_nan[kKvHeadDim];  // columns that are NaN in a channel
  __shared__ float sh_qscale[kCols];
  grid_dependency_release();
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, q = lane & 3;
  // parts are the slowest of the grid's dimensions, so that those that short sequences lack do not stand in front of any other
  const int head = int(blockIdx.x) % c.kv_heads, split = blockIdx.z;
  const int page_mask = (1 << c.page_shift) - 1;

  const int each = splits.grid > 1 ? tiles_of_part(c, splits) : INT_MAX;
  for (int b = int(blockIdx.x) / c.kv_heads; b < c.batch; b += int(gridDim.x) / c.kv_heads) {
    const KvSequence s = kv_sequence(c, b);
    const int length = length_of(c, s.length), all_tiles = tiles_of(length);
    const int used = splits.grid > 1 ? max(1, (all_tiles + each - 1) / each) : 1;  // parts of this sequence
    if (split >= used) continue;
    const int past = int(max(-0x7FFF0000ll, min(s.length, 0x7FFF0000ll) - s.rows));  // tokens in front of the new ones
    const int all_cols = s.rows * g.group;
    for (int col0 = int(blockIdx.y) * kCols; col0 < all_cols; col0 += int(gridDim.y) * kCols) {
      __syncthreads();  // what the tile in front left in shared memory has been read
      if (threadIdx.x < kKvHeadDim) sh_nan[threadIdx.x] = 0;
      // ---- this warp's tiles, the first on its way under the queries
      const int last = min(length, past + min(col0 + kCols - 1, all_cols - 1) / g.group + 1);  // keys that any column sees
      const int first_hidden = past + col0 / g.group + 1;  // ... that one of them does not
      const int tiles = (max(last, 0) + kTile - 1) / kTile;
      const int tile_end = int(min((long long)tiles, (split + 1ll) * each));
      // A tile's pages: lane c holds that of chunk c % 4 of its four chunks of 16 tokens, -1 where there is none.
      auto page_of = [&](int tile) -> int {
        const int t = tile * kTile + q * 16;
        return tile < tile_end && t < last ? kv_page(c, b, t >> c.page_shift) : -1;
      };
      const uint32_t k_sh = smem_u32(smem) + warp * 2 * kTileBytes, v_sh = k_sh + kTileBytes;
      // K: 16 bytes of four tokens at a time, the unit exclusive-or'ed with four times the token's last bit, so that the two rows that eight
      // lanes read together lie in different banks. V: 16 tokens of eight channels at a time. Chunks without a page are zeros.
      auto fetch_k = [&](int tile, int pages) {
        if (tile < tile_end) {
          const int unit = lane & 7, token0 = lane >> 3;
          const uint32_t to = k_sh + token0 * 128 + ((unit ^ ((token0 & 1) << 2)) << 4);
#pragma unroll
          for (int chunk = 0; chunk < 4; ++chunk) {
            const int page = __shfl_sync(0xffffffffu, pages, chunk);
            const int slot = (tile * kTile + chunk * 16) & page_mask;
            const uint8_t* from = page < 0 ? c.k : c.k + (((size_t(page) * c.kv_heads + head) << c.page_shift) + slot + token0) * kKvHeadDim + unit * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i) cp_async16(to + (chunk * 16 + i * 4) * 128, from + (page < 0 ? 0 : i * 4 * kKvHeadDim), page < 0 ? 0 : 16);
          }
        }
        cp_commit();
      };
      auto fetch_v = [&](int tile, int pages) {
        if (tile < tile_end) {
          const int slot = (tile * kTile + q * 16) & page_mask;
          const uint8_t* from = pages < 0 ? c.v : c.v + (((size_t(pages) * c.kv_heads + head) * kKvHeadDim + gq) << c.page_shift) + slot;
          const int step = pages < 0 ? 0 : 8 << c.page_shift;
          const uint32_t to = v_sh + gq * 64 + q * 16;
#pragma unroll
          for (int i = 0; i < 16; ++i) cp_async16(to + i * 8 * 64, from + i * step, pages < 0 ? 0 : 16);
        }
        cp_commit();
      };
      int tile = split * each + warp;
      int pages = page_of(tile), next_pages = page_of(tile + kWarps);
      fetch_k(tile, pages);
      fetch_v(tile, pages);
      // ---- the queries as fp16, each times a power of two that takes its largest element just below 2^15. Its eight significant bits are
      // exact down to 2^-31 of that; what is smaller is off by 2^-39 of it at most.
      for (int i = threadIdx.x; i < kCols * 4; i += kThreads) {
        const int col = i >> 2, quarter = i & 3;
        const int at = min(col0 + col, all_cols - 1), token = at / g.group, qh = head * g.group + at % g.group;
        const __nv_bfloat16* src = g.q + size_t(s.row0 + token) * g.ld_q + qh * kKvHeadDim + quarter * 16;
        uint32_t raw[16];
        uint32_t top = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint4 v = *reinterpret_cast<const uint4*>(src + (u >> 1) * 64 + (u & 1) * 8);
          raw[4 * u] = v.x, raw[4 * u + 1] = v.y, raw[4 * u + 2] = v.z, raw[4 * u + 3] = v.w;
        }
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          const uint32_t lo = raw[u] & 0x7FFFu, hi = (raw[u] >> 16) & 0x7FFFu;
          if (lo < 0x7F80u) top = max(top, lo);
          if (hi < 0x7F80u) top = max(top, hi);
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // Exponent of the largest element, -108 at least: bf16's smallest number is then still a normal fp16, and so is the factor of the scores.
        const int e = max(int(top >> 7) - 127, -108);
        const float up = ldexpf(1.0f, 14 - e);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t w[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t r = raw[2 * j + h];
            w[h] = half_pair(__uint_as_float(r << 16) * up, __uint_as_float(r & 0xFFFF0000u) * up);
          }
          sh_q[j][col >> 3][(col & 7) * 4 + quarter] = make_uint2(w[0], w[1]);
        }
        if (quarter == 0) sh_qscale[col] = ldexpf(g.scale_log2, e - 14);
      }
      __syncthreads();

      // ---- this warp's columns, state and tokens
      int sees[NT][2];
      float qscale[NT][2], m[NT][2], mv[NT][2], l[NT][2];
      bool seen[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int col = n * 8 + q * 2 + e;
          sees[n][e] = min(length, past + min(col0 + col, all_cols - 1) / g.group + 1);
          qscale[n][e] = sh_qscale[col];
          m[n][e] = mv[n][e] = -INFINITY, l[n][e] = 0.0f, seen[n][e] = false;
        }
      float o[8][NT][4];
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int n = 0; n < NT; ++n) o[d][n][0] = o[d][n][1] = o[d][n][2] = o[d][n][3] = 0.0f;

      for (; tile < tile_end; tile += kWarps) {
        const int t0 = tile * kTile;
        const size_t block = size_t(max(pages, 0)) * c.kv_heads + head;
        const float ks_mine = pages < 0 ? 0.0f : c.k_scale[block], vs_mine = pages < 0 ? 0.0f : c.v_scale[block];
        // ---- scores
        cp_wait<1>();
        __syncwarp();
        float sc[4][NT][4];
#pragma unroll
        for (int t = 0; t < 4; t += 2) {  // two MMAs of 16 tokens share the reads of q
          uint4 k[2][2][2];  // [MMA][row gq or gq + 8][half of the channels]
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int u = 0; u < 2; ++u)
                k[i][r][u] = lds128(k_sh + ((gq >> 1) * 16 + (t + i) * 4 + (gq & 1) + 2 * r) * 128 + (((u * 4 + q) ^ ((gq & 1) << 2)) << 4));
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint2 bq[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) bq[n] = sh_q[j][n][lane];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t a0, a1, a2, a3;
              e4m3_pairs(word_of(k[i][0][j >> 2], j & 3), a0, a2);
              e4m3_pairs(word_of(k[i][1][j >> 2], j & 3), a1, a3);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                if (j == 0)
                  mma_f16_zero(sc[t + i][n], a0, a1, a2, a3, bq[n].x, bq[n].y);
                else
                  mma_f16(sc[t + i][n], a0, a1, a2, a3, bq[n].x, bq[n].y);
              }
            }
          }
        }
        __syncwarp();
        fetch_k(tile + kWarps, next_pages);
        // this lane's rows lie in chunk gq / 2
        const int page_k = __shfl_sync(0xffffffffu, pages, gq >> 1), page_v = pages;
        const float ks = __shfl_sync(0xffffffffu, ks_mine, gq >> 1), vs = __shfl_sync(0xffffffffu, vs_mine, gq >> 1);
        const int page = page_k;
        // ---- weights
        const bool whole = __all_sync(0xffffffffu, page >= 0) && t0 + kTile <= min(first_hidden, length);
        const int mine = t0 + (gq >> 1) * 16 + (gq & 1);  // token of row gq of MMA 0; row gq + 8 is two behind, MMA t four t
        // The weights of the second product are p vs = exp2(score + e) (vs / 2^e) with |vs| / 2^e in [0.5, 1), over their own running
        // reference mv, the largest score + e less kLift: a page of small values that has all the weight keeps its bits beside one of
        // large values that has none. They go to fp16, whose eleven bits are more than those of q, the codes and the result. Weights of
        // more bits would need a second product: with two fp16 terms 32 x 4096 takes 46.9 us in place of 42.8, 1 x 131072 55.0 and not
        // 53.4, 16 x 5 new tokens 59.3 and not 52.8 (called), and the results stay 1.67e-3 of their norm from 64 bits, the rounding to
        // bf16. kLift puts the largest just below 2^15, so that all eleven bits are there down to 2^-29 of it and what is dropped is below
        // 2^-40: where a key that has no value takes nearly all the weight, the others are the result.
        const float e_mine = fabsf(vs) > 0.0f ? float(min(ilogbf(vs), 127) + 1) : 0.0f;
        const float frac = fabsf(vs) > 0.0f ? ldexpf(vs, -int(e_mine)) : vs;
        float top[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          top[n][0] = top[n][1] = -INFINITY;
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float v = sc[t][n][e] * (ks * qscale[n][e & 1]);
              if (!whole) {
                const bool there = page >= 0 && mine + t * 4 + (e >> 1) * 2 < sees[n][e & 1];
                seen[n][e & 1] |= there;
                v = there ? v : -INFINITY;
              }
              sc[t][n][e] = v;
              top[n][e & 1] = fmaxf(top[n][e & 1], v);
            }
          if (whole) seen[n][0] = seen[n][1] = true;
        }
        float top_v[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) top_v[n][0] = __fadd_ru(top[n][0], e_mine - kLift), top_v[n][1] = __fadd_ru(top[n][1], e_mine - kLift);  // no weight above 2^15
#pragma unroll
        for (int off = 4; off < 32; off <<= 1)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              top[n][e] = fmaxf(top[n][e], __shfl_xor_sync(0xffffffffu, top[n][e], off));
              top_v[n][e] = fmaxf(top_v[n][e], __shfl_xor_sync(0xffffffffu, top_v[n][e], off));
            }
        float keep[NT][2];
        bool moved = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float m_new = fmaxf(m[n][e], top[n][e]), mv_new = fmaxf(mv[n][e], top_v[n][e]);
            l[n][e] *= m_new == -INFINITY ? 1.0f : exp2_fast(m[n][e] - m_new);  // exp2(-inf - x) = 0 on the first tile
            keep[n][e] = mv_new == -INFINITY ? 1.0f : exp2_fast(mv[n][e] - mv_new);
            moved |= mv_new != mv[n][e];
            m[n][e] = m_new, mv[n][e] = mv_new;
          }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int d = 0; d < 8; ++d)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[d][n][e] *= keep[n][e & 1];
        }
        // Where the references lie near each other, as they do unless pages' scales differ by a great deal, the second weight is the first
        // times a factor. Differences of scores come before e: they are exact where they count, while a large score and e is not.
        // Which way a weight is made depends on nothing but its own query and page, so that no query changes another's bits.
        float factor[NT][2];
        uint32_t far = 0;  // bit 2 n + e
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float between = m[n][e] == -INFINITY ? 0.0f : m[n][e] - mv[n][e] + e_mine;
            if (!(fabsf(between) < 60.0f)) far |= 1u << (2 * n + e);  // NaN, too
            factor[n][e] = exp2_fast(between) * frac;
          }
        const bool near = __all_sync(0xffffffffu, far == 0);
        uint32_t p[4][NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float ref[2], ref_v[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            ref[e] = m[n][e] == -INFINITY ? 0.0f : m[n][e];
            ref_v[e] = mv[n][e] == -INFINITY ? 0.0f : mv[n][e];
          }
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              w[e] = exp2_fast(sc[t][n][e] - ref[e & 1]);
              l[n][e & 1] += w[e];
              w[e] = near || (far >> (2 * n + (e & 1)) & 1) == 0 ? w[e] * factor[n][e & 1] : exp2_fast(sc[t][n][e] - ref_v[e & 1] + e_mine) * frac;
            }
            p[t][n][0] = transpose8x8(half_pair(w[0], w[1]));
            p[t][n][1] = transpose8x8(half_pair(w[2], w[3]));
          }
        }
        const int v0 = t0 + q * 16;
        const bool ragged = t0 + kTile > length || !__all_sync(0xffffffffu, page_v >= 0);
        const bool hidden = t0 + kTile > first_hidden;
        cp_wait<1>();
        __syncwarp();
        const int live = page_v < 0 ? 0 : max(0, min(16, length - v0));  // bytes of a channel that are tokens of this sequence
#pragma unroll
        for (int part = 0; part < 4; ++part) {
          uint4 v[2][2];
#pragma unroll
          for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int h = 0; h < 2; ++h) v[d][h] = lds128(v_sh + (part * 32 + d * 16 + h * 8 + gq) * 64 + q * 16);
          if (ragged || hidden) {
            // V behind the sequence's end, or of no page, is zeros: a weight of zero does not undo NaN bytes. Of tokens that some of the
            // columns do not see, NaN bytes are taken out and noted for the columns that do.
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const int bytes = min(max(live - 4 * w, 0), 4);
              const uint32_t mask = bytes == 4 ? 0xFFFFFFFFu : (1u << (8 * bytes)) - 1u;
#pragma unroll
              for (int d = 0; d < 2; ++d)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  uint32_t& word = w == 0 ? v[d][h].x : w == 1 ? v[d][h].y : w == 2 ? v[d][h].z : v[d][h].w;
                  word &= mask;
                  const uint32_t bad = hidden ? nan_bytes(word) : 0;
                  if (bad != 0) {
                    note_nan(&sh_nan[part * 32 + d * 16 + h * 8 + gq], bad, v0 + w * 4, past + 1, col0, min(kCols, all_cols - col0), g.group);
                    word &= ~bad;
                  }
                }
            }
          }
#pragma unroll
          for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              uint32_t a0, a1, a2, a3;
              e4m3_pairs(word_of(v[d][0], t), a0, a2);
              e4m3_pairs(word_of(v[d][1], t), a1, a3);
#pragma unroll
              for (int n = 0; n < NT; ++n) mma_f16(o[part * 2 + d][n], a0, a1, a2, a3, p[t][n][0], p[t][n][1]);
            }
        }
        __syncwarp();
        fetch_v(tile + kWarps, next_pages);
        pages = next_pages;
        next_pages = page_of(tile + 2 * kWarps);
      }
      cp_wait<0>();
      __syncthreads();  // every warp's tiles have been read

      // ---- the warps joined
#pragma unroll
      for (int off = 4; off < 32; off <<= 1)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], off);
            seen[n][e] |= __shfl_xor_sync(0xffffffffu, int(seen[n][e]), off) != 0;
          }
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sh_o[(warp * kKvHeadDim + d * 16 + gq + (e >> 1) * 8) * (kCols + 1) + n * 8 + q * 2 + (e & 1)] = o[d][n][e] * kLower;
      if (gq == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int col = n * 8 + q * 2 + e;
            sh_m[warp][col] = m[n][e], sh_mv[warp][col] = mv[n][e], sh_l[warp][col] = l[n][e], sh_seen[warp][col] = seen[n][e];
          }
      }
      __syncthreads();
      const int cols = min(kCols, all_cols - col0);
      for (int i = threadIdx.x; i < cols * 32; i += kThreads) {
        const int col = i >> 5, d4 = (i & 31) * 4;
        float mm = -INFINITY, ll = 0.0f, sum[4] = {0, 0, 0, 0};
        bool any = false;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sh_m[w][col]), any |= sh_seen[w][col] != 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (sh_seen[w][col] == 0) continue;
          const float ref = mm == -INFINITY ? 0.0f : mm;
          ll = fmaf(sh_l[w][col], sh_m[w][col] == -INFINITY && sh_l[w][col] == 0.0f ? 0.0f : exp2_fast(sh_m[w][col] - ref), ll);
          const float f = sh_mv[w][col] == -INFINITY ? 1.0f : exp2_fast(sh_mv[w][col] - ref + kLift);  // a part without a finite score is 0 or NaN
#pragma unroll
          for (int k = 0; k < 4; ++k) sum[k] = fmaf(sh_o[(w * kKvHeadDim + d4 + k) * (kCols + 1) + col], f, sum[k]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (sh_nan[d4 + k] >> col & 1) sum[k] = NAN;
        const int at = col0 + col, row = s.row0 + at / g.group, qh = head * g.group + at % g.group;
        if (splits.grid > 1) {
          float* part = parts + ((size_t(row) * g.heads + qh) * splits.grid + split) * kPartFloats;
          *reinterpret_cast<float4*>(part + d4) = make_float4(sum[0], sum[1], sum[2], sum[3]);
          if (d4 == 0) *reinterpret_cast<float4*>(part + 128) = make_float4(mm, ll, any ? 1.0f : 0.0f, float(used));
        } else {
          const float inv = any ? (ll == 0.0f ? NAN : 1.0f / ll) : 0.0f;  // keys but no finite score: NaN; no key: zeros
          uint2 v;
          __nv_bfloat162 lo = __floats2bfloat162_rn(sum[0] * inv, sum[1] * inv), hi = __floats2bfloat162_rn(sum[2] * inv, sum[3] * inv);
          v.x = *reinterpret_cast<const uint32_t*>(&lo), v.y = *reinterpret_cast<const uint32_t*>(&hi);
          *reinterpret_cast<uint2*>(g.out + size_t(row) * g.ld_out + qh * kKvHeadDim + d4) = v;
        }
      }
    }
  }
}

// The parts of a row and head in order: a warp for each of them, or (WIDE, many parts) four warps with a quarter of the parts each.
template <bool WIDE>
__global__ void __launch_bounds__(128) kv_join_kernel(KvCacheView c, KvAttentionArgs g, const float* parts, int splits) {
  constexpr int kWarps = WIDE ? 4 : 1, kEach = WIDE ? kMostSplits / 32 : 1;  // parts a lane looks at
  static_assert(kNarrowSplits <= 32, "one part a lane");
  __shared__ float4 sh_o[4][32];
  __shared__ float sh_l[4];
  grid_dependency_release();
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part0 = WIDE ? warp : 0;
  for (int b = blockIdx.y; b < c.batch; b += gridDim.y) {
    const KvSequence s = kv_sequence(c, b);
    const int units = s.rows * g.heads;
    for (int unit = WIDE ? blockIdx.x : blockIdx.x * 4 + warp; unit < units; unit += gridDim.x * (WIDE ? 1 : 4)) {
      const int row = s.row0 + unit / g.heads, qh = unit % g.heads;
      const float* part = parts + (size_t(row) * g.heads + qh) * splits * kPartFloats;
      float mm = -INFINITY, f[kEach];
      bool any = false;
      float4 st[kEach];
#pragma unroll
      for (int h = 0; h < kEach; ++h) {
        const int i = lane + 32 * h;
        st[h] = i < splits ? *reinterpret_cast<const float4*>(part + i * kPartFloats + 128) : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
      }
      const int each = (splits + kWarps - 1) / kWarps, begin = part0 * each;
      constexpr int kAhead = 4;
      float4 o[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (begin + k < min(splits, begin + each)) o[k] = *reinterpret_cast<const float4*>(part + (begin + k) * kPartFloats + lane * 4);
      // The sequence's parts may be fewer than the launch's; what stands in the others' places has been read along and is not used.
      const int used = int(__shfl_sync(0xffffffffu, st[0].w, 0)), end = min(used, begin + each);
#pragma unroll
      for (int h = 0; h < kEach; ++h) {
        if (lane + 32 * h >= used) st[h] = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        mm = fmaxf(mm, st[h].x), any |= st[h].z != 0.0f;
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, off));
      any = __any_sync(0xffffffffu, any);
      // a part without a finite score has weight 1: it is zeros, or NaN
#pragma unroll
      for (int h = 0; h < kEach; ++h) f[h] = st[h].x == -INFINITY ? 1.0f : exp2_fast(st[h].x - (mm == -INFINITY ? 0.0f : mm));
      float ll = 0.0f;
      float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int i0 = begin; i0 < end; i0 += kAhead) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int i = i0 + k;
          if (i >= end) break;
          float w = f[0], li = st[0].y;
#pragma unroll
          for (int h = 1; h < kEach; ++h) w = i >= 32 * h ? f[h] : w, li = i >= 32 * h ? st[h].y : li;
          w = __shfl_sync(0xffffffffu, w, i & 31), li = __shfl_sync(0xffffffffu, li, i & 31);
          ll = fmaf(li, w, ll);
          sum.x = fmaf(o[k].x, w, sum.x), sum.y = fmaf(o[k].y, w, sum.y), sum.z = fmaf(o[k].z, w, sum.z), sum.w = fmaf(o[k].w, w, sum.w);
          if (i + kAhead < end) o[k] = *reinterpret_cast<const float4*>(part + (i + kAhead) * kPartFloats + lane * 4);
        }
      }
      if constexpr (WIDE) {
        __syncthreads();  // the row in front has been read
        sh_o[warp][lane] = sum;
        if (lane == 0) sh_l[warp] = ll;
        __syncthreads();
        if (warp != 0) continue;
        ll = 0.0f;
        sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 v = sh_o[w][lane];
          ll += sh_l[w], sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
      }
      const float inv = any ? (ll == 0.0f ? NAN : 1.0f / ll) : 0.0f;
      const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x * inv, sum.y * inv), hi = __floats2bfloat162_rn(sum.z * inv, sum.w * inv);
      *reinterpret_cast<uint2*>(g.out + size_t(row) * g.ld_out + qh * kKvHeadDim + lane * 4) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

struct AttentionPlan {
  int nt, col_tiles, warps;
  Splits splits;
};

// How a launch is divided, from the host's estimates.
AttentionPlan plan_for(const KvCacheView& c, int heads, int rows) {
  AttentionPlan p;
  const long long cols = (long long)std::min(c.max_new, rows) * (heads / c.kv_heads);
  p.nt = cols > 16 ? 3 : cols > 8 ? 2 : 1;
  p.col_tiles = int(std::min<long long>((cols + p.nt * 8 - 1) / (p.nt * 8), 4096));
  const long long ctas = (long long)c.batch * c.kv_heads * p.col_tiles;
  // Waves of CTAs times what a CTA takes: about 4 us around its tiles and, with its SM full, 4.5 us for one of a warp's tiles (one query tile
  // of eight; 6.5 and 10 with two and three), and 2 us for joining. A CTA of eight warps is alone on its SM. Sequences of different lengths
  // are taken to have three quarters of the parts that as many of the longest would have. 32 sequences, 8 kv heads, in 1 .. 6 parts: all of
  // 4096 tokens 59.3 / 66.3 / 55.4 / 60.2 / 59.0 / 61.7 us, of up to 4096 58.0 / 40.6 / 48.9 / 43.4 / 47.5 / 47.2; 16 of up to 3001 with five
  // new tokens, 10 kv heads 77.5 / 49.4 / 61.0 / 54.2 / 54.6 / 56.8; one of 131072: 58.6 / 52.8 / 70.7 in 37 / 55 / 64.
  const int per_tile = p.nt == 1 ? 45 : p.nt == 2 ? 65 : 100, tiles = (c.max_len - 1) / kTile + 1;
  // The number of parts that takes least, with all of `live` quarters of the longest sequence's parts there.
  auto best = [&](int live, int most_warps, int& parts, int& warps) {
    long long least = LLONG_MAX;
    for (int w = warps; w <= most_warps; w += 4) {
      const long long resident = (w == 4 ? kResident[p.nt] : 1) * kSms;
      for (int n = 1; n <= std::min(kMostSplits, tiles); ++n) {
        const long long waves = (ctas * n * live + 4 * resident - 1) / (4 * resident), each = ((tiles + n - 1) / n + w - 1) / w;
        const long long cost = waves * (40 + each * per_tile) + (n > 1 ? 20 : 0);
        if (cost < least) least = cost, parts = n, warps = w;
      }
    }
  };
  p.warps = 4;
  best(4, 8, p.splits.even, p.warps);
  p.splits.ragged = p.splits.even;
  if (c.batch > 1) best(3, p.warps, p.splits.ragged, p.warps);
  p.splits.grid = std::max(p.splits.even, p.splits.ragged);
  return p;
}

}  // namespace

static void check_heads(const KvCacheView& c, int heads) {
  if (heads <= 0 || heads > 32768 || heads % c.kv_heads != 0) throw std::invalid_argument("kv attention: heads must be a multiple of kv_heads");
}

static size_t workspace_of(const AttentionPlan& p, int heads, int rows) { return p.splits.grid > 1 ? size_t(rows) * heads * p.splits.grid * kPartFloats * sizeof(float) : 0; }

size_t kv_attention_workspace_bytes(const KvCacheView& c, int head_dim, int heads, int rows) {
  kv_check(c, head_dim);
  check_heads(c, heads);
  if (rows <= 0) return 0;
  return workspace_of(plan_for(c, heads, rows), heads, rows);
}

void kv_attention(KvCacheView c, int head_dim, KvAttentionArgs g, float scale, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  kv_check(c, head_dim);
  check_heads(c, g.heads);
  if (c.rows <= 0) return;
  if ((long long)c.rows * g.heads > 0x7FFFFFFF) throw std::invalid_argument("kv attention: too many rows and heads");
  if (!g.q || !g.out) throw std::invalid_argument("kv attention: null operand");
  if (g.ld_q < g.heads * kKvHeadDim || g.ld_out < g.heads * kKvHeadDim || g.ld_q % 8 != 0 || g.ld_out % 8 != 0 || !aligned16(g.q) || !aligned16(g.out))
    throw std::invalid_argument("kv attention: row pitches must cover heads * 128 columns and keep 16-byte alignment");
  if (rows_overlap(g.q, g.ld_q, g.heads * kKvHeadDim, g.out, g.ld_out, g.heads * kKvHeadDim, c.rows)) throw std::invalid_argument("kv attention: out may not overlap q");
  if (!std::isfinite(scale)) throw std::invalid_argument("kv attention: scale is not finite");
  const AttentionPlan p = plan_for(c, g.heads, c.rows);
  const size_t need = workspace_of(p, g.heads, c.rows);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
    throw std::invalid_argument("kv attention: workspace too small or not 16-byte aligned");
  g.group = g.heads / c.kv_heads;
  g.scale_log2 = (scale > 0.0f ? scale : 0.08838834764831845f) * 1.4426950408889634f;
  c.status = device_status_word();
  float* parts = static_cast<float*>(workspace);
  const dim3 grid(c.kv_heads * std::min(c.batch, 65535), p.col_tiles, p.splits.grid);
  const size_t smem = size_t(p.warps) * 2 * kTileBytes;
  const auto kernel = p.warps == 4 ? (p.nt == 1 ? kv_attention_kernel<1, 4> : p.nt == 2 ? kv_attention_kernel<2, 4> : kv_attention_kernel<3, 4>)
                                   : (p.nt == 1 ? kv_attention_kernel<1, 8> : p.nt == 2 ? kv_attention_kernel<2, 8> : kv_attention_kernel<3, 8>);
  reserve_dynamic_smem(reinterpret_cast<const void*>(kernel), smem, "kv attention");
  cudaError_t e = launch_overlapped(0, kernel, grid, dim3(p.warps * 32), smem, stream, c, g, parts, p.splits);
  if (e == cudaSuccess && p.splits.grid > 1) {
    const bool wide = p.splits.grid > kNarrowSplits;
    const long long units = (long long)std::min(c.max_new, c.rows) * g.heads, ctas = wide ? units : (units + 3) / 4;
    e = launch_overlapped(0, wide ? kv_join_kernel<true> : kv_join_kernel<false>, dim3(unsigned(std::min(ctas, 65535ll)), std::min(c.batch, 65535)), dim3(128), 0,
                          stream, c, g, static_cast<const float*>(parts), p.splits.grid);
  }
  if (e != cudaSuccess) throw std::runtime_error(std::string("kv attention: launch failed: ") + cudaGetErrorString(e));
}

}  // namespace sfq
