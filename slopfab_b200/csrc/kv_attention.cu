// Attention of a few new tokens per sequence over the paged 8-bit cache, grouped heads, causal among the new tokens.
//
// Bound by memory: every sequence's e4m3 codes of K and V are read once, 256 bytes for a token and kv head.
#include <cuda_fp8.h>

#include <cfloat>
#include <stdexcept>
#include <string>

#include "codec.cuh"
#include "kv_cache.cuh"
#include "ptx.cuh"
#include "runtime.h"

namespace sfq {
namespace {

using namespace ptx;

constexpr int kWarps = 4;

// One warp per (row, head): a lane holds four channels, one key after the other with the running maximum and sum.
__global__ void __launch_bounds__(kWarps * 32) kv_attention_kernel(KvCacheView c, KvAttentionArgs g) {
  grid_dependency_release();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int page_size = 1 << c.page_shift;
  for (int b = blockIdx.y; b < c.batch; b += gridDim.y) {
    const KvSequence s = kv_sequence(c, b);
    for (long long unit = blockIdx.x * kWarps + int(threadIdx.x >> 5); unit < (long long)s.rows * g.heads; unit += gridDim.x * kWarps) {
      const int i = int(unit / g.heads), head = int(unit % g.heads), kv_head = head / g.group;
      const __nv_bfloat16* q = g.q + size_t(s.row0 + i) * g.ld_q + head * kKvHeadDim + lane * 4;
      float qv[4], o[4] = {0, 0, 0, 0}, m = -FLT_MAX, sum = 0.0f;
      for (int e = 0; e < 4; ++e) qv[e] = __bfloat162float(q[e]);
      bool any = false;
      const long long sees = min(s.length - s.rows + i + 1, (long long)c.max_pages << c.page_shift);
      for (long long t = 0; t < sees; ++t) {
        const int page = kv_page(c, b, t >> c.page_shift);
        if (page < 0) continue;
        any = true;
        const size_t block = size_t(page) * c.kv_heads + kv_head;
        const int slot = int(t & (page_size - 1));
        const uint8_t* k = c.k + (block * page_size + slot) * kKvHeadDim + lane * 4;
        float score = 0.0f;
        for (int e = 0; e < 4; ++e) score = fmaf(qv[e], e4m3_decode(k[e]), score);
        for (int off = 16; off > 0; off >>= 1) score += __shfl_xor_sync(0xffffffffu, score, off);
        score *= c.k_scale[block] * g.scale_log2;
        float m_new = score > m ? score : m;
        if (!(score < INFINITY)) m_new = NAN;  // a NaN or +inf score makes its row NaN
        if (m != m) m_new = m;
        const float p = exp2f(score - m_new), keep = exp2f(m - m_new);
        m = m_new;
        sum = fmaf(sum, keep, p);
        const float pv = p * c.v_scale[block];
        for (int e = 0; e < 4; ++e) o[e] = fmaf(o[e], keep, pv * e4m3_decode(c.v[(block * kKvHeadDim + lane * 4 + e) * page_size + slot]));
      }
      const float inv = any ? (m > -FLT_MAX ? 1.0f / sum : NAN) : 0.0f;  // no key: zeros; no finite score: NaN
      __nv_bfloat16* out = g.out + size_t(s.row0 + i) * g.ld_out + head * kKvHeadDim + lane * 4;
      for (int e = 0; e < 4; ++e) out[e] = __float2bfloat16(o[e] * inv);
    }
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

size_t kv_attention_workspace_bytes(const KvCacheView& c, int head_dim, int heads) {
  kv_check(c, head_dim);
  if (heads <= 0 || heads > 32768 || heads % c.kv_heads != 0) throw std::invalid_argument("kv attention: heads must be a multiple of kv_heads");
  return 256;
}

void kv_attention(KvCacheView c, int head_dim, KvAttentionArgs g, float scale, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  const size_t need = kv_attention_workspace_bytes(c, head_dim, g.heads);
  if (c.rows <= 0) return;
  if (!g.q || !g.out || !workspace) throw std::invalid_argument("kv attention: null operand");
  if (workspace_bytes < need) throw std::invalid_argument("kv attention: workspace too small");
  if (g.ld_q < g.heads * kKvHeadDim || g.ld_out < g.heads * kKvHeadDim || g.ld_q % 8 != 0 || g.ld_out % 8 != 0 || !aligned16(g.q) || !aligned16(g.out))
    throw std::invalid_argument("kv attention: row pitches must cover heads * 128 columns and keep 16-byte alignment");
  if (g.q == g.out) throw std::invalid_argument("kv attention: out may not alias q");
  g.group = g.heads / c.kv_heads;
  g.scale_log2 = (scale > 0.0f ? scale : 0.08838834764831845f) * 1.4426950408889634f;
  c.status = device_status_word();
  const long long units = ((long long)c.max_new * g.heads + kWarps - 1) / kWarps;
  const cudaError_t e = launch_overlapped(0, kv_attention_kernel, dim3(unsigned(units < 65535 ? units : 65535), c.batch < 65535 ? c.batch : 65535), dim3(kWarps * 32), 0, stream, c, g);
  if (e != cudaSuccess) throw std::runtime_error(std::string("kv attention: launch failed: ") + cudaGetErrorString(e));
}

}  // namespace sfq
