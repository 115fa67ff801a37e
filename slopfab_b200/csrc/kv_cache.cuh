// What the two operators over the paged 8-bit cache share: its description on the device and how a sequence is found in it.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kernels.cuh"

namespace sfq {

constexpr int kKvHeadDim = 128;
// Codes of the device status word (sfq_device_status).
constexpr int kKvBadSequence = 40;  // row starts out of order or out of range, a length below the new tokens or above the table
constexpr int kKvBadPage = 41;      // a page index outside the pool
constexpr int kKvBadPosition = 42;  // a rotation position outside the tables

struct KvSequence {
  int row0, rows;   // its rows of q, k, v
  long long length;  // cached tokens, the new ones among them
};

__device__ __forceinline__ KvSequence kv_sequence(const KvCacheView& c, int b) {
  KvSequence s;
  const int begin = c.row_start[b], end = c.row_start[b + 1];
  s.row0 = min(max(begin, 0), c.rows);
  s.rows = min(max(end, s.row0), c.rows) - s.row0;
  s.length = c.seq_len[b];
  if (begin != s.row0 || end != s.row0 + s.rows || s.length < s.rows || s.length > ((long long)c.max_pages << c.page_shift)) {
    if (threadIdx.x == 0) atomicCAS(c.status, 0, kKvBadSequence);
  }
  return s;
}

// The pool's page of a sequence's p-th page, -1 (and a status code) where the table names none.
__device__ __forceinline__ int kv_page(const KvCacheView& c, int b, long long p) {
  if (p < 0 || p >= c.max_pages) return -1;
  const int page = c.table[(long long)b * c.max_pages + p];
  if (page < 0 || page >= c.num_pages) {
    atomicCAS(c.status, 0, kKvBadPage);
    return -1;
  }
  return page;
}

// Whether a [rows, cols_a] and b [rows, cols_b] bf16, row pitches ld_a and ld_b, share elements. With different pitches the whole extents
// are compared.
inline bool rows_overlap(const void* a, long long ld_a, int cols_a, const void* b, long long ld_b, int cols_b, int rows) {
  const long long from = static_cast<const char*>(b) - static_cast<const char*>(a), end_a = ((rows - 1) * ld_a + cols_a) * 2, end_b = ((rows - 1) * ld_b + cols_b) * 2;
  if (from >= end_a || from + end_b <= 0) return false;
  if (rows == 1 || ld_a != ld_b) return true;
  const long long pitch = ld_a * 2, apart = (from % pitch + pitch) % pitch;
  return apart < cols_a * 2ll || apart + cols_b * 2ll > pitch;
}

}  // namespace sfq
