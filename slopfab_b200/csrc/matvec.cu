// y = act(W x + b) for few rows of x, W as stored in 4 bits with group scales (NVFP4, NF4).
//
// Bound by the weight's bytes: N K / 2 codes and N K / 16 (NVFP4) or about N K / 64 (NF4) scale bytes are read once, whatever the
// number of rows. At the measured copy rate an SM is sent 41 weights a clock, and its integer pipe does 64 operations a clock, so a
// weight may cost about one and a half instructions. That decides the arithmetic:
//   - products on mma.sync m16n8k16 (fp16 operands, fp32 sums): 16 weight rows are its M, up to 8 rows of x its N. One MMA takes 256
//     weights; tcgen05 would need whole tiles of decoded weights in shared memory first.
//   - NVFP4: a byte becomes two fp16 by one conversion instruction, times its group's scale by one packed product. 2 + 4 significant bits
//     and 2^-10 .. 2688 are exact in fp16. bf16 weights would need five integer instructions a pair.
//   - NF4: a byte is looked up as two fp16 in a table of all 256 bytes that has a copy for each lane's bank; the absmax of 64 elements
//     scales the fp32 sum of their four MMAs. The 16 entries are rounded to the eleven bits of the MMA's operands, by 2^-12 of each at most
//     (the dense arm rounds every weight to the eight of bf16): a second term would take another look-up, which is what bounds this
//     form, and another MMA, for a result that differs from 64 bits by 1.667e-3 of its norm where fp32 entries leave 1.661e-3.
//   - x becomes fp16 times a power of two for each row, exactly: see stage_x.
// CTAs stay for the whole launch, so that x is made fp16 once per SM. Their warps form teams; a team takes 16 MT weight rows at a time,
// its warps take turns along K in steps of 128, each with its own ring of asynchronous copies that runs on into the next rows, and their
// sums meet in shared memory in a fixed order.
// Measured in a graph, weights in turn from HBM (a copy of the weight would take half to a quarter of this): NVFP4 1 x 5120 -> 15360
// 13.0 us (3.4 TB/s), 8 x 5120 -> 27648 with SwiGLU 21.0 (3.8), NF4 3 x 13824 -> 5120 21.5 (1.7), 16 x 5120 -> 13824 with GELU 27.2 (1.3).
// About 5 us are the launch, x and the first loads; without the products the four take 9.9, 18.1, 12.2 and 20.2 us, so that NVFP4 is near
// what its loads take and NF4 is bound by the reads of its table and of x from shared memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "codec.cuh"
#include "kernels.cuh"
#include "ptx.cuh"
#include "runtime.h"

namespace sfq {
namespace {

using namespace ptx;

constexpr size_t kMostSmem = 229376;  // dynamic; the kernel has about 2 KB of its own
constexpr int kMostRows = 16;      // rows of x in one launch
constexpr int kStep = 128;         // elements of K a warp takes at a time
constexpr int kTableBytes = 65536; // NF4: entry of byte b for lane l at b * 256 + l * 4

// Floats of a row of a warp's sums: one more than it has, against bank conflicts, where there is room.
__host__ __device__ constexpr int sum_pitch(bool nf4, int nt) { return nt * 8 + (nf4 && nt == 2 ? 0 : 1); }

struct Zero {  // a number that is known to be 0
  __device__ __forceinline__ Zero(int) {}
  __device__ __forceinline__ constexpr operator int() const { return 0; }
};

// What a team's sums of a unit take in a cluster's exchange: at most 256 outputs, halves of SwiGLU pairs counted, and a share that is rounded up.
constexpr int kSwapBytes = 1024 + 64;

struct Plan {
  int units = 0;  // groups of MT tiles of 16 weight rows
  int ring_off = 0, part_off = 0, swap_off = 0, x_off = 0;  // byte offsets into shared memory
  int cluster = 1;  // CTAs that divide K
};

__device__ __forceinline__ void named_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4_or_zero(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}

__device__ __forceinline__ void st_cluster(uint32_t cluster_addr, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory"); }

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The four bytes of w as pairs of fp16, low nibble in the low half, each pair times the scale pair s.
__device__ __forceinline__ void decode_e2m1(uint32_t w, uint32_t s, uint32_t (&v)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t.reg .b32 t;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 t, b0;\n\tmul.f16x2 %0, t, %5;\n\tcvt.rn.f16x2.e2m1x2 t, b1;\n\tmul.f16x2 %1, t, %5;\n\t"
      "cvt.rn.f16x2.e2m1x2 t, b2;\n\tmul.f16x2 %2, t, %5;\n\tcvt.rn.f16x2.e2m1x2 t, b3;\n\tmul.f16x2 %3, t, %5;\n\t}"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
      : "r"(w), "r"(s));
}
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t two) {
  uint32_t v;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(v) : "h"(uint16_t(two)));
  return v;
}

__device__ __forceinline__ float activated(float z, float up, int act) {
  if (act == SFQ_ACT_GELU_TANH) return 0.5f * z * (1.0f + tanhf(0.7978845608028654f * (z + 0.044715f * z * z * z)));
  if (act == SFQ_ACT_SWIGLU) return z / (1.0f + __expf(-z)) * up;
  return z;
}

// The weight row that is row i of 16-row tile t. NVFP4 keeps the scales of rows n, n + 32, n + 64, n + 96 side by side, so a tile takes four
// neighbours from each of the four quarters of 128 rows, whose scales for 64 elements are 64 bytes in a piece (with SwiGLU two quarters
// of gate rows, and the same of up rows). Rows past the end of an NF4 weight stand for its last one and are not stored.
template <bool NF4> __device__ __forceinline__ int weight_row(int t, int i, int out, bool swiglu) {
  if (swiglu) {
    const int j = i & 7, half = out >> 1;
    const int col = NF4 ? min(t * 8 + j, half - 1) : (t >> 3) * 64 + (j >> 2) * 32 + (t & 7) * 4 + (j & 3);
    return (i < 8 ? 0 : half) + col;
  }
  return NF4 ? min(t * 16 + i, out - 1) : (t >> 3) * 128 + (i >> 2) * 32 + (t & 7) * 4 + (i & 3);
}

// fp16 is as good as bf16 for x where every element of a row lies within 32 binades: times a power of two, its eight significant bits fit
// (as subnormals at the lower end). The first attempt takes 2^6, good for zeros and 2^-23 <= |x| < 2^10. Rows with others are sent
// through the weight again, with the exponent of their own largest element and, where they span more than 32 binades, in bands of 32
// binades, the smallest first. Infinities and NaN go with the topmost band. What that costs, 13824 -> 5120 in a graph, 1 / 3 / 8 rows: NVFP4
// 15.3 / 16.6 / 24.5 us in the first attempt, 45 / 50 / 53 off its range, 60 / 71 / 144 in two bands; NF4 20.2 / 21.6 / 25.9, 43 / 56 / 55,
// 58 / 77 / 150. Of calls on silu(g) u, 13824 wide, with deviations of 1 and 1, 3 / 10 / 24 % are off the range; of 0.2 and 0.1, 70 / 97 / 100 %.
constexpr int kFixedExponent = 8;  // the largest exponent of the first attempt's range is one above it

// One element of x for band `band` below row exponent e: times 2^(14 - e + 32 band), 0 where it belongs to another band.
__device__ __forceinline__ float banded(float f, int e, int band) {
  const uint32_t u = __float_as_uint(f) & 0x7FFFFFFFu;
  if (u >= 0x7F800000u) return band == 0 ? f : 0.0f;
  if (u == 0) return 0.0f;
  const int mine = u >= 0x800000u ? int(u >> 23) - 127 : 31 - __clz(int(u)) - 149;
  const int which = (e - mine) >> 5;
  if (which != band) return 0.0f;
  return ldexpf(f, 14 - e + 32 * band);
}

template <bool NF4, int NT, int MT, int D, int WARPS, int kTeamWarps, bool CLUSTER>
__global__ void __launch_bounds__(WARPS * 32, (!NF4 && D == 4) ? 2 : 1) matvec_kernel(MatvecArgs g, Plan p) {
  constexpr int kThreads = WARPS * 32, TEAMS = WARPS / kTeamWarps;
  constexpr int kStage = MT * 1024 + (NF4 ? 0 : MT * 128);  // codes [MT][16 rows][64 bytes], scales [MT][2 slabs][16 rows][4 bytes]
  constexpr int kPitch = sum_pitch(NF4, NT);
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int row_e[kMostRows], row_low[kMostRows];
  __shared__ float nested_map[NF4 ? 256 : 1];
  const int warp = (threadIdx.x >> 5) % kTeamWarps, team = threadIdx.x / (kTeamWarps * 32), lane = threadIdx.x & 31, gq = lane >> 2, q = lane & 3;
  const bool swiglu = g.act == SFQ_ACT_SWIGLU;
  // A cluster's CTAs take the same rows and each its part of K, steps begin .. end - 1.
  const int cluster = CLUSTER ? p.cluster : 1, rank = CLUSTER ? int(cluster_ctarank()) : 0;
  const int first_cta = CLUSTER ? int(blockIdx.x) / cluster : int(blockIdx.x), all_ctas = CLUSTER ? int(gridDim.x) / cluster : int(gridDim.x);
  const int all_steps = (g.in + kStep - 1) / kStep, steps = CLUSTER ? all_steps * (rank + 1) / cluster : all_steps;
  const std::conditional_t<CLUSTER, int, Zero> begin = all_steps * rank / cluster;
  const uint32_t base = smem_u32(smem);
  const uint32_t ring = base + p.ring_off + (threadIdx.x >> 5) * D * kStage;
  const int first_unit = team * all_ctas + first_cta, all_teams = all_ctas * TEAMS;  // what is left over falls on different CTAs
  grid_dependency_release();
  if constexpr (CLUSTER) cluster_arrive();  // this CTA's shared memory is there

  // The copies under way: the next one is step `fs` of unit `fu`.
  int fu, fs;
  const uint8_t* src[MT][2];     // this lane's 16 bytes of rows gq and gq + 8 of each tile
  const uint8_t* scale_src[MT];  // NVFP4: four scales of row lane % 16, slab lane / 16
  auto seek = [&](int unit) {
    fu = unit, fs = int(begin) + warp;
    if (unit >= p.units) return;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        src[m][h] = g.data + size_t(weight_row<NF4>(unit * MT + m, gq + 8 * h, g.out, swiglu)) * (g.in / 2) + q * 16 + size_t(int(begin) + warp) * (kStep / 2);
      if constexpr (!NF4)
        scale_src[m] = g.scale + nvfp4_scale_offset(weight_row<NF4>(unit * MT + m, lane & 15, g.out, swiglu), (lane >> 4) * 4, g.in / 16) + size_t(int(begin) + warp) * (kStep * 8);
    }
  };
  const uint32_t code_at = gq * 64 + (NF4 ? q ^ (gq & 2) : q) * 16;  // in a tile's codes; NF4 is read in 8-byte pieces of four rows at a time
  auto fetch = [&](uint32_t to, int end_unit) {
    if (fs < steps && fu < end_unit) {
      if ((fs + 1) * kStep <= g.in) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          cp_async16(to + m * 1024 + code_at, src[m][0]);
          cp_async16(to + m * 1024 + code_at + 512, src[m][1]);
          if constexpr (!NF4) cp_async4(to + MT * 1024 + m * 128 + lane * 4, scale_src[m]);
        }
      } else {  // the half step at the end of a row: zeros in the place of the rest
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          cp_async16_or_zero(to + m * 1024 + code_at, q < 2 ? src[m][0] : g.data, q < 2);
          cp_async16_or_zero(to + m * 1024 + code_at + 512, q < 2 ? src[m][1] : g.data, q < 2);
          if constexpr (!NF4) cp_async4_or_zero(to + MT * 1024 + m * 128 + lane * 4, lane < 16 ? scale_src[m] : g.scale, lane < 16);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        src[m][0] += kTeamWarps * kStep / 2, src[m][1] += kTeamWarps * kStep / 2;
        if constexpr (!NF4) scale_src[m] += kTeamWarps * kStep * 8;
      }
      fs += kTeamWarps;
      if (fs >= steps) seek(fu + all_teams);
    }
    cp_commit();
  };
  // NF4: lane l holds the absmax of row l / 2, group l % 2 of a step: its byte and its nested scale, fetched a step ahead.
  const int last_group = g.in / 64 - 1;
  uint32_t absmax_byte[MT];
  float absmax_outer[MT], absmax[MT];
  uint32_t absmax_row[MT];  // its row's first group of 64
  auto seek_absmax = [&](int unit) {
    if constexpr (NF4) {
#pragma unroll
      for (int m = 0; m < MT; ++m) absmax_row[m] = uint32_t(weight_row<true>(unit * MT + m, lane >> 1, g.out, swiglu)) * uint32_t(last_group + 1);
    }
  };
  auto fetch_absmax = [&](int s) {
    if constexpr (NF4) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint32_t block = (absmax_row[m] + uint32_t(min(s * 2 + (lane & 1), last_group))) >> (g.block_shift - 6);
        absmax_byte[m] = g.scale[block], absmax_outer[m] = g.nested_absmax[block >> g.nested_shift];
      }
    }
  };

  float acc[MT][NT][4];
  auto scale_sums = [&](float by) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[m][n][e] = by == 0.0f ? 0.0f : acc[m][n][e] * by;
  };

  // x [rows, in] as fp16: 16 bytes of eight elements, pairs with the odd element in the low half, at unit
  // ((step * 4 + piece) * rows + row) * 4 + lane % 4, which is the order in which the MMAs' lanes read them.
  auto stage_x = [&](int band) -> bool {  // band < 0: the first attempt; true where an element does not fit it
    const int units = (steps - int(begin)) * kStep / 8, k0 = int(begin) * kStep;
    const __nv_bfloat162 least = __halves2bfloat162(__ushort_as_bfloat16(0x3400), __ushort_as_bfloat16(0x3400));  // 2^-23
    const __nv_bfloat162 sixty_four = __halves2bfloat162(__ushort_as_bfloat16(0x4280), __ushort_as_bfloat16(0x4280));
    const __nv_bfloat162 zero = __halves2bfloat162(__ushort_as_bfloat16(0), __ushort_as_bfloat16(0));
    uint32_t low = 0;
    __nv_bfloat162 top = zero;
    constexpr int kBatch = (!NF4 && D == 4) || WARPS > 16 ? 4 : 8;  // loads in flight
    int r = 0, k8 = threadIdx.x;
    if (CLUSTER && units == 0) return false;
    while (k8 >= units) k8 -= units, ++r;
    while (r < g.rows) {
      uint4 raw[kBatch];
      int rr[kBatch], kk[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        rr[i] = r, kk[i] = k8;
        raw[i] = r < g.rows && k0 + k8 * 8 < g.in ? *reinterpret_cast<const uint4*>(g.x + size_t(r) * g.in + k0 + k8 * 8) : make_uint4(0, 0, 0, 0);
        k8 += kThreads;
        while (k8 >= units) k8 -= units, ++r;
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (rr[i] >= g.rows) break;
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float even, odd;
          if (band < 0) {
            const uint32_t mag = w[j] & 0x7FFF7FFFu;
            const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&mag);
            low |= __hlt2_mask(a, least) & __hgt2_mask(a, zero);
            top = __hmax2(top, a);
            const __nv_bfloat162 up = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]), sixty_four);  // exact
            even = __low2float(up), odd = __high2float(up);
          } else {
            even = banded(__uint_as_float(w[j] << 16), row_e[rr[i]], band), odd = banded(__uint_as_float(w[j] & 0xFFFF0000u), row_e[rr[i]], band);
          }
          asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(o[j]) : "f"(even), "f"(odd));
        }
        const int step = kk[i] >> 4;
        const int piece = NF4 ? ((kk[i] >> 3) & 1) * 2 + (kk[i] & 1) : kk[i] & 3, quarter = NF4 ? (kk[i] >> 1) & 3 : (kk[i] >> 2) & 3;
        *reinterpret_cast<uint4*>(smem + p.x_off + (((step * 4 + piece) * g.rows + rr[i]) * 4 + quarter) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
    return low != 0 || fmaxf(__low2float(top), __high2float(top)) >= 1024.0f;
  };

  // Lanes of columns that stand for no row of x read another row's; what they add up is not stored.
  uint32_t x_at[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) x_at[n] = base + p.x_off + (min(gq + 8 * n, g.rows - 1) * 4 + q) * 16;
  const uint32_t x_piece = g.rows * 64;
  auto multiply = [&](int s, uint32_t from) {
    const uint32_t xs = (s - int(begin)) * 4 * x_piece;
    if constexpr (!NF4) {
      uint4 w[MT][2];
      uint32_t sc[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = gq + 8 * h;
          w[m][h] = lds128(from + m * 1024 + row * 64 + q * 16);
          sc[m][h] = e4m3_pair(lds16(from + MT * 1024 + m * 128 + (q >> 1) * 64 + row * 4 + (q & 1) * 2));
        }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint4 xv[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) xv[n] = lds128(x_at[n] + xs + j * x_piece);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          uint32_t a[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t word = j == 0 ? w[m][h].x : j == 1 ? w[m][h].y : j == 2 ? w[m][h].z : w[m][h].w;
            decode_e2m1(word, __byte_perm(sc[m][h], 0, j < 2 ? 0x1010 : 0x3232), a[h]);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_f16(acc[m][n], a[0][0], a[1][0], a[0][1], a[1][1], xv[n].x, xv[n].y);
            mma_f16(acc[m][n], a[0][2], a[1][2], a[0][3], a[1][3], xv[n].z, xv[n].w);
          }
        }
      }
    } else {  // a group past the end of a row: x is zeros, the codes are, too, and the absmax is the last group's
      const uint32_t lane4 = lane * 4;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint4 xv[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) xv[n][j] = lds128(x_at[n] + xs + (c * 2 + j) * x_piece);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          uint2 w[2];
          float scale[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = gq + 8 * h;
            w[h] = lds64(from + m * 1024 + row * 64 + ((c * 2 + (q >> 1)) ^ (row & 2)) * 16 + (q & 1) * 8);
            scale[h] = __shfl_sync(0xffffffffu, absmax[m], row * 2 + c);
          }
          float d[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.0f;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t a[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t word = j == 0 ? w[h].x : w[h].y;
#pragma unroll
              for (int i = 0; i < 4; ++i) a[h][i] = lds32(base + __byte_perm(word, lane4, 0x7704 | (i << 4)));
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_f16(d[n], a[0][0], a[1][0], a[0][1], a[1][1], xv[n][j].x, xv[n][j].y);
              mma_f16(d[n], a[0][2], a[1][2], a[0][3], a[1][3], xv[n][j].z, xv[n][j].w);
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            acc[m][n][0] = fmaf(d[n][0], scale[0], acc[m][n][0]), acc[m][n][1] = fmaf(d[n][1], scale[0], acc[m][n][1]);
            acc[m][n][2] = fmaf(d[n][2], scale[1], acc[m][n][2]), acc[m][n][3] = fmaf(d[n][3], scale[1], acc[m][n][3]);
          }
        }
      }
    }
  };

  // This warp's steps of a unit. Their first D - 1 copies are under way, and go on with the units up to end_unit.
  uint32_t slot = 0;  // byte offset into the ring
  auto walk = [&](int unit, int end_unit) {
    for (int s = int(begin) + warp; s < steps; s += kTeamWarps) {
      cp_wait<D - 2>();
      __syncwarp();  // the copies have landed in every lane, and the step in front has been read
      fetch(ring + (slot == 0 ? (D - 1) * kStage : slot - kStage), end_unit);
      if constexpr (NF4) {  // this step's absmax, and the loads of the next one's, which have the products' time to arrive
#pragma unroll
        for (int m = 0; m < MT; ++m) absmax[m] = fmaf(nested_map[absmax_byte[m]], absmax_outer[m], g.offset);
        if (s + kTeamWarps < steps) {
          fetch_absmax(s + kTeamWarps);
        } else if (unit + all_teams < end_unit) {
          seek_absmax(unit + all_teams);
          fetch_absmax(int(begin) + warp);
        }
      }
      multiply(s, ring + slot);
      slot = slot == (D - 1) * kStage ? 0 : slot + kStage;
    }
  };
  auto start = [&](int unit, int end_unit) {
    slot = 0;
    __syncwarp();
    seek(unit);
    for (int i = 0; i < D - 1; ++i) fetch(ring + i * kStage, end_unit);
    if (unit < end_unit && int(begin) + warp < steps) {
      seek_absmax(unit);
      fetch_absmax(int(begin) + warp);
    }
  };

  // The team's sums of a unit, added in the order of its warps, finished and stored. NF4 keeps them in the unused halves of the table's
  // lines. In a cluster each CTA finishes its share of the outputs: the others' shares go to them, over the row's power of two and the
  // tensor scale, and are added in the order of the ranks. Every team of every CTA takes part for every unit (those without one as -1),
  // and the two buffers take turns, so that one barrier a unit is enough.
  const int part0 = team * kTeamWarps * MT * 16 * kPitch;
  auto part = [&](int i) -> float& {
    const int at = part0 + i;
    return *reinterpret_cast<float*>(smem + (NF4 ? (at >> 5) * 256 + 128 + (at & 31) * 4 : p.part_off + at * 4));
  };
  const int cols = swiglu ? g.out / 2 : g.out, per_tile = swiglu ? 8 : 16, halves = swiglu ? 2 : 1;
  const int outputs = MT * per_tile * g.rows, share = (outputs + cluster - 1) / cluster;
  auto gather = [&](int unit) {  // every warp's sums into shared memory
    named_barrier(team + 1, kTeamWarps * 32);  // those of the unit in front have been read
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) part((warp * MT * 16 + m * 16 + gq + (e >> 1) * 8) * kPitch + n * 8 + q * 2 + (e & 1)) = acc[m][n][e];
    named_barrier(team + 1, kTeamWarps * 32);
  };
  int map_e = 0;  // NF4: exponent that the table is over
  auto summed = [&](int r, int row) {  // the team's sum of a row of the tiles and a row of x
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kTeamWarps; ++w) s += part((w * MT * 16 + row) * kPitch + r);
    return ldexpf(s * g.global_scale, row_e[r] - 14 + map_e);
  };
  auto bias_of = [&](int at) {
    return g.bias == nullptr ? 0.0f : g.bias_is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(g.bias)[at]) : static_cast<const float*>(g.bias)[at];
  };
  int turn = 0;
  auto finish = [&](int unit) {
    const uint32_t swap = base + p.swap_off + turn * TEAMS * kSwapBytes + team * kSwapBytes;  // cluster: [rank][halves][share]
    if (unit >= 0) {
      gather(unit);
      for (int i = warp * 32 + lane; i < outputs; i += kTeamWarps * 32) {
        const int r = i / (MT * per_tile), local = i - r * (MT * per_tile), m = local / per_tile, j = local - m * per_tile;
        if constexpr (!CLUSTER) {
          const int n = weight_row<NF4>(unit * MT + m, j, g.out, swiglu);
          if (NF4 && (unit * MT + m) * per_tile + j >= cols) continue;
          float z[2] = {0.0f, 0.0f};
          for (int h = 0; h < (swiglu ? 2 : 1); ++h) z[h] = summed(r, m * 16 + j + 8 * h) + bias_of(n + h * cols);
          g.y[size_t(r) * cols + n] = __float2bfloat16(activated(z[0], z[1], g.act));
        } else {
          const int owner = i / share;
          for (int h = 0; h < halves; ++h)
            st_cluster(map_to_rank(swap + ((rank * halves + h) * share + i - owner * share) * 4, owner), summed(r, m * 16 + j + 8 * h));
        }
      }
    }
    if constexpr (CLUSTER) {
      cluster_sync_all();
      if (unit >= 0) {
        for (int i = rank * share + warp * 32 + lane; i < min(outputs, (rank + 1) * share); i += kTeamWarps * 32) {
          const int r = i / (MT * per_tile), local = i - r * (MT * per_tile), m = local / per_tile, j = local - m * per_tile;
          const int n = weight_row<NF4>(unit * MT + m, j, g.out, swiglu);
          if (NF4 && (unit * MT + m) * per_tile + j >= cols) continue;
          float z[2] = {0.0f, 0.0f};
          for (int h = 0; h < halves; ++h) {
            for (int k = 0; k < cluster; ++k) z[h] += __uint_as_float(lds32(swap + ((k * halves + h) * share + i - rank * share) * 4));
            z[h] += bias_of(n + h * cols);
          }
          g.y[size_t(r) * cols + n] = __float2bfloat16(activated(z[0], z[1], g.act));
        }
      }
      turn ^= 1;
    }
  };

  grid_dependency_wait();
  start(first_unit, p.units);
  if (threadIdx.x < kMostRows) row_e[threadIdx.x] = kFixedExponent;
  const float map = NF4 ? g.map[lane & 15] : 0.0f, nested = NF4 ? g.nested_map[threadIdx.x & 255] : 0.0f;
  const bool misfit = stage_x(-1);
  if constexpr (NF4) {
    // the table: the entry of a byte, odd element (low nibble) in the low half, and its 32 copies. Entries are over the exponent of the
    // largest finite one, so that a map of any size is as good in fp16.
    const uint32_t size = __float_as_uint(map) & 0x7FFFFFFFu, top = __reduce_max_sync(0xffffffffu, size < 0x7F800000u ? size : 0u);
    map_e = top == 0 ? 0 : max(int(top >> 23), 1) - 127;
    const float even = ldexpf(map, -map_e);
    for (uint32_t i = threadIdx.x; i < 256 * 8; i += kThreads) {  // whole warps
      const uint32_t b = i >> 3;
      const __half2 pair = __floats2half2_rn(__shfl_sync(0xffffffffu, even, b & 15), __shfl_sync(0xffffffffu, even, b >> 4));
      const uint32_t v = *reinterpret_cast<const uint32_t*>(&pair);
      *reinterpret_cast<uint4*>(smem + b * 256 + (i & 7) * 16) = make_uint4(v, v, v, v);
    }
    if (threadIdx.x < 256) nested_map[threadIdx.x] = nested;
  }
  int bands = 0;
  if (__syncthreads_or(misfit)) {
    // Each row's largest exponent and lowest band, over its finite elements that are not zero.
    for (int r = threadIdx.x >> 5; r < g.rows; r += kThreads / 32) {
      int most = -1000, least = 1000;
      for (int k = int(begin) * kStep + lane; k < min(steps * kStep, g.in); k += 32) {
        const uint32_t u = __float_as_uint(__bfloat162float(g.x[size_t(r) * g.in + k])) & 0x7FFFFFFFu;
        if (u == 0 || u >= 0x7F800000u) continue;
        const int e = u >= 0x800000u ? int(u >> 23) - 127 : 31 - __clz(int(u)) - 149;
        most = max(most, e), least = min(least, e);
      }
      most = __reduce_max_sync(0xffffffffu, most), least = __reduce_min_sync(0xffffffffu, least);
      if (lane == 0) row_e[r] = most == -1000 ? 0 : most, row_low[r] = most == -1000 ? 0 : (most - least) >> 5;
    }
    __syncthreads();
    for (int r = 0; r < g.rows; ++r) bands = max(bands, row_low[r]);
    if (bands == 0) {
      stage_x(0);
      __syncthreads();
    }
  }
  if constexpr (CLUSTER) cluster_wait();
  if constexpr (!CLUSTER) {
    if (bands == 0) {
      for (int unit = first_unit; unit < p.units; unit += all_teams) {
        scale_sums(0.0f);
        walk(unit, p.units);
        finish(unit);
      }
    } else {
      for (int first = first_cta; first < p.units; first += all_teams) {  // the teams in step, since x changes under them
        const int unit = first + team * all_ctas;
        scale_sums(0.0f);
        for (int band = bands; band >= 0; --band) {
          cp_wait<0>();
          __syncthreads();
          stage_x(band);
          __syncthreads();
          start(unit, min(unit + 1, p.units));
          if (band < bands) scale_sums(0x1p-32f);
          if (unit < p.units) walk(unit, unit + 1);
        }
        if (unit < p.units) finish(unit);
      }
    }
  } else {
    for (int first = first_cta; first < p.units; first += all_teams) {  // all teams of all CTAs in step
      const int unit = first + team * all_ctas;
      scale_sums(0.0f);
      for (int band = bands; band >= 0; --band) {
        if (bands > 0) {
          cp_wait<0>();
          __syncthreads();
          stage_x(band);
          __syncthreads();
          start(unit, min(unit + 1, p.units));
          if (band < bands) scale_sums(0x1p-32f);
        }
        if (unit < p.units) walk(unit, bands > 0 ? unit + 1 : p.units);
      }
      finish(unit < p.units ? unit : -1);
    }
  }
  cp_wait<0>();
}

int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}
bool power_of_two(int v) { return v > 0 && (v & (v - 1)) == 0; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// What a launch with this kernel takes of shared memory for `rows` rows of x, with K divided over `cluster` CTAs.
template <bool NF4, int NT, int MT, int D, int WARPS> size_t plan(const MatvecArgs& g, int rows, int cluster, Plan& p) {
  const bool swiglu = g.act == SFQ_ACT_SWIGLU;
  const int tiles = NF4 ? ((swiglu ? g.out / 2 : g.out) + (swiglu ? 7 : 15)) / (swiglu ? 8 : 16) : g.out / 16;
  p.units = (tiles + MT - 1) / MT;
  p.cluster = cluster;
  size_t at = NF4 ? kTableBytes : 0;
  p.ring_off = int(at);
  at += size_t(WARPS) * D * (MT * 1024 + (NF4 ? 0 : MT * 128));
  p.part_off = int(at);
  const size_t sums = size_t(WARPS) * MT * 16 * sum_pitch(NF4, NT) * 4;
  if (!NF4) at += sums;
  static_assert(!NF4 || WARPS * MT * 16 * sum_pitch(NF4, NT) * 4 <= kTableBytes / 2, "the sums lie in the table's gaps");
  p.swap_off = int(at);
  if (cluster > 1) at += 2 * (WARPS / 4) * kSwapBytes;
  p.x_off = int(at);
  const int steps = (g.in + kStep - 1) / kStep;
  return at + size_t((steps + cluster - 1) / cluster) * kStep * rows * 2;
}

template <bool NF4, int NT, int MT, int D, int WARPS> bool fits(const MatvecArgs& g, int rows, int cluster) {
  Plan p;
  return plan<NF4, NT, MT, D, WARPS>(g, rows, cluster, p) <= kMostSmem;
}

template <bool NF4, int NT, int MT, int D, int WARPS, int TEAM, bool CLUSTER> void launch_team(const MatvecArgs& g, const Plan& p, size_t bytes, int resident, cudaStream_t stream) {
  const auto kernel = matvec_kernel<NF4, NT, MT, D, WARPS, TEAM, CLUSTER>;
  reserve_dynamic_smem(reinterpret_cast<const void*>(kernel), bytes, "matvec");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(std::min(p.units, resident * device_sm_count() / p.cluster) * p.cluster);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (p.cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = p.cluster, attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (size_t(g.out) * g.in / 2 <= kOverlapBytes) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr, cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, g, p);
  if (e != cudaSuccess) throw std::runtime_error(std::string("matvec: launch failed: ") + cudaGetErrorString(e));
}

// Whether the device runs clusters of four such CTAs, with all of an SM's shared memory each.
bool clusters_run() {
  static PerDevice<bool> cache;
  return cache.get([] {
    const auto kernel = matvec_kernel<true, 2, 1, 2, 16, 8, true>;
    reserve_dynamic_smem(reinterpret_cast<const void*>(kernel), kMostSmem, "matvec");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(4), cfg.blockDim = dim3(512), cfg.dynamicSmemBytes = kMostSmem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 4, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr, cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();
      return false;
    }
    return n >= 16;
  });
}

// Teams of eight warps, or of four where that takes no more steps: a warp then walks longer rows of steps and fewer sums are joined.
// 1 x 5120 -> 15360 NVFP4 13.4 us with eight, 12.1 with four (without the code for clusters beside them); NF4 3 x 13824 -> 5120, where eight take half the steps, 21.4 against 24.4.
template <bool NF4, int NT, int MT, int D, int WARPS, bool CLUSTER = false> void launch(const MatvecArgs& g, int cluster, cudaStream_t stream) {
  Plan p;
  const size_t bytes = plan<NF4, NT, MT, D, WARPS>(g, g.rows, cluster, p);
  const int resident = !NF4 && D == 4 && bytes <= kMostSmem / 2 - 1024 ? 2 : 1;
  const int steps = ((g.in + kStep - 1) / kStep + cluster - 1) / cluster, ctas = resident * device_sm_count() / cluster;
  auto cost = [&](int team) {
    const int teams = WARPS / team * ctas;
    return ((p.units + teams - 1) / teams) * ((steps + team - 1) / team);
  };
  if (cost(4) <= cost(8))
    launch_team<NF4, NT, MT, D, WARPS, 4, CLUSTER>(g, p, bytes, resident, stream);
  else
    launch_team<NF4, NT, MT, D, WARPS, 8, CLUSTER>(g, p, bytes, resident, stream);
}

// The most rows of x, up to `rows`, that one launch takes.
template <bool NF4> int most_rows(const MatvecArgs& g, int rows, int cluster) {
  int most = std::min(rows, kMostRows);
  while (most > 0 && !(most > 8 ? fits<NF4, 2, 1, 2, 16>(g, most, cluster) : fits<NF4, 1, 1, 2, 16>(g, most, cluster))) --most;
  return most;
}

template <bool NF4> void launch_rows(MatvecArgs g, int cols, cudaStream_t stream) {
  // Where x is too large for the shared memory of one CTA, it goes through in several launches, each of which reads the weight, or K is
  // divided over clusters of two CTAs, or of four where the weight has few rows. A cluster's CTAs meet for every 16 rows of W, which costs
  // about a microsecond: NF4 16 x 5120 -> 13824 33.7 us in two launches, 27.7 in clusters of two; 10 x 13376 -> 648 37.0 in three launches,
  // 17.2 in clusters of four.
  int rows = g.rows, cluster = 1, most = most_rows<NF4>(g, rows, 1);
  const int wanted = std::min(rows, kMostRows);
  for (int c = 2; most < wanted && c <= (g.out / 16 <= device_sm_count() || most == 0 ? 4 : 2) && clusters_run(); c *= 2) {
    const int with = most_rows<NF4>(g, rows, c);
    if (most == 0 || (with > 0 && (rows + with - 1) / with < (rows + most - 1) / most)) cluster = c, most = with;
  }
  if (most == 0) throw std::invalid_argument("matvec: in_features too large");
  for (int parts = (rows + most - 1) / most; rows > 0; --parts) {
    g.rows = (rows + parts - 1) / parts;
    // Two tiles a step share the reads of x. NVFP4 needs them from three rows of x on and has two CTAs an SM below that; NF4, bound by its
    // table's lookups, is better off with 24 warps up to four rows (3 x 13824 -> 5120 21.4 us; 16 warps 26.3; with two tiles, 8 rows
    // 5120 -> 13824 17.5 against 18.8).
    constexpr int kTwoTiles = NF4 ? 2 : 3;  // ring stages
    if (cluster > 1 && g.rows > 8)
      launch<NF4, 2, 1, 2, 16, true>(g, cluster, stream);
    else if (cluster > 1)
      launch<NF4, 1, 1, 2, 16, true>(g, cluster, stream);
    else if (g.rows > 8)
      launch<NF4, 2, 1, 2, 16>(g, 1, stream);
    else if (g.rows > (NF4 ? 4 : 2) && fits<NF4, 1, 2, kTwoTiles, 16>(g, g.rows, 1) && g.out >= 64 * device_sm_count())
      launch<NF4, 1, 2, kTwoTiles, 16>(g, 1, stream);
    else if (fits<NF4, 1, 1, NF4 ? 3 : 4, NF4 ? 24 : 16>(g, g.rows, 1))
      launch<NF4, 1, 1, NF4 ? 3 : 4, NF4 ? 24 : 16>(g, 1, stream);
    else
      launch<NF4, 1, 1, 2, 16>(g, 1, stream);
    rows -= g.rows;
    g.x += size_t(g.rows) * g.in;
    g.y += size_t(g.rows) * cols;
  }
}

}  // namespace

void linear_matvec(MatvecArgs g, int nf4_block, int nf4_nested_block, cudaStream_t stream) {
  if (g.rows <= 0) return;
  if (g.out <= 0 || g.in <= 0) throw std::invalid_argument("matvec: features must be positive");
  if (!g.x || !g.y || !g.data) throw std::invalid_argument("matvec: null operand");
  if (g.nf4) {
    if (!g.scale || !g.map || !g.nested_map || !g.nested_absmax) throw std::invalid_argument("matvec: nf4 weight without complete double-quant state");
    if (!aligned(g.map, 4) || !aligned(g.nested_map, 4) || !aligned(g.nested_absmax, 4)) throw std::invalid_argument("matvec: nf4 tables must be 4-byte aligned");
    if (!power_of_two(nf4_block) || nf4_block < 64 || !power_of_two(nf4_nested_block)) throw std::invalid_argument("matvec: nf4 blocks must be powers of two, of 64 elements at least");
    if (g.in % 64 != 0) throw std::invalid_argument("matvec: nf4 needs in_features % 64 == 0");
    if ((size_t(g.out) * g.in) >> 38 != 0) throw std::invalid_argument("matvec: nf4 weight of more than 2^38 elements");
    g.block_shift = log2_of(nf4_block), g.nested_shift = log2_of(nf4_nested_block);
    g.global_scale = 1.0f;
  } else {
    if (!g.scale) throw std::invalid_argument("matvec: block_scale is null");
    if (g.out % 128 != 0 || g.in % 64 != 0) throw std::invalid_argument("matvec: nvfp4 needs out_features % 128 == 0 and in_features % 64 == 0");
    if (!aligned(g.scale, 4)) throw std::invalid_argument("matvec: block_scale must be 4-byte aligned");
  }
  if (g.act == SFQ_ACT_SWIGLU && g.out % 2 != 0) throw std::invalid_argument("matvec: SwiGLU needs an even out_features");
  if (!aligned(g.data, 16) || !aligned(g.x, 16) || !aligned(g.y, 2)) throw std::invalid_argument("matvec: x and the weight must be 16-byte aligned");
  if (!aligned(g.bias, g.bias_is_bf16 ? 2 : 4)) throw std::invalid_argument("matvec: bias must be aligned to its elements");
  const int cols = g.act == SFQ_ACT_SWIGLU ? g.out / 2 : g.out;
  {
    const auto x0 = reinterpret_cast<uintptr_t>(g.x), x1 = x0 + size_t(g.rows) * g.in * 2, y0 = reinterpret_cast<uintptr_t>(g.y), y1 = y0 + size_t(g.rows) * cols * 2;
    if (x0 < y1 && y0 < x1) throw std::invalid_argument("matvec: x and y may not overlap");
  }
  if (g.nf4)
    launch_rows<true>(g, cols, stream);
  else
    launch_rows<false>(g, cols, stream);
}

}  // namespace sfq
