// Microscaled 4-bit rows: what their kernels share.  A row of K values holds
//   codes   ceil(K / 32) * 16 bytes, the even element in the low nibble, zeros past K
//   scales  one byte per block: mxfp4 2^(byte - 127) per 32 values, nvfp4 an e4m3 value per 16 (and one float32
//           scale t for the whole tensor)
// The scale bytes lie in the order the tensor cores take them: atoms of 512 bytes hold 128 rows x 4 block columns,
// byte (r % 32) * 16 + (r / 32 % 4) * 4 + c % 4, so that one 32 x 128-bit copy into tensor memory puts the four
// columns of row r into lane r % 32 of column r / 32.  Atoms of a row block follow each other along the columns,
// padded with zero bytes to whole 256 values (2 atoms for mxfp4, 4 for nvfp4).  A tensor of groups (experts) begins
// each group on a row block of its own, so a tile of 128 rows never takes scales from two groups.
#pragma once
#include "lb_common.cuh"
#include "../../include/apsi_lowbit.h"

namespace lb {
namespace mx {

__host__ __device__ constexpr int block_of(int fmt) { return fmt == LB_FMT_MXFP4 ? 32 : 16; }
// atoms of a row block per 256 values
__host__ __device__ constexpr int atoms256(int fmt) { return fmt == LB_FMT_MXFP4 ? 2 : 4; }
__host__ __device__ inline int64_t row_bytes(int64_t K) { return (K + 31) / 32 * 16; }
__host__ __device__ inline int64_t atom_cols(int fmt, int64_t K) { return (K + 255) / 256 * atoms256(fmt); }

// byte offset of the scale of (row in its group, block column) from the group's first row block
__host__ __device__ inline int64_t scale_at(int64_t r, int64_t c, int64_t acols) {
  return ((r >> 7) * acols + (c >> 2)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (c & 3);
}

// The row groups of a tensor: G == 0: one group of all rows; per > 0: groups of `per` rows each (expert weights);
// otherwise rows [offsets[e], offsets[e + 1]) are group e (offsets on the device).
struct Groups {
  const int* offsets;
  int G;
  int64_t per;
};

// Ragged groups in shared memory: off[e] (made non-decreasing and held in [0, R], so that no bad offset can lead
// outside the tensor; LB_DEVERR_BAD_INDEX says that it happened) and base[e], the row blocks before group e.  All
// threads of the block call it; off and base have G + 1 words.  One warp scans, 32 groups at a time.
__device__ __forceinline__ void load_groups(const Groups& g, int64_t R, int* off, int* base) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int top = 0, blocks = 0;
    bool bad = false;
    for (int e0 = 0; e0 <= g.G; e0 += 32) {
      const int e = e0 + lane;
      const int raw = e <= g.G ? g.offsets[e] : 0;
      int v = raw < 0 ? 0 : (raw > R ? static_cast<int>(R) : raw);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o && u > v) v = u;
      }
      if (top > v) v = top;
      bad |= e <= g.G && v != raw;
      int prev = __shfl_up_sync(0xffffffffu, v, 1);
      if (lane == 0) prev = e0 ? top : v;
      // row blocks of the group that ends at v
      int n = (v - prev + 127) >> 7;
      if (e > g.G) n = 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += u;
      }
      if (e <= g.G) {
        off[e] = v;
        base[e] = blocks + n;
      }
      blocks += __shfl_sync(0xffffffffu, n, 31);
      top = __shfl_sync(0xffffffffu, v, 31);
    }
    if (bad) atomicOr(&g_dev_errors, LB_DEVERR_BAD_INDEX);
  }
  __syncthreads();
}

// the group of row r: the last e < G with off[e] <= r (-1: r lies before the first or past the last group)
__device__ __forceinline__ int group_of(const int* off, int G, int64_t r) {
  if (r < off[0] || r >= off[G]) return -1;
  int lo = 0, hi = G;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= r) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ float pow2f(int e) {   // 2^e, e in [-127, 127]
  return e > -127 ? __uint_as_float(static_cast<uint32_t>(e + 127) << 23) : 5.8774717541114375e-39f;
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b16 a;\n\tcvt.u16.u32 a, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(h) : "r"(byte & 0xFFu));
  return __half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xFFFFu)));
}
// nearest e4m3 byte of a non-negative a, saturating at 448
__device__ __forceinline__ uint32_t e4m3_byte(float a) {
  uint32_t d;
  asm("{\n\t.reg .b16 h;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %2, %1;\n\tcvt.u32.u16 %0, h;\n\t}" : "=r"(d) : "f"(a), "f"(0.f));
  return d & 0xFFu;
}
// scale byte -> value (0xFF mxfp4 and 0x7F nvfp4 are NaN)
template <int FMT>
__device__ __forceinline__ float scale_value(uint32_t b) {
  if (FMT == LB_FMT_MXFP4) return b == 255u ? __uint_as_float(0x7FFFFFFFu) : pow2f(static_cast<int>(b) - 127);
  return e4m3_value(b);
}
// eight values to eight codes (nearest, ties to the even code, saturating at 6; value 0 in the low nibble)
__device__ __forceinline__ uint32_t e2m1_codes(const float* v) {
  uint32_t d;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(d)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return d;
}

}  // namespace mx
}  // namespace lb
