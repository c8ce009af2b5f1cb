// Microscaled 4-bit floating point: quantise rows, dequantise, lay scales out.
//
//   mxfp4   E = clamp(floor(log2 max|x|) - 2, -127, 127) per 32 values, code = e2m1(x / 2^E)
//   nvfp4   x' = x / t;  s = e4m3(max|x'| / 6) per 16 values, code = e2m1(x' / s)      (t: the tensor's scale)
//
// e2m1 rounds to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to the even code, and saturates.  Every decision is the
// exact one: x / 2^E is exact, and the float32 quotients amax / 6 and x' / s never round onto a tie they are not on,
// since the divisors have at most 4 significant bits below 2 and the ties at most 5 (the nearest other quotient is more
// than half an ulp away).  A block with a NaN or an infinity gets a NaN scale, so it stands for NaNs: nothing
// is replaced in silence.  A zero block has scale byte 0.
#include "lb_mx.cuh"
#include "lb_kernels.h"

namespace lb {
namespace mx {

template <int DT>
struct In {};
template <>
struct In<LB_DT_F32> {
  static constexpr int SIZE = 4;
  static __device__ __forceinline__ float one(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
};
template <>
struct In<LB_DT_BF16> {
  static constexpr int SIZE = 2;
  static __device__ __forceinline__ float one(const void* p, int64_t i) {
    return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]) << 16);
  }
};
template <>
struct In<LB_DT_F16> {
  static constexpr int SIZE = 2;
  static __device__ __forceinline__ float one(const void* p, int64_t i) { return __half2float(static_cast<const __half*>(p)[i]); }
};

// 16 values of a row from column c0 (zeros past K); vec: rows are aligned to 32 bytes (2), 16 (1) or their elements (0)
template <int DT>
__device__ __forceinline__ void load16(const void* row, int64_t c0, int64_t K, int vec, float (&v)[16]) {
  if (vec && c0 + 16 <= K) {
    const char* p = static_cast<const char*>(row) + c0 * In<DT>::SIZE;
    uint32_t w[DT == LB_DT_F32 ? 16 : 8];
#pragma unroll
    for (int i = 0; i < In<DT>::SIZE / 2; ++i) {
      if (vec == 2) {
        ldg_nc_v8(p + 32 * i, *reinterpret_cast<uint32_t(*)[8]>(&w[8 * i]));
      } else {
        const uint4 a = ldg_nc_v4(p + 32 * i), b = ldg_nc_v4(p + 32 * i + 16);
        w[8 * i] = a.x; w[8 * i + 1] = a.y; w[8 * i + 2] = a.z; w[8 * i + 3] = a.w;
        w[8 * i + 4] = b.x; w[8 * i + 5] = b.y; w[8 * i + 6] = b.z; w[8 * i + 7] = b.w;
      }
    }
    if constexpr (DT == LB_DT_F32) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (DT == LB_DT_BF16) {
          v[2 * i] = __uint_as_float(w[i] << 16);
          v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = c0 + i < K ? In<DT>::one(row, c0 + i) : 0.f;
  }
}

// Codes of y / s without 16 divisions.  y of a 16-bit type scaled by a power of two has at most 11 significant bits and
// s 4, so a quotient that is no tie is at least 2^-11 away from every tie, relatively: y times the rounded inverse is
// within 2^-22 of it, and rounding that to 16 significant bits puts every tie back on its place and moves nothing across one.
__device__ __forceinline__ void codes_short(const float (&y)[16], float rs, uint32_t& lo, uint32_t& hi) {
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float((__float_as_uint(y[i] * rs) + 0x80u) & 0xFFFFFF00u);
  lo = e2m1_codes(v);
  hi = e2m1_codes(v + 8);
}
// For any y: the codes of slightly more and slightly less than y / s (2^-20 either way, past the rounding of the inverse and
// the product).  The quotient's code lies between; where the two differ (about one group of eight in 10^5 of random values)
// the eight quotients are divided out.
__device__ __forceinline__ uint32_t codes8_any(const float* y, float s, float rs) {
  float up[8], dn[8];
  const float ru = rs * (1.f + 0x1p-20f), rd = rs * (1.f - 0x1p-20f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    up[i] = y[i] * ru;
    dn[i] = y[i] * rd;
  }
  const uint32_t a = e2m1_codes(up);
  if (a == e2m1_codes(dn)) return a;
#pragma unroll
  for (int i = 0; i < 8; ++i) up[i] = __fdiv_rn(y[i], s);
  return e2m1_codes(up);
}

struct QuantParams {
  const void* x;            // [Rin, K], row stride ldx
  int64_t Rin, R, K, ldx;   // R rows out: row r is x[rows[r]], or x[r]
  const int* rows;
  Groups g;
  const float* t;           // nvfp4: the tensor's scale
  const float* part;        // nvfp4, scale to be found: partial maxima of |x|, `nparts` of them
  float* t_out;             //   and where it is written
  int nparts;
  uint8_t* codes;
  uint8_t* scales;
  int vec;
};

// The smallest power of two t with amax / t <= 448 * 6 = 1.3125 * 2^11 (1 for a zero tensor), so that dividing
// by it is exact.
__device__ __forceinline__ float auto_scale(float amax) {
  if (!(amax > 0.f)) return 1.f;
  int e;
  const float f = frexpf(amax, &e);           // amax = f 2^e, f in [0.5, 1)
  e -= f <= 0.65625f ? 12 : 11;
  return pow2f(e < -126 ? -126 : e);
}

// Where row r lies: its place in its group and the group's first row block (false: it is in no group).
__device__ __forceinline__ bool place_of(const Groups& g, const int* off, const int* base, int64_t gblocks, int64_t r,
                                         int64_t& rg, int64_t& blk0) {
  rg = r;
  blk0 = 0;
  if (g.G == 0) return true;
  int64_t e;
  if (g.per > 0) {
    e = static_cast<uint32_t>(r) / static_cast<uint32_t>(g.per);
    rg = r - e * g.per;
    blk0 = e * gblocks;
  } else {
    e = group_of(off, g.G, r);
    if (e < 0) return false;
    rg = r - off[e];
    blk0 = base[e];
  }
  return true;
}

// One thread per 16 values, a warp per 512 values of one row.  Memory-bound: 32-byte loads, whole sectors; the next row's
// index is on its way while this row is rounded.
template <int FMT, int DT>
__global__ void __launch_bounds__(256) quant_kernel(const QuantParams p) {
  extern __shared__ int sm[];
  pdl_launch_dependents();
  pdl_wait();
  int* off = sm;
  int* base = sm + p.g.G + 1;
  __shared__ float s_t;
  const int lane = threadIdx.x & 31;
  if (p.g.G > 0 && p.g.per == 0) load_groups(p.g, p.R, off, base);
  if (FMT == LB_FMT_NVFP4) {
    if (p.part) {
      if (threadIdx.x < 32) {
        float m = 0.f;
        for (int i = lane; i < p.nparts; i += 32) m = fmaxf(m, p.part[i]);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane == 0) {
          s_t = auto_scale(m);
          if (blockIdx.x == 0) *p.t_out = s_t;
        }
      }
    } else if (threadIdx.x == 0) {
      s_t = *p.t;
    }
    __syncthreads();
  }
  const float t = FMT == LB_FMT_NVFP4 ? s_t : 1.f;
  // dividing by a power of two is multiplying by its inverse, exactly
  const bool pow2 = FMT == LB_FMT_NVFP4 && (__float_as_uint(t) & 0x807FFFFFu) == 0 && t >= pow2f(-126) && t <= pow2f(126);
  const float inv = 1.0f / t;
  const int64_t rb = row_bytes(p.K), acols = atom_cols(FMT, p.K);
  const uint32_t segs = static_cast<uint32_t>((p.K + 511) / 512);
  const int64_t nseg = p.R * segs, step = static_cast<int64_t>(gridDim.x) * 8;
  const int64_t gblocks = p.g.per > 0 ? (p.g.per + 127) / 128 : 0;
  auto split = [&](int64_t w, int64_t& r, int64_t& c) {          // warp item -> row, first column
    r = nseg <= 0xFFFFFFFFll ? static_cast<uint32_t>(w) / segs : w / segs;
    c = (w - r * segs) * 512;
  };
  int64_t w = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5), r, c0;
  split(w < nseg ? w : 0, r, c0);
  int64_t src = p.rows && w < nseg ? p.rows[r] : r;
  while (w < nseg) {
    const int64_t wn = w + step;
    int64_t rn, cn;
    split(wn < nseg ? wn : 0, rn, cn);
    c0 += lane * 16;
    float v[16];
    if (src >= 0 && src < p.Rin) {
      load16<DT>(static_cast<const char*>(p.x) + src * p.ldx * In<DT>::SIZE, c0, p.K, p.vec, v);
    } else {                                                     // no such row: zeros, and the error word says so
      if (lane == 0) atomicOr(&g_dev_errors, LB_DEVERR_BAD_INDEX);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
    }
    const int64_t srcn = p.rows && wn < nseg ? p.rows[rn] : rn;
    int64_t rg, blk0;
    const bool in = place_of(p.g, off, base, gblocks, r, rg, blk0);   // rows of no group are left alone
    uint32_t am = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
      am = b > am ? b : am;
    }
    uint32_t byte, lo, hi;
    if (FMT == LB_FMT_MXFP4) {
      const uint32_t o = __shfl_xor_sync(0xffffffffu, am, 1);
      am = o > am ? o : am;
      const uint32_t f = am >> 23;             // exponent field: floor(log2) + 127, 255 for inf / NaN
      byte = f == 255u ? 255u : (f > 2u ? f - 2u : 0u);
      const float mul = byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] *= mul;
      lo = e2m1_codes(v);
      hi = e2m1_codes(v + 8);
    } else {
      const bool bad = am >= 0x7F800000u;
      float a = __uint_as_float(am);
      a = pow2 ? a * inv : __fdiv_rn(a, t);
      byte = bad ? 0x7Fu : e4m3_byte(__fdiv_rn(a, 6.0f));
      const float s = e4m3_value(byte), rs = byte == 0u || bad ? 0.f : 1.0f / s;   // no scale: zeros with their signs
      if (pow2) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] *= inv;
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __fdiv_rn(v[i], t);
      }
      if (DT != LB_DT_F32 && pow2) {
        codes_short(v, rs, lo, hi);
      } else {
        lo = codes8_any(v, s, rs);
        hi = codes8_any(v + 8, s, rs);
      }
    }
    if (in && c0 < rb * 2) *reinterpret_cast<uint2*>(p.codes + r * rb + c0 / 2) = make_uint2(lo, hi);
    // four scale bytes of neighbouring blocks make one word
    constexpr int PER = FMT == LB_FMT_MXFP4 ? 2 : 1;
    uint32_t word = byte;
    word |= __shfl_down_sync(0xffffffffu, word, PER) << 8;
    word = (word & 0xFFFFu) | (__shfl_down_sync(0xffffffffu, word, 2 * PER) << 16);
    const int64_t c = c0 / block_of(FMT);
    if (in && lane % (4 * PER) == 0 && c < acols * 4)
      *reinterpret_cast<uint32_t*>(p.scales + blk0 * acols * 512 + scale_at(rg, c, acols)) = word;
    w = wn;
    r = rn;
    c0 = cn;
    src = srcn;
  }
}

// Partial maxima of |x| over finite values, one per block.
template <int DT>
__global__ void __launch_bounds__(256) amax_kernel(const void* __restrict__ x, int64_t R, int64_t K, int64_t ldx, int vec,
                                                   float* __restrict__ part) {
  __shared__ uint32_t red[8];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t segs = (K + 511) / 512, nseg = R * segs;
  uint32_t am = 0;
  for (int64_t w = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); w < nseg;
       w += static_cast<int64_t>(gridDim.x) * 8) {
    const int64_t r = w / segs;
    float v[16];
    load16<DT>(static_cast<const char*>(x) + r * ldx * In<DT>::SIZE, (w - r * segs) * 512 + lane * 16, K, vec, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
      am = b > am && b < 0x7F800000u ? b : am;
    }
  }
  am = __reduce_max_sync(0xffffffffu, am);
  if (lane == 0) red[threadIdx.x >> 5] = am;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < 8; ++i) am = red[i] > am ? red[i] : am;
    part[blockIdx.x] = __uint_as_float(am);
  }
}

struct DequantParams {
  const uint8_t* codes;
  const uint8_t* scales;
  const float* t;           // or null: 1
  int64_t R, K, ldo;
  Groups g;
  void* out;
  int vec;                  // as load16's
};

// One thread per 16 values.
template <int FMT, int ODT>
__global__ void __launch_bounds__(256) dequant_kernel_mx(const DequantParams p) {
  extern __shared__ int sm[];
  pdl_launch_dependents();
  pdl_wait();
  int* off = sm;
  int* base = sm + p.g.G + 1;
  if (p.g.G > 0 && p.g.per == 0) load_groups(p.g, p.R, off, base);
  const float t = FMT == LB_FMT_NVFP4 && p.t ? *p.t : 1.f;
  const int lane = threadIdx.x & 31;
  const int64_t rb = row_bytes(p.K), acols = atom_cols(FMT, p.K);
  const uint32_t segs = static_cast<uint32_t>((p.K + 511) / 512);
  const int64_t nseg = p.R * segs;
  const int64_t gblocks = p.g.per > 0 ? (p.g.per + 127) / 128 : 0;
  for (int64_t w = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); w < nseg;
       w += static_cast<int64_t>(gridDim.x) * 8) {
    const int64_t r = nseg <= 0xFFFFFFFFll ? static_cast<uint32_t>(w) / segs : w / segs;
    const int64_t c0 = (w - r * segs) * 512 + lane * 16;
    int64_t rg, blk0;
    if (c0 >= p.K || !place_of(p.g, off, base, gblocks, r, rg, blk0)) continue;
    const uint2 q = *reinterpret_cast<const uint2*>(p.codes + r * rb + c0 / 2);
    const float s = scale_value<FMT>(p.scales[blk0 * acols * 512 + scale_at(rg, c0 / block_of(FMT), acols)]);
    uint32_t h[8];
    {
      uint32_t a[4], b[4];
      deq_fp4_word(q.x, a);
      deq_fp4_word(q.y, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) { h[i] = a[i]; h[4 + i] = b[i]; }
    }
    float v[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
      v[2 * i] = f.x * s;                      // exact: 2 significant bits times a power of two or 4 bits
      v[2 * i + 1] = f.y * s;
    }
    if (FMT == LB_FMT_NVFP4) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] *= t;
    }
    constexpr int NW = ODT == LB_DT_F32 ? 16 : 8, ES = ODT == LB_DT_F32 ? 4 : 2;
    uint32_t u[NW];
    if constexpr (ODT == LB_DT_F32) {
#pragma unroll
      for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (ODT == LB_DT_BF16) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
          u[i] = *reinterpret_cast<const uint32_t*>(&b);
        } else {
          const __half2 b = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
          u[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
      }
    }
    char* o = static_cast<char*>(p.out) + (r * p.ldo + c0) * ES;
    if (p.vec && c0 + 16 <= p.K) {
#pragma unroll
      for (int i = 0; i < NW / 8; ++i) {
        if (p.vec == 2) {
          stg_v8(o + 32 * i, u + 8 * i);
        } else {
          reinterpret_cast<uint4*>(o)[2 * i] = make_uint4(u[8 * i], u[8 * i + 1], u[8 * i + 2], u[8 * i + 3]);
          reinterpret_cast<uint4*>(o)[2 * i + 1] = make_uint4(u[8 * i + 4], u[8 * i + 5], u[8 * i + 6], u[8 * i + 7]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (c0 + i >= p.K) continue;
        if constexpr (ODT == LB_DT_F32) reinterpret_cast<uint32_t*>(o)[i] = u[i];
        else reinterpret_cast<uint16_t*>(o)[i] = static_cast<uint16_t>(u[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
}

// Row-major scale bytes [G * N, ld] (nb blocks of each row) into atoms, or back (to_atoms == 0); padding gets zeros.
template <int FMT>
__global__ void __launch_bounds__(256) scales_kernel(uint8_t* __restrict__ plain, int64_t ld, int64_t N, int64_t K,
                                                     int64_t G, uint8_t* __restrict__ atoms, int to_atoms) {
  const int64_t acols = atom_cols(FMT, K), blocks = (N + 127) / 128, nb = (K + block_of(FMT) - 1) / block_of(FMT);
  const int64_t total = G * blocks * 128 * acols;          // words of four block columns
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t c4 = i % acols, row = i / acols;         // neighbours read neighbouring words of a row
    const int64_t e = row / (blocks * 128), r = row - e * blocks * 128;
    uint8_t* a = atoms + e * blocks * acols * 512 + scale_at(r, c4 * 4, acols);
    uint8_t* s = plain + (e * N + r) * ld + c4 * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = r < N && c4 * 4 + j < nb;
      if (to_atoms) a[j] = in ? s[j] : 0;
      else if (in) s[j] = a[j];
    }
  }
}

constexpr int MAX_PARTS = LB_MX_PARTIALS;
static int quant_blocks(int64_t R, int64_t K, int sms) {
  const int64_t nseg = R * ((K + 511) / 512), b = (nseg + 7) / 8;
  return static_cast<int>(b < static_cast<int64_t>(sms) * 8 ? b : static_cast<int64_t>(sms) * 8);
}
// 2: rows are 32-byte aligned, 1: 16, 0: neither
static int row_vec(const void* p, int64_t ld, int es) {
  return aligned(p, 32) && ld * es % 32 == 0 ? 2 : (aligned(p, 16) && ld * es % 16 == 0 ? 1 : 0);
}
// A launch that may begin while the kernel before it ends (it waits for that one before it touches memory).
template <typename P>
static cudaError_t launch_early(void (*kernel)(P), int blocks, size_t smem, cudaStream_t st, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}
static bool is_mx(int fmt) { return fmt == LB_FMT_MXFP4 || fmt == LB_FMT_NVFP4; }
static int dt_size(int dt) { return dt == LB_DT_F32 ? 4 : 2; }

// the checks of a tensor's groups; 0 or a status
static int check_groups(const char* who, const int* offsets, int64_t G, int64_t per, int64_t R) {
  if (G < 0 || G > LB_MX_MAX_GROUPS) return fail(LB_E_ARG, "%s: G must be in [0, %d]", who, LB_MX_MAX_GROUPS);
  if (per < 0 || (per > 0 && (G == 0 || per * G != R))) return fail(LB_E_ARG, "%s: G groups of `per` rows must make R", who);
  if (G > 0 && per == 0 && !offsets) return fail(LB_E_ARG, "%s: ragged groups need offsets", who);
  if (G > 0 && per == 0 && !aligned(offsets, 4)) return fail(LB_E_ALIGN, "%s: offsets must be 4-byte aligned", who);
  return LB_OK;
}

}  // namespace mx
}  // namespace lb

using namespace lb;

extern "C" {

int64_t lb_mx_row_bytes(int64_t K) { return K <= 0 ? -1 : mx::row_bytes(K); }

int64_t lb_mx_scale_bytes(int fmt, int64_t R, int64_t K, int64_t G, int64_t per) {
  if (!mx::is_mx(fmt) || R < 0 || K <= 0 || G < 0 || per < 0) return -1;
  int64_t blocks;
  if (G == 0) blocks = (R + 127) / 128;
  else if (per > 0) blocks = G * ((per + 127) / 128);
  else blocks = R / 128 + (G < R ? G : R);
  return blocks * mx::atom_cols(fmt, K) * 512;
}

int lb_mx_quant(int fmt, const void* x, int x_dtype, int64_t Rin, int64_t K, int64_t ldx, const int* rows, int64_t R,
                const int* offsets, int64_t G, int64_t per, const float* tensor_scale, float* auto_scale, uint8_t* codes,
                uint8_t* scales, void* stream) {
  if (!mx::is_mx(fmt)) return fail(LB_E_ARG, "lb_mx_quant: format %d is not microscaled", fmt);
  if (x_dtype != LB_DT_F32 && x_dtype != LB_DT_BF16 && x_dtype != LB_DT_F16)
    return fail(LB_E_ARG, "lb_mx_quant: x_dtype must be LB_DT_F32, LB_DT_BF16 or LB_DT_F16");
  if (Rin < 0 || R < 0 || K <= 0 || ldx < K) return fail(LB_E_ARG, "lb_mx_quant: bad sizes (K positive, ldx >= K)");
  if (Rin > 0x7FFFFFFF || R > 0x7FFFFFFF) return fail(LB_E_ARG, "lb_mx_quant: at most 2^31 - 1 rows");
  if (!rows && R != Rin) return fail(LB_E_ARG, "lb_mx_quant: R must be the rows of x when none are chosen");
  int r = mx::check_groups("lb_mx_quant", offsets, G, per, R);
  if (r) return r;
  if (fmt == LB_FMT_NVFP4 && !tensor_scale && !auto_scale)
    return fail(LB_E_ARG, "lb_mx_quant: nvfp4 needs tensor_scale, or auto_scale to find it");
  if (R == 0) return LB_OK;
  if (!codes || !scales || (!x && Rin > 0)) return fail(LB_E_ARG, "lb_mx_quant: x, codes and scales are required");
  const int es = mx::dt_size(x_dtype);
  if (!aligned(x, es) || !aligned(codes, 16) || !aligned(scales, 16) || !aligned(rows, 4) || !aligned(tensor_scale, 4) ||
      !aligned(auto_scale, 4))
    return fail(LB_E_ALIGN, "lb_mx_quant: codes and scales must be 16-byte, the others element aligned");
  DevInfo* d;
  if ((r = current(&d))) return r;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  mx::QuantParams p;
  p.x = x; p.Rin = Rin; p.R = R; p.K = K; p.ldx = ldx;
  p.rows = rows;
  p.g = {offsets, static_cast<int>(G), per};
  p.t = tensor_scale;
  p.part = nullptr; p.t_out = nullptr; p.nparts = 0;
  p.codes = codes; p.scales = scales;
  p.vec = mx::row_vec(x, ldx, es);
  if (fmt == LB_FMT_NVFP4 && !tensor_scale) {
    int nb = mx::quant_blocks(Rin, K, d->sms);
    if (nb > mx::MAX_PARTS) nb = mx::MAX_PARTS;
    if (nb < 1) nb = 1;
    p.part = auto_scale + 1;
    p.t_out = auto_scale;
    p.nparts = nb;
    if (x_dtype == LB_DT_F32) mx::amax_kernel<LB_DT_F32><<<nb, 256, 0, st>>>(x, Rin, K, ldx, p.vec, auto_scale + 1);
    else if (x_dtype == LB_DT_BF16) mx::amax_kernel<LB_DT_BF16><<<nb, 256, 0, st>>>(x, Rin, K, ldx, p.vec, auto_scale + 1);
    else mx::amax_kernel<LB_DT_F16><<<nb, 256, 0, st>>>(x, Rin, K, ldx, p.vec, auto_scale + 1);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return launched(e, "mx_amax");
  }
  const int blocks = mx::quant_blocks(R, K, d->sms);
  const size_t sm = G > 0 && per == 0 ? 2 * (G + 1) * sizeof(int) : 0;
  cudaError_t e;
#define LB_MX_QUANT(F)                                                                                              \
  e = x_dtype == LB_DT_F32    ? mx::launch_early(mx::quant_kernel<F, LB_DT_F32>, blocks, sm, st, p)                 \
      : x_dtype == LB_DT_BF16 ? mx::launch_early(mx::quant_kernel<F, LB_DT_BF16>, blocks, sm, st, p)                \
                              : mx::launch_early(mx::quant_kernel<F, LB_DT_F16>, blocks, sm, st, p)
  if (fmt == LB_FMT_MXFP4) LB_MX_QUANT(LB_FMT_MXFP4);
  else LB_MX_QUANT(LB_FMT_NVFP4);
#undef LB_MX_QUANT
  return launched(e, "mx_quant");
}

int lb_mx_dequant(int fmt, const uint8_t* codes, const uint8_t* scales, const float* tensor_scale, int64_t R, int64_t K,
                  const int* offsets, int64_t G, int64_t per, void* out, int out_dtype, int64_t ldo, void* stream) {
  if (!mx::is_mx(fmt)) return fail(LB_E_ARG, "lb_mx_dequant: format %d is not microscaled", fmt);
  if (out_dtype != LB_DT_F32 && out_dtype != LB_DT_BF16 && out_dtype != LB_DT_F16)
    return fail(LB_E_ARG, "lb_mx_dequant: out_dtype must be LB_DT_F32, LB_DT_BF16 or LB_DT_F16");
  if (R < 0 || K <= 0 || ldo < K || R > 0x7FFFFFFF) return fail(LB_E_ARG, "lb_mx_dequant: bad sizes");
  int r = mx::check_groups("lb_mx_dequant", offsets, G, per, R);
  if (r) return r;
  if (R == 0) return LB_OK;
  if (!codes || !scales || !out) return fail(LB_E_ARG, "lb_mx_dequant: codes, scales and out are required");
  const int es = mx::dt_size(out_dtype);
  if (!aligned(out, es) || !aligned(codes, 16) || !aligned(scales, 16) || !aligned(tensor_scale, 4))
    return fail(LB_E_ALIGN, "lb_mx_dequant: codes and scales must be 16-byte, the others element aligned");
  DevInfo* d;
  if ((r = current(&d))) return r;
  mx::DequantParams p{codes, scales, tensor_scale, R, K, ldo, {offsets, static_cast<int>(G), per}, out,
                      mx::row_vec(out, ldo, es)};
  const int blocks = mx::quant_blocks(R, K, d->sms);
  const size_t sm = G > 0 && per == 0 ? 2 * (G + 1) * sizeof(int) : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
#define LB_MX_DEQUANT(F)                                                                                            \
  e = out_dtype == LB_DT_F32    ? mx::launch_early(mx::dequant_kernel_mx<F, LB_DT_F32>, blocks, sm, st, p)           \
      : out_dtype == LB_DT_BF16 ? mx::launch_early(mx::dequant_kernel_mx<F, LB_DT_BF16>, blocks, sm, st, p)          \
                                : mx::launch_early(mx::dequant_kernel_mx<F, LB_DT_F16>, blocks, sm, st, p)
  if (fmt == LB_FMT_MXFP4) LB_MX_DEQUANT(LB_FMT_MXFP4);
  else LB_MX_DEQUANT(LB_FMT_NVFP4);
#undef LB_MX_DEQUANT
  return launched(e, "mx_dequant");
}

int lb_mx_scales(int fmt, uint8_t* plain, int64_t ld, int64_t G, int64_t N, int64_t K, uint8_t* scales, int to_atoms,
                 void* stream) {
  if (!mx::is_mx(fmt)) return fail(LB_E_ARG, "lb_mx_scales: format %d is not microscaled", fmt);
  const int b = mx::block_of(fmt);
  if (G <= 0 || N <= 0 || K <= 0 || ld < (K + b - 1) / b)
    return fail(LB_E_ARG, "lb_mx_scales: bad sizes (ld at least the blocks of a row)");
  if (!plain || !scales) return fail(LB_E_ARG, "lb_mx_scales: plain and scales are required");
  if (!aligned(scales, 16)) return fail(LB_E_ALIGN, "lb_mx_scales: scales must be 16-byte aligned");
  DevInfo* d;
  int r = current(&d);
  if (r) return r;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t words = G * ((N + 127) / 128) * 128 * mx::atom_cols(fmt, K);
  int64_t blocks = (words + 255) / 256;
  if (blocks > static_cast<int64_t>(d->sms) * 16) blocks = static_cast<int64_t>(d->sms) * 16;
  if (fmt == LB_FMT_MXFP4)
    mx::scales_kernel<LB_FMT_MXFP4><<<static_cast<unsigned>(blocks), 256, 0, st>>>(plain, ld, N, K, G, scales, to_atoms);
  else
    mx::scales_kernel<LB_FMT_NVFP4><<<static_cast<unsigned>(blocks), 256, 0, st>>>(plain, ld, N, K, G, scales, to_atoms);
  return launched(cudaGetLastError(), "mx_scales");
}

}  // extern "C"
