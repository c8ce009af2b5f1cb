// Products of microscaled 4-bit operands:  y[m, n] = tx tw sum_b sx[m, b] sw[n, b] sum_{k in b} qx[m, k] qw[n, k]
// (+ bias[n]) (+ y[m, n]), dense or with one weight per group of rows (experts).
#include "lb_mx.cuh"
#include "lb_kernels.h"

namespace lb {
namespace mx {

struct GemmMxParams {
  const uint8_t* xc;
  const uint8_t* xs;
  const float* xt;          // or null: 1
  const uint8_t* wc;
  const uint8_t* ws;
  const float* wt;
  const uint16_t* bias;     // bf16 [G, N] or null
  uint16_t* y;
  int64_t M, N, K, ldy;
  int acc;
  Groups g;                 // of the rows of x (ragged); G == 0: dense
};

// One warp per output, lanes along K.
template <int FMT>
__global__ void __launch_bounds__(256) simple_kernel(const GemmMxParams p) {
  extern __shared__ int sm[];
  int* off = sm;
  int* base = sm + p.g.G + 1;
  if (p.g.G) load_groups(p.g, p.M, off, base);
  const int lane = threadIdx.x & 31;
  const int64_t rb = row_bytes(p.K), acols = atom_cols(FMT, p.K), wblocks = (p.N + 127) / 128;
  const float alpha = (p.xt ? *p.xt : 1.f) * (p.wt ? *p.wt : 1.f);
  for (int64_t o = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); o < p.M * p.N;
       o += static_cast<int64_t>(gridDim.x) * 8) {
    const int64_t m = o / p.N, n = o - m * p.N;
    int64_t e = 0, mg = m, xb = 0;
    if (p.g.G) {
      e = group_of(off, p.g.G, m);
      if (e < 0) continue;
      mg = m - off[e];
      xb = base[e];
    }
    const uint8_t* xr = p.xc + m * rb;
    const uint8_t* wr = p.wc + (e * p.N + n) * rb;
    const uint8_t* xsb = p.xs + xb * acols * 512;
    const uint8_t* wsb = p.ws + e * wblocks * acols * 512;
    float s = 0.f;
    for (int64_t w = lane; w < rb / 4; w += 32) {
      uint32_t a[4], b[4];
      deq_fp4_word(*reinterpret_cast<const uint32_t*>(xr + 4 * w), a);
      deq_fp4_word(*reinterpret_cast<const uint32_t*>(wr + 4 * w), b);
      float d = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&a[i]));
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&b[i]));
        d = fmaf(u.x, v.x, fmaf(u.y, v.y, d));
      }
      const int64_t c = w * 8 / block_of(FMT);
      s = fmaf(scale_value<FMT>(xsb[scale_at(mg, c, acols)]) * scale_value<FMT>(wsb[scale_at(n, c, acols)]), d, s);
    }
    s = rms_butterfly(s);
    if (lane == 0) {
      float v = s * alpha;
      if (p.bias) v += __uint_as_float(static_cast<uint32_t>(p.bias[e * p.N + n]) << 16);
      uint16_t* yp = p.y + m * p.ldy + n;
      if (p.acc) v += __uint_as_float(static_cast<uint32_t>(*yp) << 16);
      *yp = f32_to_bf16_bits_g(v);
    }
  }
}

static int launch_product(const char* who, int fmt, const GemmMxParams& p, cudaStream_t st) {
  if (!is_mx(fmt)) return fail(LB_E_ARG, "%s: format %d is not microscaled", who, fmt);
  if (p.M < 0 || p.N <= 0 || p.K <= 0 || p.ldy < p.N) return fail(LB_E_ARG, "%s: bad sizes (ldy >= N)", who);
  if (p.M > 0x7FFFFFFF || p.N > 0x7FFFFF00 || p.K > 0x7FFFFF00) return fail(LB_E_ARG, "%s: M, N and K must be below 2^31", who);
  if (p.M == 0) return LB_OK;
  if (!p.xc || !p.xs || !p.wc || !p.ws || !p.y) return fail(LB_E_ARG, "%s: codes, scales and y are required", who);
  if (!aligned(p.xc, 16) || !aligned(p.xs, 16) || !aligned(p.wc, 16) || !aligned(p.ws, 16))
    return fail(LB_E_ALIGN, "%s: codes and scales must be 16-byte aligned", who);
  if (!aligned(p.y, 2) || !aligned(p.bias, 2) || !aligned(p.xt, 4) || !aligned(p.wt, 4))
    return fail(LB_E_ALIGN, "%s: y, bias and the tensor scales must be element aligned", who);
  DevInfo* d;
  int r = current(&d);
  if (r) return r;
  const int64_t nb = (p.M * p.N + 7) / 8;
  const unsigned blocks = static_cast<unsigned>(nb < d->sms * 8 ? nb : d->sms * 8);
  const size_t sm = p.g.G ? 2 * (p.g.G + 1) * sizeof(int) : 0;
  if (fmt == LB_FMT_MXFP4) simple_kernel<LB_FMT_MXFP4><<<blocks, 256, sm, st>>>(p);
  else simple_kernel<LB_FMT_NVFP4><<<blocks, 256, sm, st>>>(p);
  return launched(cudaGetLastError(), who);
}

}  // namespace mx
}  // namespace lb

using namespace lb;

extern "C" {

int lb_mx_linear(int fmt, const uint8_t* x_codes, const uint8_t* x_scales, const float* x_tscale, int64_t M, int64_t K,
                 const uint8_t* w_codes, const uint8_t* w_scales, const float* w_tscale, int64_t N, const void* bias,
                 int accumulate, void* y, int64_t ldy, void* stream) {
  mx::GemmMxParams p{x_codes, x_scales, x_tscale, w_codes, w_scales, w_tscale, static_cast<const uint16_t*>(bias),
                     static_cast<uint16_t*>(y), M, N, K, ldy, accumulate ? 1 : 0, {nullptr, 0, 0}};
  return mx::launch_product("lb_mx_linear", fmt, p, static_cast<cudaStream_t>(stream));
}

int lb_mx_linear_grouped(int fmt, const uint8_t* x_codes, const uint8_t* x_scales, const float* x_tscale, int64_t M,
                         int64_t K, const int* offsets, int64_t G, const uint8_t* w_codes, const uint8_t* w_scales,
                         const float* w_tscale, int64_t N, const void* bias, int accumulate, void* y, int64_t ldy,
                         void* stream) {
  if (G <= 0) return fail(LB_E_ARG, "lb_mx_linear_grouped: G must be positive");
  int r = mx::check_groups("lb_mx_linear_grouped", offsets, G, 0, M);
  if (r) return r;
  mx::GemmMxParams p{x_codes, x_scales, x_tscale, w_codes, w_scales, w_tscale, static_cast<const uint16_t*>(bias),
                     static_cast<uint16_t*>(y), M, N, K, ldy, accumulate ? 1 : 0, {offsets, static_cast<int>(G), 0}};
  return mx::launch_product("lb_mx_linear_grouped", fmt, p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
