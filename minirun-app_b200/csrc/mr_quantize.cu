// mr_quantize.cu — bf16 / f16 / fp32 rows to MXFP4, plain and of
// silu(gate) * up.
//
// Per block of 32 elements (OCP MX): e = floor(log2 max|x|) - 2 (the largest
// e2m1 number is 1.5 * 2^2), clamped to the e8m0 range, and every element
// x * 2^-e rounded to the nearest e2m1 number, ties to the even code,
// saturating at 6. 2^-e is a power of two, so the product is exact and the
// codes are the same whatever computes them. A block with an infinity or a
// NaN has no MXFP4 number: its exponent is 255 (NaN) and its codes are 0, so
// the block reads back as NaN. Blocks of zeros have exponent 0.
//
// Bound by HBM: element bytes in, 17/32 byte an element out (and the values).
// Four lanes share a block: 8 elements each make one 16-byte load (bf16) and
// one 4-byte word of codes, both coalesced over the warp.
#include "mr_host.h"

#include <algorithm>

namespace mr {
namespace {

struct QuantParams {
  const char* x;
  int64_t stride;   // bytes between rows
  uint32_t opr;     // octets of elements a row of the output
  int64_t n;        // octets in all
  uint32_t* packed; // [n]
  uint8_t* scales;  // [n / 4]
  void* values;     // x's type, contiguous, or NULL
  float limit;      // SwiGLU clamp, 0: none
};

constexpr int kQThreads = 256;

template <int DT>
struct Raw {
  static constexpr int kWords = DT == MR_DTYPE_F32 ? 8 : 4;  // 8 elements
  uint32_t w[kWords];
};

// 8 elements at `p`; ALIGNED: 16-byte aligned.
template <int DT, bool ALIGNED>
MR_DEVICE Raw<DT> load8(const char* p) {
  Raw<DT> r;
  if constexpr (ALIGNED) {
#pragma unroll
    for (int i = 0; i < Raw<DT>::kWords / 4; ++i) {
      const uint4 v = ldg_stream_u128(reinterpret_cast<const uint32_t*>(p) + 4 * i);
      memcpy(r.w + 4 * i, &v, 16);
    }
  } else if constexpr (DT == MR_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned short* h = reinterpret_cast<const unsigned short*>(p) + 2 * i;
      r.w[i] = (uint32_t)__ldg(h) | ((uint32_t)__ldg(h + 1) << 16);
    }
  }
  return r;
}

template <int DT>
MR_DEVICE void to_float(const Raw<DT>& r, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (DT == MR_DTYPE_F32) {
      f[i] = __uint_as_float(r.w[i]);
    } else {
      const uint32_t h = (i & 1) ? r.w[i / 2] >> 16 : r.w[i / 2] & 0xFFFFu;
      f[i] = DT == MR_DTYPE_BF16 ? bf16_bits_to_f32(h) : __half2float(__ushort_as_half((unsigned short)h));
    }
  }
}

template <int DT>
MR_DEVICE void store8(void* base, int64_t o, const float (&f)[8]) {
  if constexpr (DT == MR_DTYPE_F32) {
    float4* d = reinterpret_cast<float4*>(base) + 2 * o;
    d[0] = make_float4(f[0], f[1], f[2], f[3]);
    d[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = DT == MR_DTYPE_BF16 ? f32_to_bf16_bits(f[2 * i])
                                              : __half_as_ushort(__float2half_rn(f[2 * i]));
      const uint32_t hi = DT == MR_DTYPE_BF16 ? f32_to_bf16_bits(f[2 * i + 1])
                                              : __half_as_ushort(__float2half_rn(f[2 * i + 1]));
      w[i] = lo | (hi << 16);
    }
    reinterpret_cast<uint4*>(base)[o] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Eight fp32 numbers to e2m1, element 0 in the low nibble; round to nearest
// even, saturating.
MR_DEVICE uint32_t e2m1x8(const float (&f)[8]) {
  uint32_t w;
  asm("{ .reg .b8 b0, b1, b2, b3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      "mov.b32 %0, {b0, b1, b2, b3}; }"
      : "=r"(w)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return w;
}

// One octet of a block held by lanes 4i .. 4i+3 (all four call together).
template <int DT>
MR_DEVICE void quantize8(const QuantParams& p, int64_t o, const float (&f)[8]) {
  uint32_t most = 0;  // of the magnitudes' bits: orders like the numbers, NaN above all
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(f[i]) & 0x7FFFFFFFu);
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
  const uint32_t ex = most >> 23;
  const bool finite = ex != 255;
  const uint32_t e = ex > 2 ? ex - 2 : 0;  // floor(log2) - 2 + 127, at least 0
  const float down = __uint_as_float((254u - e) << 23);
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = f[i] * down;
  const uint32_t code = finite ? e2m1x8(s) : 0u;
  if (o < p.n) {
    p.packed[o] = code;
    if ((o & 3) == 0) p.scales[o >> 2] = finite ? (uint8_t)e : (uint8_t)255;
    if (p.values) {
      const float up = e8m0_to_f32(finite ? e : 255u);
      uint32_t h[4];
      e2m1x8_to_f16x2(code, h);
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = __half2float(__ushort_as_half((unsigned short)((i & 1) ? h[i / 2] >> 16 : h[i / 2] & 0xFFFFu))) * up;
      store8<DT>(p.values, o, v);
    }
  }
}

// silu(gate) * up for any gate. Far below zero 1 + exp(-gate) overflows and
// 1 + exp(gate) is 1: gate * exp(gate / 2) * up * exp(gate / 2), of which no step
// leaves fp32's range before the result does. CUDA's expf is within 2 ulp. (A
// call: in line it took eight registers of the whole kernel, 18.1 us for 17.2.)
__device__ __noinline__ float silu_times(float gate, float up) {
  if (gate < -80.f) {
    const float e = expf(0.5f * gate);
    return gate * e * up * e;
  }
  return gate / (1.f + expf(-gate)) * up;
}
// f = silu(f) * g of eight. For gates of 80 units at most exp(-f) is 2^t with t =
// -f log2(e) rounded, times 1 + r for what the rounding left, r = -f - t ln(2) (a
// residual as in Cody and Waite's reductions). ex2.approx is within 2 ulp,
// rcp.approx within 1 and the rounded ln(2) costs 2 at f = -80, so all of it is
// within 7 ulp, 2^-20. (2^t alone loses an ulp for every unit of f.)
MR_DEVICE void silu8(float (&f)[8], const float (&g)[8]) {
  float most = fabsf(f[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) most = fmaxf(most, fabsf(f[i]));
  if (most > 80.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = silu_times(f[i], g[i]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = f[i] * -1.44269504088896341f;
    const float r = fmaf(t, -0.693147180559945309f, -f[i]);
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    float q;  // 1 + exp(-f) is between 1 and 2^116: no step of this is subnormal
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.f + fmaf(e, r, e)));
    f[i] = f[i] * q * g[i];
  }
}

// Four lanes a block of 32: one 16-byte load (two of fp32) and one word of codes
// a lane, the block's maximum by two shuffles. U octets a thread, a CTA apart,
// all loads first. Bound by HBM: fp32 16384 x 7168 with the values back 150 us
// (the copy rate); bf16 8192 x 2048 with SwiGLU 16 us (floor 12); bf16 64 x 7168
// 1.9 us, a launch.
template <int DT, bool ALIGNED, bool SWIGLU, int U>
__global__ void __launch_bounds__(kQThreads) quantize_kernel(const QuantParams p) {
  constexpr int kOct = DT == MR_DTYPE_F32 ? 32 : 16;  // bytes of an octet
  pdl_wait_and_release();
  const int64_t o0 = (int64_t)blockIdx.x * (kQThreads * U) + threadIdx.x;
  Raw<DT> a[U], b[SWIGLU ? U : 1];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t o = min(o0 + u * kQThreads, p.n - 1);
    const uint32_t row = (uint32_t)o / p.opr, c = (uint32_t)o - row * p.opr;
    const char* src = p.x + row * p.stride + (int64_t)c * kOct;
    a[u] = load8<DT, ALIGNED>(src);
    if constexpr (SWIGLU) b[u] = load8<DT, ALIGNED>(src + (int64_t)p.opr * kOct);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float f[8];
    to_float<DT>(a[u], f);
    if constexpr (SWIGLU) {
      float g[8];
      to_float<DT>(b[u], g);
      if (p.limit > 0.f) {
        // comparisons, not fmin/fmax: a NaN stays one
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (f[i] > p.limit) f[i] = p.limit;
          if (g[i] > p.limit) g[i] = p.limit;
          if (g[i] < -p.limit) g[i] = -p.limit;
        }
      }
      silu8(f, g);
    }
    quantize8<DT>(p, o0 + u * kQThreads, f);
  }
}

template <int DT, bool ALIGNED, bool SWIGLU>
cudaError_t launch_u(const mr_ctx* ctx, const QuantParams& p, cudaStream_t s) {
  constexpr int kU = 4;
  // four octets a thread once that still gives every SM eight CTAs
  const int64_t ctas = (p.n + kQThreads - 1) / kQThreads;
  if (ctas >= (int64_t)kU * 8 * ctx->sm_count)
    return launch_pdl(quantize_kernel<DT, ALIGNED, SWIGLU, kU>,
                      dim3((unsigned)((ctas + kU - 1) / kU)), kQThreads, 0, s, p);
  return launch_pdl(quantize_kernel<DT, ALIGNED, SWIGLU, 1>, dim3((unsigned)ctas), kQThreads, 0, s,
                    p);
}
template <int DT>
cudaError_t launch_q(const mr_ctx* ctx, const QuantParams& p, bool aligned, bool swiglu,
                     cudaStream_t s) {
  if (aligned)
    return swiglu ? launch_u<DT, true, true>(ctx, p, s) : launch_u<DT, true, false>(ctx, p, s);
  return swiglu ? launch_u<DT, false, true>(ctx, p, s) : launch_u<DT, false, false>(ctx, p, s);
}

mr_status quantize(mr_ctx* ctx, const void* x, mr_dtype dt, int64_t rows, int64_t width,
                   int64_t stride, bool swiglu, float limit, uint32_t* packed, uint8_t* scales,
                   void* values, void* stream) {
  if (!ctx) return MR_ERR_INVALID_ARGUMENT;
  if (dt != MR_DTYPE_BF16 && dt != MR_DTYPE_F16 && dt != MR_DTYPE_F32)
    return fail(ctx, MR_ERR_INVALID_ARGUMENT, "x must be bf16, f16 or f32");
  if (rows < 0 || width <= 0)
    return fail(ctx, MR_ERR_INVALID_ARGUMENT,
                "x must be [rows, inFeatures] with rows >= 0 and inFeatures > 0");
  if (width % 32 != 0)
    return fail(ctx, MR_ERR_INVALID_ARGUMENT,
                "inFeatures " + std::to_string(width) +
                    " is not a multiple of groupSize 32; partial final groups are not supported");
  if (width > INT32_MAX || stride < (swiglu ? 2 * width : width))
    return fail(ctx, MR_ERR_INVALID_ARGUMENT, "row stride is smaller than the row");
  if (!(limit >= 0.f))
    return fail(ctx, MR_ERR_INVALID_ARGUMENT, "SwiGLU limit must be >= 0 (0: off)");
  if (rows == 0) return MR_OK;
  if (!x || !packed || !scales)
    return fail(ctx, MR_ERR_INVALID_ARGUMENT, "x, packed and scales must be non-NULL");
  const int es = dt == MR_DTYPE_F32 ? 4 : 2;
  if (addr(x) % es || addr(packed) % 4 || addr(values) % 16)
    return fail(ctx, MR_ERR_INVALID_ARGUMENT,
                "x and packed must be aligned to their types and values to 16 bytes");
  if (rows > UINT32_MAX / (width / 8))
    return fail(ctx, MR_ERR_UNSUPPORTED, "more than 2^35 elements in one call");
  QuantParams p{static_cast<const char*>(x), stride * es, (uint32_t)(width / 8),
                rows * (width / 8), packed, scales, values, limit};
  const bool aligned = addr(x) % 16 == 0 && (p.stride % 16 == 0 || rows == 1);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const DeviceScope on(ctx);
  cudaError_t e = on.err;
  if (e == cudaSuccess)
    e = dt == MR_DTYPE_BF16  ? launch_q<MR_DTYPE_BF16>(ctx, p, aligned, swiglu, s)
        : dt == MR_DTYPE_F16 ? launch_q<MR_DTYPE_F16>(ctx, p, aligned, swiglu, s)
                             : launch_q<MR_DTYPE_F32>(ctx, p, aligned, swiglu, s);
  return cuda_check(ctx, e, "MXFP4 quantisation");
}

}  // namespace
}  // namespace mr

extern "C" {

mr_status mr_mxfp4_quantize(mr_ctx* ctx, const void* x, mr_dtype dtype, int64_t rows,
                            int64_t in_features, int64_t x_stride, uint32_t* packed,
                            uint8_t* scales, void* values, void* stream) {
  return mr::guarded([&] {
    return mr::quantize(ctx, x, dtype, rows, in_features, x_stride, false, 0.f, packed, scales,
                        values, stream);
  });
}

mr_status mr_mxfp4_quantize_swiglu(mr_ctx* ctx, const void* gate_up, mr_dtype dtype, int64_t rows,
                                   int64_t inter, int64_t stride, float swiglu_limit,
                                   uint32_t* packed, uint8_t* scales, void* stream) {
  return mr::guarded([&] {
    return mr::quantize(ctx, gate_up, dtype, rows, inter, stride, true, swiglu_limit, packed,
                        scales, nullptr, stream);
  });
}

}  // extern "C"
