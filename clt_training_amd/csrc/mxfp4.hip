// MXFP4 on gfx950: quantisation of rows to 4-bit microscaled codes, the way back, and the encoder product on the codes
// (format: include/clt_mi355.h).
#include "common.h"

namespace clt {
namespace {

constexpr int KPAD = 128;  // columns are padded to whole matrix-instruction steps: no bounds in the product's inner loop

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Eight elements from an address with no more than the element's own alignment.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Raw8 {
  T e[8];
};

// ---- quantisation ----------------------------------------------------------------------------------------------------
// HBM-bound: sizeof(x) + 17/32 bytes per value.  A lane holds 8 consecutive values, a block of 32 is a quad of lanes (its
// maximum is two DPP quad permutations).  The scale is a power of two, so x 2^-e is exact (ldexp, which keeps the smallest
// values too) and the only rounding is the hardware's conversion to e2m1 (nearest even, saturating at 6).
// this lane's 8 codes and, the same in the four lanes of a block, its scale byte
__device__ __forceinline__ uint32_t quantise_lane(const float (&x)[8], int& scale) {
  uint32_t top = 0;  // bit patterns of magnitudes are ordered like the values, with infinity and NaN on top
#pragma unroll
  for (int q = 0; q < 8; ++q) top = max(top, __float_as_uint(x[q]) & 0x7fffffffu);
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, true));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, true));
  const bool bad = top >= 0x7f800000u;
  const int s = max((int)(top >> 23) - 2, 0);  // biased exponent of e
  scale = bad ? 255 : s;
  uint32_t w = 0;
  float y[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) y[q] = bad ? 0.f : __builtin_amdgcn_ldexpf(x[q], 127 - s);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], 1.0f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], 1.0f, 3);
  return w;
}

template <typename T>
__device__ __forceinline__ void load_row8(const T* row, int64_t c, int64_t K, float (&f)[8]) {
  if (c + 8 <= K) {
    const Raw8<T> r = *reinterpret_cast<const Raw8<T>*>(row + c);
#pragma unroll
    for (int q = 0; q < 8; ++q) f[q] = (float)r.e[q];
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) f[q] = c + q < K ? (float)row[c + q] : 0.f;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void mxfp4_quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t R, int64_t K,
                                                             int64_t lanes_per_row, uint32_t* __restrict__ codes,
                                                             uint8_t* __restrict__ scales) {
  const int64_t total = R * lanes_per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / lanes_per_row, c = (i - row * lanes_per_row) * 8;
    float f[8];
    load_row8(x + row * ldx, c, K, f);
    int s;
    const uint32_t w = quantise_lane(f, s);  // (a quad of lanes is one block: lanes_per_row is a multiple of 16)
    codes[i] = w;
    if ((i & 3) == 0) scales[i >> 2] = (uint8_t)s;
  }
}

// ---- and back --------------------------------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void mxfp4_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales, int64_t R, int64_t K,
                                                               int64_t lanes_per_row, T* __restrict__ out) {
  const int64_t total = R * lanes_per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / lanes_per_row, c = (i - row * lanes_per_row) * 8;
    if (c >= K) continue;
    const uint32_t w = codes[i];
    const int s = scales[i >> 2];
    float f[8];
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y, f[4] = d.x, f[5] = d.y, f[6] = e.x, f[7] = e.y;
#pragma unroll
    for (int q = 0; q < 8; ++q) f[q] = s == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(f[q], s - 127);
    T* o = out + row * K + c;
    if (c + 8 <= K) {
      Raw8<T> r;
#pragma unroll
      for (int q = 0; q < 8; ++q) r.e[q] = (T)f[q];
      *reinterpret_cast<Raw8<T>*>(o) = r;
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (c + q < K) o[q] = (T)f[q];
    }
  }
}

// ---- product ---------------------------------------------------------------------------------------------------------
// v_mfma_scale_f32_32x32x64_f8f6f4 with 4-bit operands: lane l of an operand holds row l % 32, columns 32 (l / 32) .. + 31 of
// a step of 64 -- one block, 16 bytes of codes and one scale.  D: lane l holds column l % 32, rows 8 (i / 4) + 4 (l / 32) + i % 4.
__device__ __forceinline__ f32x16 mfma4(const i32x4& a, const i32x4& b, const f32x16& c, int sa, int sb) {
  const i32x8 A = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8 B = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, c, 4, 4, 0, sa, 0, sb);
}

struct LinearArgs {
  const uint8_t *xc, *xs, *wc, *ws;
  const void* bias;
  void* out;
  int64_t N, M, ldo;
  int kp, bias_dtype, relu;
};

// One wave per 32 latents x 32 tokens, operands straight from memory.
template <typename T>
__global__ __launch_bounds__(64) void mxfp4_linear_kernel(const LinearArgs p) {
  const int lane = threadIdx.x, r = lane & 31, h = lane >> 5;
  const int64_t m0 = (int64_t)blockIdx.x * 32, n0 = (int64_t)blockIdx.y * 32;
  const int64_t wr = min(m0 + r, p.M - 1), xr = min(n0 + r, p.N - 1);
  const uint8_t* wc = p.wc + wr * (p.kp / 2) + 16 * h;
  const uint8_t* xc = p.xc + xr * (p.kp / 2) + 16 * h;
  const uint8_t* ws = p.ws + wr * (p.kp / 32) + h;
  const uint8_t* xs = p.xs + xr * (p.kp / 32) + h;
  f32x16 acc = {};
  for (int k = 0; k < p.kp / 64; ++k)
    acc = mfma4(*(const i32x4*)(xc + 32 * k), *(const i32x4*)(wc + 32 * k), acc, xs[2 * k], ws[2 * k]);
  const int64_t m = m0 + r;
  if (m >= p.M) return;
  const float b = p.bias ? load_scalar(p.bias, p.bias_dtype, m) : 0.f;
  T* out = reinterpret_cast<T*>(p.out);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t n = n0 + 8 * (i / 4) + 4 * h + i % 4;
    float v = acc[i] + b;
    if (p.relu) v = v < 0.f ? 0.f : v;
    if (n < p.N) out[n * p.ldo + m] = (T)v;
  }
}

}  // namespace
}  // namespace clt

using namespace clt;

static int64_t padded(int64_t K) { return (K + KPAD - 1) / KPAD * KPAD; }
static unsigned blocks_for(int64_t lanes) { return (unsigned)((lanes + 255) / 256 < 16384 ? (lanes + 255) / 256 : 16384); }

extern "C" int clt_mxfp4_quantize(const void* x, int x_dtype, int64_t ldx, int64_t R, int64_t K, uint8_t* codes,
                                  uint8_t* scales, clt_stream_t stream) {
  CLT_CHECK_ARG(x && codes && scales, "clt_mxfp4_quantize: null pointer");
  CLT_CHECK_ARG(valid_dtype(x_dtype), "clt_mxfp4_quantize: dtype");
  CLT_CHECK_ARG(R > 0 && K > 0 && K < (1ll << 30) && R < (1ll << 40) / K && ldx >= 0, "clt_mxfp4_quantize: bad sizes");
  CLT_CHECK_ARG(aligned16(codes) && !((uintptr_t)scales & 3) && !((uintptr_t)x & (dtype_size(x_dtype) - 1)),
                "clt_mxfp4_quantize: misaligned pointer");
  const int64_t lpr = padded(K) / 8;
  if (x_dtype == CLT_BF16)
    hipLaunchKernelGGL(mxfp4_quantize_kernel<bf16_t>, dim3(blocks_for(R * lpr)), dim3(256), 0, (hipStream_t)stream,
                       (const bf16_t*)x, ldx, R, K, lpr, (uint32_t*)codes, scales);
  else
    hipLaunchKernelGGL(mxfp4_quantize_kernel<float>, dim3(blocks_for(R * lpr)), dim3(256), 0, (hipStream_t)stream,
                       (const float*)x, ldx, R, K, lpr, (uint32_t*)codes, scales);
  CLT_CHECK_LAUNCH("clt_mxfp4_quantize");
  return CLT_OK;
}

extern "C" int clt_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t R, int64_t K, void* out,
                                    int out_dtype, clt_stream_t stream) {
  CLT_CHECK_ARG(codes && scales && out, "clt_mxfp4_dequantize: null pointer");
  CLT_CHECK_ARG(valid_dtype(out_dtype), "clt_mxfp4_dequantize: dtype");
  CLT_CHECK_ARG(R > 0 && K > 0 && K < (1ll << 30) && R < (1ll << 40) / K, "clt_mxfp4_dequantize: bad sizes");
  CLT_CHECK_ARG(aligned16(codes) && !((uintptr_t)scales & 3) && !((uintptr_t)out & (dtype_size(out_dtype) - 1)),
                "clt_mxfp4_dequantize: misaligned pointer");
  const int64_t lpr = padded(K) / 8;
  if (out_dtype == CLT_BF16)
    hipLaunchKernelGGL(mxfp4_dequantize_kernel<bf16_t>, dim3(blocks_for(R * lpr)), dim3(256), 0, (hipStream_t)stream,
                       (const uint32_t*)codes, scales, R, K, lpr, (bf16_t*)out);
  else
    hipLaunchKernelGGL(mxfp4_dequantize_kernel<float>, dim3(blocks_for(R * lpr)), dim3(256), 0, (hipStream_t)stream,
                       (const uint32_t*)codes, scales, R, K, lpr, (float*)out);
  CLT_CHECK_LAUNCH("clt_mxfp4_dequantize");
  return CLT_OK;
}

extern "C" int clt_mxfp4_linear(const uint8_t* x_codes, const uint8_t* x_scales, const uint8_t* w_codes,
                                const uint8_t* w_scales, const void* bias, int bias_dtype, int64_t N, int64_t M, int64_t K,
                                int relu, void* out, int out_dtype, int64_t ldo, clt_stream_t stream) {
  CLT_CHECK_ARG(x_codes && x_scales && w_codes && w_scales && out, "clt_mxfp4_linear: null pointer");
  CLT_CHECK_ARG(valid_dtype(out_dtype) && (!bias || valid_dtype(bias_dtype)), "clt_mxfp4_linear: dtype");
  CLT_CHECK_ARG(N > 0 && M > 0 && K > 0 && ldo >= M, "clt_mxfp4_linear: bad sizes");
  CLT_UNSUPPORTED(N <= 32 * 65535ll && M < (1ll << 31) && K < (1ll << 24), "clt_mxfp4_linear: N <= %lld, M < 2^31, K < 2^24",
                  32 * 65535ll);
  CLT_CHECK_ARG(aligned16(x_codes) && aligned16(w_codes) && !((uintptr_t)x_scales & 3) && !((uintptr_t)w_scales & 3) &&
                    !((uintptr_t)out & (dtype_size(out_dtype) - 1)),
                "clt_mxfp4_linear: misaligned pointer");
  LinearArgs a{x_codes, x_scales, w_codes, w_scales, bias, out, N, M, ldo, (int)padded(K), bias_dtype, relu};
  const dim3 grid((unsigned)((M + 31) / 32), (unsigned)((N + 31) / 32));
  if (out_dtype == CLT_BF16)
    hipLaunchKernelGGL(mxfp4_linear_kernel<bf16_t>, grid, dim3(64), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(mxfp4_linear_kernel<float>, grid, dim3(64), 0, (hipStream_t)stream, a);
  CLT_CHECK_LAUNCH("clt_mxfp4_linear");
  return CLT_OK;
}
