// Multi-tensor AdamW for gfx950 with moments of their own width: fp32, or 8 bits with one power of two for 128 elements.
//
//   m <- m + (1 - b1) (g - m)          v <- b2 v + (1 - b2) g^2
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// HBM-bound: per element 2 sizeof(p) + sizeof(g) bytes of parameter and gradient plus 16 (fp32 moments) or 4 + 4/128 (8-bit
// moments).  Measured on four 98304 x 768 bf16 tables with bf16 gradients: 1.22 ms, 5.46 TB/s (fp32 moments), 0.53 ms, 5.74 TB/s
// (8-bit moments); a large copy reaches 4.9 TB/s here.  The 8-bit path is near the vector units' limit, too: with the
// stochastic rounding written out in integer arithmetic instead of the hardware's conversion it took 0.61 ms.  One launch takes
// up to MAX_TENSORS tensors, whose records travel in the kernel's arguments: no table in device memory, so nothing is uploaded,
// kept between calls or shared by two streams.  A workgroup owns one chunk of one tensor.
//
// 8-bit moments.  m and r = sqrt(v) are e4m3 (v itself spans twice the binades: a factor 2^17.8 between the largest and
// the smallest gradient of a block is what r holds), scaled by 2^E for 128 consecutive elements: 16 lanes of 8 elements,
// so that the block's maximum is four DPP steps inside a row of 16 lanes.  E is the least integer with max 2^-E <= 448.
// Rounding is stochastic: with b2 = 0.999 r changes by 0.05 % a step and half a step of e4m3 is 3 to 6 %, so rounding to
// nearest would freeze it.  The 16 random bits per value are a hash of (seed, tensor, step, element): the same call gives
// the same bits.  r > 0 is never rounded to 0 (the update m / r would jump to m / eps); v is formed in fp32, so r is 0 where v is
// below 2^-150.  A NaN or infinite value is stored as NaN and does not count for its block's scale.
#include <math.h>

#include "common.h"

namespace clt {
namespace {

constexpr int MAX_TENSORS = 40;   // records in one launch's arguments (40 x 88 bytes: the argument segment holds 4 KiB)
constexpr int VEC = 8;            // elements per lane and pass
// Elements per workgroup: one pass.  (Two passes: +3 % with fp32 and +6 % with 8-bit moments, four: +4 and +11 %, 302 M elements.)
constexpr int CHUNK = 256 * VEC;
constexpr int BLOCK8 = 128;       // elements per scale
constexpr int64_t MAX_CHUNKS = (1 << 24) - 1;  // workgroups of a launch (its threads are counted in 32 bits)

struct Rec {
  char* p;
  const char* g;
  char* m;
  char* v;
  uint8_t* ms;  // null: fp32 moments
  uint8_t* vs;
  int64_t numel;
  float decay;      // 1 - lr wd
  float step_size;  // lr / (1 - b1^t)
  uint32_t key;     // hash of (seed, tensor, step)
  uint32_t chunk0;  // first workgroup
  int32_t p_dtype, g_dtype;
};

struct Args {
  Rec rec[MAX_TENSORS];
  int n;
  float c1, b2, c2, inv_sqrt_bc2, eps;  // 1 - b1, b2, 1 - b2
};
static_assert(sizeof(Args) <= 4096, "kernel arguments");

// Two rounds of xor-shift and multiply, a permutation of 32 bits; shifts and factors are a set of low bias that the public
// "hash prospector" search for such mixers lists.
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x21F0AAADu;
  x = (x ^ (x >> 15)) * 0x735A2D97u;
  return x ^ (x >> 15);
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Eight elements from an address with no more than the element's own alignment (gfx950 takes dword loads at any byte), each
// read and written once.  TB/s with fp32 moments and with 8-bit moments of four 98304 x 768 bf16 tables, and with 8-bit moments of
// three 4099 x 769 fp32 tables:
//   stores non-temporal, loads plain (this): 5.46, 5.74, 5.3    both non-temporal: 5.29, 5.96, 4.9
//   loads non-temporal, stores plain:        5.21, 5.45, 4.9    both plain:        5.49, 5.61, 5.4
template <typename T>
struct Vec8;
template <>
struct Vec8<float> {
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
  static constexpr int N = 2;
};
template <>
struct Vec8<bf16_t> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2)));
  static constexpr int N = 1;
};
template <>
struct Vec8<uint8_t> {
  typedef uint32_t type __attribute__((ext_vector_type(2), aligned(1)));
  static constexpr int N = 1;
};
template <typename T>
struct Raw8 {
  T e[8];
};
template <typename T>
__device__ __forceinline__ Raw8<T> read8(const void* p) {
  typedef typename Vec8<T>::type V;
  constexpr int N = Vec8<T>::N;
  V v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = reinterpret_cast<const V*>(p)[i];
  Raw8<T> r;
  __builtin_memcpy(&r, v, sizeof(r));
  return r;
}
template <typename T>
__device__ __forceinline__ void write8(void* p, const Raw8<T>& r) {
  typedef typename Vec8<T>::type V;
  constexpr int N = Vec8<T>::N;
  V v[N];
  __builtin_memcpy(v, &r, sizeof(r));
#pragma unroll
  for (int i = 0; i < N; ++i) __builtin_nontemporal_store(v[i], reinterpret_cast<V*>(p) + i);
}
template <typename T>
__device__ __forceinline__ void load8(const char* base, int64_t i, int n, float (&f)[8]) {
  const T* p = reinterpret_cast<const T*>(base) + i;
  if (n >= 8) {
    const Raw8<T> r = read8<T>(p);
#pragma unroll
    for (int q = 0; q < 8; ++q) f[q] = (float)r.e[q];
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) f[q] = q < n ? (float)p[q] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(char* base, int64_t i, int n, const float (&f)[8]) {
  T* p = reinterpret_cast<T*>(base) + i;
  if (n >= 8) {
    Raw8<T> r;
    if constexpr (sizeof(T) == 2) {  // (in pairs: one v_cvt_pk_bf16_f32)
      bf16x2 w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = __builtin_convertvector(f32x2{f[2 * q], f[2 * q + 1]}, bf16x2);
      __builtin_memcpy(&r, w, sizeof(r));
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) r.e[q] = (T)f[q];
    }
    write8<T>(p, r);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q < n) p[q] = (T)f[q];
  }
}

// eight e4m3 codes
__device__ __forceinline__ void load_codes(const char* base, int64_t i, int n, float scale, float (&f)[8]) {
  uint32_t w[2] = {0, 0};
  if (n >= 8) {
    const Raw8<uint8_t> r = read8<uint8_t>(base + i);
    __builtin_memcpy(w, &r, 8);
  } else {
    for (int q = 0; q < n; ++q) w[q >> 2] |= (uint32_t)(uint8_t)base[i + q] << (8 * (q & 3));
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], false);
    const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], true);
    f[4 * h] = a.x * scale, f[4 * h + 1] = a.y * scale, f[4 * h + 2] = b.x * scale, f[4 * h + 3] = b.y * scale;
  }
}
__device__ __forceinline__ void store_codes(char* base, int64_t i, int n, const uint32_t (&w)[2]) {
  if (n >= 8) {
    Raw8<uint8_t> r;
    __builtin_memcpy(&r, w, 8);
    write8<uint8_t>(base + i, r);
  } else {
    for (int q = 0; q < n; ++q) base[i + q] = (char)(w[q >> 2] >> (8 * (q & 3)));
  }
}

// maximum over a row of 16 lanes, in every lane of the row (magnitudes as bit patterns: NaN above infinity above the rest)
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true));  // row_ror:8
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, true));  // row_ror:4
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, true));  // row_ror:2
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, true));  // row_ror:1
  return v;
}

// biased exponent E + 127 of the least E with top 2^-E <= 448 = 1.75 * 2^8, E >= -126; 0 for an empty block
__device__ __forceinline__ int scale_code(uint32_t top) {
  const int s = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return top ? max(s, 1) : 0;
}

// x 2^-E to e4m3 with 16 random bits each (at the top of `bits`): up with the probability of the part that is cut off.  That is
// the hardware's stochastic conversion, which also turns NaN and infinity into NaN.  KEEP (x >= 0): no value but 0 becomes 0.
template <bool KEEP>
__device__ __forceinline__ void quantise8(char* codes, uint8_t* scales, int64_t i, int n, const float (&x)[8],
                                          const uint32_t (&bits)[8]) {
  float m = fabsf(x[0]);
#pragma unroll
  for (int q = 1; q < 8; ++q) m = __builtin_elementwise_maximum(m, fabsf(x[q]));  // (NaN stays NaN)
  uint32_t top = row_max(__float_as_uint(m) & 0x7fffffffu);
  if (__builtin_amdgcn_ballot_w64(top >= 0x7f800000u)) {  // some block has a value that is not finite: leave those out
    uint32_t t = 0;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const uint32_t b = __float_as_uint(x[q]) & 0x7fffffffu;
      t = max(t, b < 0x7f800000u ? b : 0);
    }
    top = row_max(t);
  }
  const int s = scale_code(top);
  const float inv = __uint_as_float((uint32_t)(254 - max(s, 1)) << 23);  // 2^-E (an empty block: any)
  uint32_t w[2] = {0, 0};
  auto value = [&](int q) {
    float y = x[q] * inv;
    // 0 -> 0, what is below the least code -> the least code, the rest (NaN too) as it is
    if (KEEP) y = __builtin_elementwise_maximum(y, __builtin_elementwise_minimum(y * 0x1p126f, 0x1p-9f));
    return y;
  };
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    w[h] = __builtin_amdgcn_cvt_sr_fp8_f32(value(4 * h), bits[4 * h], w[h], 0);
    w[h] = __builtin_amdgcn_cvt_sr_fp8_f32(value(4 * h + 1), bits[4 * h + 1], w[h], 1);
    w[h] = __builtin_amdgcn_cvt_sr_fp8_f32(value(4 * h + 2), bits[4 * h + 2], w[h], 2);
    w[h] = __builtin_amdgcn_cvt_sr_fp8_f32(value(4 * h + 3), bits[4 * h + 3], w[h], 3);
  }
  if (n > 0) {
    store_codes(codes, i, n, w);
    if ((threadIdx.x & 15) == 0) scales[i / BLOCK8] = (uint8_t)s;
  }
}

// Eight elements per lane from element `start` of the tensor on.  (Lanes behind the end stay: a block's lanes work together.)
template <typename PT, typename GT, bool EIGHT>
__device__ __forceinline__ void chunk(const Rec& t, const Args& a, int64_t start) {
  const int64_t i = start + (int64_t)threadIdx.x * VEC;
  const int n = (int)max((int64_t)0, min((int64_t)VEC, t.numel - i));
  float p[8], g[8], m[8], v[8], r[8];
  load8<PT>(t.p, i, n, p);
  load8<GT>(t.g, i, n, g);
  if constexpr (EIGHT) {
    const float sm = n > 0 ? __uint_as_float((uint32_t)t.ms[i / BLOCK8] << 23) : 0.f;
    const float sv = n > 0 ? __uint_as_float((uint32_t)t.vs[i / BLOCK8] << 23) : 0.f;
    load_codes(t.m, i, n, sm, m);
    load_codes(t.v, i, n, sv, r);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = r[q] * r[q];
  } else {
    load8<float>(t.m, i, n, m);
    load8<float>(t.v, i, n, v);
  }
  bool tiny = false;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    m[q] = fmaf(g[q] - m[q], a.c1, m[q]);
    v[q] = fmaf(g[q] * a.c2, g[q], v[q] * a.b2);
    r[q] = __builtin_amdgcn_sqrtf(v[q]);
    tiny |= __builtin_amdgcn_classf(v[q], 0x80);
  }
  // The instruction takes a subnormal v, 2^-149 .. 2^-126, for 0.  (302 M bf16 elements with 8-bit moments: 533 us, without this
  // 527; the same with the least bit pattern of the eight values as the question.)
  if (__builtin_amdgcn_ballot_w64(tiny)) {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (v[q] < 0x1p-126f) r[q] = __builtin_amdgcn_sqrtf(v[q] * 0x1p100f) * 0x1p-50f;
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    // 1-ulp square root and reciprocal: the update they feed is a small part of p, and r is rounded to 4 bits (of 18.6 million
    // stored codes 2 differ from those of 64-bit arithmetic; of a form with correctly rounded fp32 roots 3 did)
    const float upd = m[q] * __builtin_amdgcn_rcpf(fmaf(r[q], a.inv_sqrt_bc2, a.eps));
    p[q] = fmaf(-t.step_size, upd, p[q] * t.decay);
  }
  store8<PT>(t.p, i, n, p);
  if constexpr (EIGHT) {
    uint32_t lo[8], hi[8];
    const uint32_t seg = (uint32_t)((uint64_t)i >> 32);
    const uint32_t key = seg == 0 ? t.key : mix32(t.key + seg * 0x9E3779B9u);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const uint32_t h = mix32(((uint32_t)i ^ key) ^ q);  // (i is a multiple of 8)
      lo[q] = h << 16;
      hi[q] = h & 0xffff0000u;
    }
    quantise8<false>(t.m, t.ms, i, n, m, lo);
    quantise8<true>(t.v, t.vs, i, n, r, hi);
  } else {
    store8<float>(t.m, i, n, m);
    store8<float>(t.v, i, n, v);
  }
}

__global__ __launch_bounds__(256) void adamw_kernel(const Args a) {
  int lo = 0, hi = a.n - 1;  // the last tensor whose first workgroup is not behind this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.rec[mid].chunk0 <= blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const Rec& t = a.rec[lo];
  const int64_t start = (int64_t)(blockIdx.x - t.chunk0) * CHUNK;
  const bool eight = t.ms != nullptr;
  if (t.p_dtype == CLT_BF16) {
    if (t.g_dtype == CLT_BF16) {
      if (eight) chunk<bf16_t, bf16_t, true>(t, a, start);
      else chunk<bf16_t, bf16_t, false>(t, a, start);
    } else {
      if (eight) chunk<bf16_t, float, true>(t, a, start);
      else chunk<bf16_t, float, false>(t, a, start);
    }
  } else {
    if (t.g_dtype == CLT_BF16) {
      if (eight) chunk<float, bf16_t, true>(t, a, start);
      else chunk<float, bf16_t, false>(t, a, start);
    } else {
      if (eight) chunk<float, float, true>(t, a, start);
      else chunk<float, float, false>(t, a, start);
    }
  }
}

}  // namespace
}  // namespace clt

using namespace clt;

extern "C" int clt_adamw_step(const clt_adamw_tensor* h_tensors, int n_tensors, double b1, double b2, double eps,
                              int64_t step, uint32_t seed, clt_stream_t stream) {
  CLT_CHECK_ARG(n_tensors >= 0 && (n_tensors == 0 || h_tensors), "clt_adamw_step: null pointer");
  CLT_CHECK_ARG(step >= 1, "clt_adamw_step: step is counted from 1");
  CLT_CHECK_ARG(b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0 && eps >= 0.0, "clt_adamw_step: betas in [0, 1), eps >= 0");
  for (int i = 0; i < n_tensors; ++i) {
    const clt_adamw_tensor& t = h_tensors[i];
    CLT_CHECK_ARG(t.numel >= 0, "clt_adamw_step: tensor %d: negative size", i);
    CLT_CHECK_ARG(valid_dtype(t.p_dtype) && valid_dtype(t.g_dtype), "clt_adamw_step: tensor %d: dtype", i);
    CLT_CHECK_ARG(t.numel == 0 || (t.p && t.g && t.m && t.v), "clt_adamw_step: tensor %d: null pointer", i);
    CLT_CHECK_ARG((t.m_scale == nullptr) == (t.v_scale == nullptr), "clt_adamw_step: tensor %d: one moment in 8 bits", i);
    const uintptr_t pm = dtype_size(t.p_dtype) - 1, gm = dtype_size(t.g_dtype) - 1, mm = t.m_scale ? 0 : 3;
    CLT_CHECK_ARG(!((uintptr_t)t.p & pm) && !((uintptr_t)t.g & gm) && !(((uintptr_t)t.m | (uintptr_t)t.v) & mm),
                  "clt_adamw_step: tensor %d: misaligned pointer", i);
    CLT_UNSUPPORTED(t.numel <= MAX_CHUNKS * CHUNK, "clt_adamw_step: tensor %d: fewer than 2^35 - 2047 elements", i);
  }
  const double bc1 = 1.0 - pow(b1, (double)step), bc2 = 1.0 - pow(b2, (double)step);
  Args a;
  a.c1 = (float)(1.0 - b1), a.b2 = (float)b2, a.c2 = (float)(1.0 - b2);
  a.inv_sqrt_bc2 = (float)(1.0 / sqrt(bc2)), a.eps = (float)eps;
  a.n = 0;
  int64_t chunks = 0;
  for (int i = 0; i <= n_tensors; ++i) {
    const int64_t mine = i < n_tensors ? (h_tensors[i].numel + CHUNK - 1) / CHUNK : 0;
    if (a.n && (i == n_tensors || a.n == MAX_TENSORS || chunks + mine > MAX_CHUNKS)) {
      hipLaunchKernelGGL(adamw_kernel, dim3((unsigned)chunks), dim3(256), 0, (hipStream_t)stream, a);
      CLT_CHECK_LAUNCH("clt_adamw_step");
      a.n = 0;
      chunks = 0;
    }
    if (mine == 0) continue;
    const clt_adamw_tensor& t = h_tensors[i];
    Rec& r = a.rec[a.n++];
    r.p = (char*)t.p, r.g = (const char*)t.g, r.m = (char*)t.m, r.v = (char*)t.v;
    r.ms = t.m_scale, r.vs = t.v_scale;
    r.numel = t.numel;
    r.decay = (float)(1.0 - t.lr * t.weight_decay);
    r.step_size = (float)(t.lr / bc1);
    r.key = mix32(mix32(seed + 0x9E3779B9u * (uint32_t)(i + 1)) + (uint32_t)step);
    r.chunk0 = (uint32_t)chunks;
    r.p_dtype = t.p_dtype, r.g_dtype = t.g_dtype;
    chunks += mine;
  }
  return CLT_OK;
}
