// MXFP4 on gfx950: quantisation of rows to 4-bit microscaled codes, the way back, and the encoder product on the codes
// (format: include/clt_mi355.h).
#include <type_traits>

#include "common.h"

namespace clt {
namespace {

constexpr int KPAD = 128;  // columns are padded to whole matrix-instruction steps: no bounds in the product's inner loop

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

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

// Row and column of lane i (8 columns each): FLAT: the rows are contiguous and whole blocks, so no division is needed.
template <bool FLAT>
struct Place {
  int64_t row, c;
  __device__ __forceinline__ Place(int64_t i, int64_t lanes_per_row, int64_t total) {
    if (FLAT) {
      row = 0, c = 8 * i;
    } else if (total < (1ll << 32)) {
      const uint32_t r = (uint32_t)i / (uint32_t)lanes_per_row;
      row = r, c = (int64_t)((uint32_t)i - r * (uint32_t)lanes_per_row) * 8;
    } else {
      row = i / lanes_per_row, c = (i - row * lanes_per_row) * 8;
    }
  }
};

template <typename T, bool FLAT>
__global__ __launch_bounds__(256) void mxfp4_quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t K, int64_t total,
                                                             int64_t lanes_per_row, uint32_t* __restrict__ codes,
                                                             uint8_t* __restrict__ scales) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;  // (a quad of lanes is one block and goes the same way: total and lanes_per_row are multiples of 16)
  const Place<FLAT> at(i, lanes_per_row, total);
  float f[8];
  load_row8(x + at.row * ldx, at.c, FLAT ? INT64_MAX : K, f);
  int s;
  codes[i] = quantise_lane(f, s);
  if ((i & 3) == 0) scales[i >> 2] = (uint8_t)s;
}

// ---- and back --------------------------------------------------------------------------------------------------------
template <typename T, bool FLAT>
__global__ __launch_bounds__(256) void mxfp4_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales, int64_t K, int64_t total,
                                                               int64_t lanes_per_row, T* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const Place<FLAT> at(i, lanes_per_row, total);
  if (!FLAT && at.c >= K) return;
  const uint32_t w = codes[i];
  const int s = scales[i >> 2];
  float f[8];
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
  f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y, f[4] = d.x, f[5] = d.y, f[6] = e.x, f[7] = e.y;
#pragma unroll
  for (int q = 0; q < 8; ++q) f[q] = s == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(f[q], s - 127);
  T* o = out + at.row * K + at.c;
  if (FLAT || at.c + 8 <= K) {
    Raw8<T> r;
#pragma unroll
    for (int q = 0; q < 8; ++q) r.e[q] = (T)f[q];
    *reinterpret_cast<Raw8<T>*>(o) = r;
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (at.c + q < K) o[q] = (T)f[q];
  }
}

// ---- product ---------------------------------------------------------------------------------------------------------
// v_mfma_scale_f32_32x32x64_f8f6f4 with 4-bit operands: lane l of an operand holds row l % 32, columns 32 (l / 32) .. + 31 of
// a step of 64 -- one block, 16 bytes of codes and one scale.  D: lane l holds column l % 32, rows 8 (i / 4) + 4 (l / 32) + i % 4.
template <int T>  // 64 columns: byte 2 T of the scales
__device__ __forceinline__ f32x16 mfma4s(const i32x4& a, const i32x4& b, const f32x16& c, int sa, int sb) {
  const i32x8 A = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8 B = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, c, 4, 4, 2 * T, sa, 2 * T, sb);
}

// (what lies behind `size` reads as zero, dword by dword)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const void* base, int64_t size) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)max(min(size, (int64_t)0x7fffffff), (int64_t)0), 0x00020000);
}

struct LinearArgs {
  const uint8_t *xc, *xs, *wc, *ws;
  const void* bias;
  void* out;
  int64_t N, M, ldo;
  int kp, bias_dtype, relu;
  int lines;  // the rows of out begin with a whole 128-byte line
};

// 16 bytes of a row to an address with the element's own alignment.  LINES: the row's pieces of 128 bytes are whole lines, and
// go past L2, where the operands stay (8192 tokens x 98304 x 768, bf16: 457 us, through L2 552; fp32 636, 820).  Else through
// L2, which joins the parts of a line (2048 x 43579 x 64: 43 us, past it 103).
typedef uint32_t u32x4_any2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_any4 __attribute__((ext_vector_type(4), aligned(4)));
template <bool LINES>
__device__ __forceinline__ void store_row16(bf16_t* to, u32x4 w) {
  if constexpr (LINES) __builtin_nontemporal_store((u32x4_any2)w, reinterpret_cast<u32x4_any2*>(to));
  else *reinterpret_cast<u32x4_any2*>(to) = (u32x4_any2)w;
}
template <bool LINES>
__device__ __forceinline__ void store_row16(float* to, u32x4 w) {
  if constexpr (LINES) __builtin_nontemporal_store((u32x4_any4)w, reinterpret_cast<u32x4_any4*>(to));
  else *reinterpret_cast<u32x4_any4*>(to) = (u32x4_any4)w;
}

// Few tokens (at most 16): bound by reading W, so W goes from memory to registers once and nothing else is in the way.  A wave
// takes 16 rows of W at a time (v_mfma_scale_f32_16x16x128_f8f6f4: lane l holds row l % 16, columns 32 (l / 16) .. + 31 of 128),
// with the loads of the next 512 columns -- of the next rows, at a row's end -- in flight while it multiplies.  The tokens
// lie in LDS, quantised there by every workgroup for itself when they are so few that this is cheaper than a launch (XT: float /
// bf16), else copied (XT: uint8_t).  Row pitch kp / 2 + 16 bytes: the 16 lanes of a fragment read hit different banks.
typedef __attribute__((ext_vector_type(4))) float f32x4;

__device__ __forceinline__ f32x4 mfma4_16(const i32x4& a, const i32x4& b, const f32x4& c, int sa, int sb) {
  const i32x8 A = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8 B = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, 0, sa, 0, sb);
}
// Latents m .. m + 3 of a token: bias, ReLU, one rounding.
__device__ __forceinline__ f32x4 bias_four(const LinearArgs& p, int64_t m) {
  f32x4 b = {};
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = load_scalar(p.bias, p.bias_dtype, min(m + i, p.M - 1));
  }
  return b;
}
template <typename T>
__device__ __forceinline__ void store_four(const LinearArgs& p, T* row, int64_t m, const f32x4& acc, const f32x4& b) {
  struct __attribute__((packed, aligned(sizeof(T)))) Four {
    T e[4];
  };
  Four o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float v = acc[i] + b[i];
    o.e[i] = (T)(p.relu ? __builtin_elementwise_maximum(v, 0.f) : v);
  }
  if (m + 4 <= p.M) {
    *reinterpret_cast<Four*>(row + m) = o;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (m + i < p.M) row[m + i] = o.e[i];
  }
}
template <typename XT, typename T>
__global__ __launch_bounds__(256) void mxfp4_few_kernel(const LinearArgs p, const XT* __restrict__ x, int64_t ldx, int K) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int rowb = p.kp / 2, sb = p.kp / 32, pitch = rowb + 16, nks = p.kp / 128;
  const int N = (int)p.N;
  char* xs = lds + 16 * pitch;  // scales, sb bytes a row
  if constexpr (sizeof(XT) == 1) {
    for (int i = threadIdx.x; i < N * (rowb / 16); i += 256) {
      const int row = i / (rowb / 16), c = i - row * (rowb / 16);
      *reinterpret_cast<uint4*>(lds + row * pitch + 16 * c) = reinterpret_cast<const uint4*>(p.xc)[i];
    }
    for (int i = threadIdx.x; i < N * (sb / 4); i += 256) reinterpret_cast<uint32_t*>(xs)[i] = reinterpret_cast<const uint32_t*>(p.xs)[i];
  } else {
    const int lpr = p.kp / 8;  // (a multiple of 16: the four lanes of a block go the same way)
    for (int i = threadIdx.x; i < N * lpr; i += 256) {
      const int row = i / lpr, c = i - row * lpr;
      float f[8];
      load_row8(x + row * ldx, 8 * c, K, f);
      int s;
      *reinterpret_cast<uint32_t*>(lds + row * pitch + 4 * c) = quantise_lane(f, s);
      if ((c & 3) == 0) xs[row * sb + c / 4] = (char)s;
    }
  }
  __syncthreads();

  const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
  const int64_t groups = (p.M + 15) / 16, step = (int64_t)gridDim.x * 4;
  const int nch = (nks + 3) / 4;  // pieces of 512 columns
  int64_t g = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (g >= groups) return;
  struct Piece {
    u32x4 w[4], s;
  };
  auto load = [&](int64_t group, int c, Piece& v) {
    const auto codes = resource(p.wc + group * 16 * rowb, (p.M - group * 16) * rowb);
    const auto scales = resource(p.ws + group * 16 * sb, (p.M - group * 16) * sb);
    v.s = __builtin_amdgcn_raw_buffer_load_b128(scales, r16 * sb + 16 * c, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (4 * c + j < nks) v.w[j] = __builtin_amdgcn_raw_buffer_load_b128(codes, r16 * rowb + 256 * c + 64 * j + 16 * q, 0, 0);
  };
  T* out = reinterpret_cast<T*>(p.out);
  Piece now, then;
  load(g, 0, now);
  while (g < groups) {
    const int64_t m = g * 16 + 4 * q;  // this lane's four latents
    const f32x4 b = bias_four(p, m);
    f32x4 acc = {};
    const int64_t next = g + step;
    for (int c = 0; c < nch; ++c) {
      if (c + 1 < nch) load(g, c + 1, then);
      else if (next < groups) load(next, 0, then);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (4 * c + j >= nks) break;
        const i32x4 xf = *reinterpret_cast<const i32x4*>(lds + r16 * pitch + 256 * c + 64 * j + 16 * q);
        const uint32_t xsc = *reinterpret_cast<const uint32_t*>(xs + r16 * sb + 16 * c + 4 * j);
        acc = mfma4_16(__builtin_bit_cast(i32x4, now.w[j]), xf, acc, (int)(now.s[j] >> (8 * q)), (int)(xsc >> (8 * q)));
      }
      now = then;
    }
    if (r16 < N) store_four(p, out + r16 * p.ldo, m, acc, b);
    g = next;
  }
}

// Small and middle-sized problems.  A workgroup of four waves computes 64 B latents x 64 B tokens, a wave a quarter of them; four
// (B = 1) or two workgroups share a CU, so that the waits, the first loads and the stores of one run beside the matrix
// instructions of the others.  Per stage of 256 columns both operands come as whole lines of 128 bytes by LDS-DMA into a ring of
// two slots, one stage ahead; what lies behind an array's last row reads as zeros.  Chunk c of a row lies at c ^ (row / 2 % 8):
// fragment reads (16 rows, one chunk) hit every bank once.  The finished tile goes through the ring's LDS once, so that a store
// instruction writes rows of 64 to 256 bytes.
//   Bound by a stage's chain of fetch, fragment reads and matrix instructions (0.3 us with B = 1, 0.7 with B = 2) while there is
// a workgroup or two a CU, then by LDS and the matrix instructions together: B = 2 reads LDS half as often per product.  950 tokens x
// 2048 x 4096: 11.0 us with B = 1, 17.1 with B = 2 (256 x 128 tiles, stages of 128 columns: 26); 950 x 16384 x 768: 18.7, 16.9.
//   Three or four slots with one workgroup a CU: the same at 512 x 6151 x 4096, up to 1.7 x the time where tiles are many.  A
// second barrier that lets a slot be refilled a step earlier saves 15 % where W comes from HBM for one row of tiles (128 x 98304 x
// 768: 18 for 21 us, B = 2) and costs 3 to 9 % elsewhere.
constexpr int BPANEL = 16;  // latent tiles that run through all tokens together

typedef __attribute__((address_space(3))) void* lds_ptr_t;
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ i32x4 buffer_of(const uint8_t* base, int64_t size) {
  const uint64_t a = (uint64_t)base;
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32) & 0xffff);
  r[2] = __builtin_amdgcn_readfirstlane((int)(uint32_t)min(size, (int64_t)0x80000000));
  r[3] = 0x00020000;
  return r;
}
// LDS[lds_dst + 16 * lane] = buf[voff .. voff + 15]; what lies behind the buffer's end reads as zero.
__device__ __forceinline__ void dma16_buffer(const i32x4& buf, uint32_t voff, uint32_t lds_dst) {
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %3\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(voff), "s"(buf), "s"(lds_dst)
      : "memory");
}

// The same for some of the lanes (all lanes are active where this stands).
__device__ __forceinline__ void dma16_lanes(const i32x4& buf, uint32_t voff, uint32_t lds_dst, int low, int high) {
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %3\n\t"
      "s_mov_b32 exec_lo, %4\n\t"
      "s_mov_b32 exec_hi, %5\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds\n\t"
      "s_mov_b64 exec, -1\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(voff), "s"(buf), "s"(lds_dst), "i"(low), "i"(high)
      : "memory");
}

// The same, and with four bytes a lane, for all lanes (mask -1) or none (0); all lanes are active where these stand.
__device__ __forceinline__ void dma16_masked(const i32x4& buf, uint32_t voff, uint32_t lds_dst, int mask) {
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %3\n\t"
      "s_mov_b32 exec_lo, %4\n\t"
      "s_mov_b32 exec_hi, %4\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds\n\t"
      "s_mov_b64 exec, -1\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(voff), "s"(buf), "s"(lds_dst), "s"(mask)
      : "memory");
}
__device__ __forceinline__ void dma4_masked(const i32x4& buf, uint32_t voff, uint32_t lds_dst, int mask) {
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %3\n\t"
      "s_mov_b32 exec_lo, %4\n\t"
      "s_mov_b32 exec_hi, %4\n\t"
      "buffer_load_dword %1, %2, 0 offen lds\n\t"
      "s_mov_b64 exec, -1\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(voff), "s"(buf), "s"(lds_dst), "s"(mask)
      : "memory");
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {  // one v_cvt_pk_bf16_f32
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}

// One step of a transposition of 16-byte chunks between the lanes l and l ^ 1 (or l ^ 2): lanes with that bit clear keep p and
// take the other's p as q, the others keep q and take the other's q as p.  (DPP reads a register two slots after its write.)
template <int XOR>
__device__ __forceinline__ void exchange(u32x4& p, u32x4& q) {
  u32x4 a, b;
  const uint64_t low = XOR == 1 ? 0x5555555555555555ull : 0x3333333333333333ull;
#define CLT_STEP(PERM)                                                                                  \
  asm("s_mov_b64 vcc, %8\n\ts_nop 1\n\t"                                                              \
      "v_cndmask_b32_dpp %0, %6, %4, vcc " PERM "\n\tv_cndmask_b32_dpp %1, %7, %5, vcc " PERM           \
      "\n\ts_not_b64 vcc, vcc\n\t"                                                                     \
      "v_cndmask_b32_dpp %2, %4, %6, vcc " PERM "\n\tv_cndmask_b32_dpp %3, %5, %7, vcc " PERM           \
      : "=&v"(o[0]), "=&v"(o[1]), "=&v"(o[2]), "=&v"(o[3])                                              \
      : "v"(p[d]), "v"(p[d + 1]), "v"(q[d]), "v"(q[d + 1]), "s"(low)                                    \
      : "vcc", "scc")
#pragma unroll
  for (int d = 0; d < 4; d += 2) {
    uint32_t o[4];
    if constexpr (XOR == 1) CLT_STEP("quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf");
    else CLT_STEP("quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf");
    a[d] = o[0], a[d + 1] = o[1], b[d] = o[2], b[d + 1] = o[3];
  }
#undef CLT_STEP
  p = a;
  q = b;
}
// Eight chunks of a lane (a line of 128 bytes of its token) -> line[s]: the chunk l % 4 + 4 (l / 16 % 2) of token 4 (l / 4 % 4) + s
// + 16 (s >> 2) of this half of the wave.
__device__ __forceinline__ void lines_of(u32x4 (&c)[8]) {
#pragma unroll
  for (int g = 0; g < 8; g += 4) {
    exchange<1>(c[g], c[g + 1]);
    exchange<1>(c[g + 2], c[g + 3]);
    exchange<2>(c[g], c[g + 2]);
    exchange<2>(c[g + 1], c[g + 3]);
  }
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const auto r = __builtin_amdgcn_permlane16_swap(c[s][d], c[s + 4][d], false, false);
      c[s][d] = r[0], c[s + 4][d] = r[1];
    }
}

template <typename T, int B>
__global__ __launch_bounds__(256, 4 / B) void mxfp4_tile_kernel(const LinearArgs p) {
  constexpr int TS = 64 * B, WS = 32 * B, SLOT = 2 * TS * (128 + 16);  // side of a tile, of a wave's part; bytes of a stage
  static_assert(4 / B * 2 * SLOT <= 160 * 1024, "LDS of 4 / B workgroups");
  __shared__ __attribute__((aligned(1024))) char lds[2 * SLOT];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5, wm = wave >> 1, wn = wave & 1;

  // ---- tile: an XCD (workgroup id % 8) owns a contiguous range of positions; a panel of latent tiles runs through all tokens
  const int64_t nlt = (p.M + TS - 1) / TS, ntt = (p.N + TS - 1) / TS, ntiles = nlt * ntt;
  const int64_t xg = blockIdx.x & 7, q = ntiles >> 3, rest = ntiles & 7;
  const int64_t pos = xg * q + min(xg, rest) + (blockIdx.x >> 3);
  const int64_t panel = pos / (ntt * BPANEL), in = pos - panel * ntt * BPANEL;
  const int64_t width = min((int64_t)BPANEL, nlt - panel * BPANEL);
  const int64_t n0 = in / width * TS, m0 = (panel * BPANEL + in % width) * TS;

  // ---- loader: WS rows a wave (waves 0, 1: W, 2, 3: x), in pieces of eight rows, and their scales
  const int rowb = p.kp / 2, sb = p.kp / 32, nst = (p.kp + 255) / 256;
  const int64_t row0 = (wave < 2 ? m0 : n0) + WS * (wave & 1), left = max((wave < 2 ? p.M : p.N) - row0, (int64_t)0);
  const i32x4 cbuf = buffer_of((wave < 2 ? p.wc : p.xc) + row0 * rowb, left * rowb);
  const i32x4 sbuf = buffer_of((wave < 2 ? p.ws : p.xs) + row0 * sb, left * sb);
  const uint32_t chunk = ((lane & 7) ^ (lane >> 4)) << 4;
  const uint32_t even = (uint32_t)(lane >> 3) * rowb + chunk, odd = even - chunk + (chunk ^ 64);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds + wave * (WS * 128);
  const uint32_t sc0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds + 2 * TS * 128 + wave * (WS * 16);
  auto fetch = [&](int s, int slot) {
#pragma unroll
    for (int i = 0; i < WS / 8; ++i)
      dma16_buffer(cbuf, ((i & 1) ? odd : even) + (uint32_t)(128 * s + i * 8 * rowb), lds0 + slot * SLOT + i * 1024);
    dma16_lanes(sbuf, (uint32_t)(lane * sb + 8 * s), sc0 + slot * SLOT, -1, B == 1 ? 0 : -1);
  };

  // ---- multiplier
  f32x16 acc[B][B] = {};  // [latents][tokens]; lane (r32, h): token r32, latents 8 g + 4 h + j
  const uint32_t at = r32 * 128 + ((h ^ (r32 >> 1 & 7)) << 4);
  const uint32_t wat = wm * (WS * 128) + at, xat = (2 + wn) * (WS * 128) + at;
  fetch(0, 0);
  for (int s = 0; s < nst; ++s) {
    // stage s is there, and every wave is past stage s - 1
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (s + 1 < nst) fetch(s + 1, ~s & 1);
    const char* base = lds + (s & 1) * SLOT;
    i32x4 w[B][4], x[B][4];
    u32x2 sw[B], sx[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      sw[i] = *reinterpret_cast<const u32x2*>(base + 2 * TS * 128 + (wm * WS + 32 * i + r32) * 16);
      sx[i] = *reinterpret_cast<const u32x2*>(base + 2 * TS * 128 + (TS + wn * WS + 32 * i + r32) * 16);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < B; ++i) {
        w[i][j] = *reinterpret_cast<const i32x4*>(base + i * 4096 + (wat ^ (32 * j)));
        x[i][j] = *reinterpret_cast<const i32x4*>(base + i * 4096 + (xat ^ (32 * j)));
      }
    const bool cut = 256 * s + 128 >= p.kp;  // (behind a row's last 128 columns stands the next row: counted 2^-254 times)
#pragma unroll
    for (int i = 0; i < B; ++i) {
      sw[i][1] = cut ? 0 : sw[i][1];
      sx[i][1] = cut ? 0 : sx[i][1];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < B; ++i)
#pragma unroll
        for (int k = 0; k < B; ++k) {
          const int s1 = (int)(sw[i][j >> 1] >> (8 * h)), s2 = (int)(sx[k][j >> 1] >> (8 * h));
          acc[i][k] = j & 1 ? mfma4s<1>(w[i][j], x[k][j], acc[i][k], s1, s2) : mfma4s<0>(w[i][j], x[k][j], acc[i][k], s1, s2);
        }
  }

  // ---- epilogue: bias, ReLU, one rounding
  __syncthreads();  // (the ring is free)
  constexpr int OPITCH = WS * sizeof(T) + 16, VEC = 16 / sizeof(T), ROWL = WS / VEC, ROWS = 64 / ROWL;
  float* bias = reinterpret_cast<float*>(lds + 4 * 32 * OPITCH);
  if (threadIdx.x < TS) {
    const int64_t m = m0 + threadIdx.x;
    bias[threadIdx.x] = p.bias && m < p.M ? load_scalar(p.bias, p.bias_dtype, m) : 0.f;
  }
  __syncthreads();
  char* mine = lds + wave * 32 * OPITCH;
  T* out = reinterpret_cast<T*>(p.out);
#pragma unroll
  for (int k = 0; k < B; ++k) {
#pragma unroll
    for (int i = 0; i < B; ++i) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int lat = i * 32 + 8 * g + 4 * h;
        const float4 b = *reinterpret_cast<const float4*>(bias + wm * WS + lat);
        float v[4] = {acc[i][k][4 * g] + b.x, acc[i][k][4 * g + 1] + b.y, acc[i][k][4 * g + 2] + b.z, acc[i][k][4 * g + 3] + b.w};
        if (p.relu) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = __builtin_elementwise_maximum(v[e], 0.f);
        }
        char* to = mine + r32 * OPITCH + lat * sizeof(T);
        if constexpr (sizeof(T) == 2) {
          uint2 w;
          w.x = pack_bf16x2(v[0], v[1]), w.y = pack_bf16x2(v[2], v[3]);
          *reinterpret_cast<uint2*>(to) = w;
        } else {
          *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
        }
      }
    }
    asm volatile("" ::: "memory");  // (one wave, and a wave's LDS accesses are carried out in order)
    __builtin_amdgcn_wave_barrier();
    const int64_t m = m0 + wm * WS + (lane % ROWL) * VEC;
#pragma unroll
    for (int i = 0; i < 32 / ROWS; ++i) {
      const int tok = ROWS * i + lane / ROWL;
      const u32x4 w = *reinterpret_cast<const u32x4*>(mine + tok * OPITCH + (lane % ROWL) * 16);
      const int64_t n = n0 + wn * WS + k * 32 + tok;
      if (n >= p.N) continue;
      T* to = out + n * p.ldo + m;
      if (m + VEC <= p.M) {
        store_row16<false>(to, w);
      } else {
        T e[VEC];
        __builtin_memcpy(e, &w, 16);
#pragma unroll
        for (int c = 0; c < VEC; ++c)
          if (m + c < p.M) to[c] = e[c];
      }
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
}

// Long rows, few tiles.  32 latents x 32 tokens by four waves, each with a contiguous quarter of the columns; they add up in LDS,
// in their order.  A wave works by itself: it fetches its rows 256 columns at a time, whole lines of 128 bytes, into two slots of
// its own, so that no barrier stands in the loop.  (With fragments straight from memory, 16 lanes that are served together read
// 16 lines: four times the accesses, and 7.2 us instead of 4.7 for 128 tokens x 2048 x 4096.)  Bound by the loads' latency.
constexpr int SB_ROW = 16;  // bytes of scales kept with a row and 256 columns (8 are its own)
template <typename T>
__global__ __launch_bounds__(256) void mxfp4_split_kernel(const LinearArgs p) {
  constexpr int S = 4, ROWS = 32, CODES = 2 * ROWS * 128, SLOT = CODES + 2 * ROWS * SB_ROW, PIECES = 2 * ROWS / 8 + 2;
  constexpr int PITCH = ROWS + 8;  // of the sums, in floats
  static_assert(ROWS * PITCH * 4 <= 2 * SLOT && 8 * SLOT <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(1024))) char lds[8 * SLOT];
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char* own = lds + wave * 2 * SLOT;
  const uint32_t own0 = (uint32_t)(uintptr_t)(lds_ptr_t)own;

  // ---- tile: an XCD (workgroup id % 8) owns a contiguous range, tokens fastest: W comes to one L2 only
  const int64_t nlt = (p.M + ROWS - 1) / ROWS, ntt = (p.N + ROWS - 1) / ROWS, ntiles = nlt * ntt;
  const int64_t xg = blockIdx.x & 7, share = ntiles >> 3, rest = ntiles & 7;
  const int64_t pos = xg * share + min(xg, rest) + (blockIdx.x >> 3);
  const int64_t m0 = pos / ntt * ROWS, n0 = pos % ntt * ROWS;

  const int rowb = p.kp / 2, sb = p.kp / 32, nch = (p.kp + 255) / 256, per = (nch + S - 1) / S;
  const int first = wave * per, stop = min(nch, first + per);
  const int64_t mleft = p.M - m0, nleft = p.N - n0;
  const i32x4 wbuf = buffer_of(p.wc + m0 * rowb, mleft * rowb), xbuf = buffer_of(p.xc + n0 * rowb, nleft * rowb);
  const i32x4 wsbuf = buffer_of(p.ws + m0 * sb, mleft * sb), xsbuf = buffer_of(p.xs + n0 * sb, nleft * sb);
  auto none = [](i32x4 buf, bool on) {
    buf[2] = on ? buf[2] : 0;
    return buf;
  };
  // Chunk c of a row lies at c ^ (row / 2 % 8): fragment reads (16 rows, one chunk) hit every bank once.
  const uint32_t chunk = ((lane & 7) ^ (lane >> 4)) << 4;
  const uint32_t even = (uint32_t)(lane >> 3) * rowb + chunk, odd = even - chunk + (chunk ^ 64);
  auto fetch = [&](int c, int slot) {  // (behind `stop`: zeros, so that the pieces in flight are always as many)
    const bool on = c < stop;
    const i32x4 wb = none(wbuf, on), xb = none(xbuf, on);
    const uint32_t to = own0 + slot * SLOT;
#pragma unroll
    for (int i = 0; i < 2 * ROWS / 8; ++i) {  // eight rows each: W's, then x's
      const int piece = i % (ROWS / 8);
      dma16_buffer(i < ROWS / 8 ? wb : xb, ((piece & 1) ? odd : even) + (uint32_t)(128 * c + piece * 8 * rowb), to + i * 1024);
    }
    dma16_lanes(none(wsbuf, on), (uint32_t)(r * sb + 8 * c), to + CODES, -1, 0);
    dma16_lanes(none(xsbuf, on), (uint32_t)(r * sb + 8 * c), to + CODES, 0, -1);
  };
  f32x16 acc = {};  // lane (r, h): latent r, tokens 8 g + 4 h + j
  const uint32_t at = r * 128 + ((h ^ (r >> 1 & 7)) << 4);
  auto multiply = [&](int c, int slot) {
    const char* base = own + slot * SLOT;
    i32x4 w[4], x[4];
    u32x2 sw = *reinterpret_cast<const u32x2*>(base + CODES + r * SB_ROW);
    u32x2 sx = *reinterpret_cast<const u32x2*>(base + CODES + (ROWS + r) * SB_ROW);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = *reinterpret_cast<const i32x4*>(base + (at ^ (32 * j)));
      x[j] = *reinterpret_cast<const i32x4*>(base + ROWS * 128 + (at ^ (32 * j)));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot is free
    fetch(c + 2, slot);
    if (256 * c + 128 >= p.kp) sw[1] = sx[1] = 0;  // (behind a row's last 128 columns stands the next row: counted 2^-254 times)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int s1 = (int)(sx[j >> 1] >> (8 * h)), s2 = (int)(sw[j >> 1] >> (8 * h));
      acc = j & 1 ? mfma4s<1>(x[j], w[j], acc, s1, s2) : mfma4s<0>(x[j], w[j], acc, s1, s2);
    }
  };
  if (first < stop) {
    fetch(first, 0);
    fetch(first + 1, 1);
    for (int c = first; c < stop; ++c) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PIECES) : "memory");
      multiply(c, (c - first) & 1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the sums go where the slots are)
  }
  float* sums = reinterpret_cast<float*>(own);
#pragma unroll
  for (int e = 0; e < 16; ++e) sums[(8 * (e / 4) + 4 * h + e % 4) * PITCH + r] = acc[e];
  __syncthreads();
  // four latents of a token per thread
  T* out = reinterpret_cast<T*>(p.out);
  constexpr int QUADS = ROWS / 4;
#pragma unroll
  for (int e = 0; e < ROWS * QUADS / 256; ++e) {
    const int item = e * 256 + (int)threadIdx.x, n = item / QUADS, m = item % QUADS * 4;
    f32x4 v = *reinterpret_cast<const f32x4*>(lds + (n * PITCH + m) * 4);
#pragma unroll
    for (int k = 1; k < S; ++k) v += *reinterpret_cast<const f32x4*>(lds + k * 2 * SLOT + (n * PITCH + m) * 4);
    if (n < nleft && m < mleft) store_four(p, out + (n0 + n) * p.ldo, m0 + m, v, bias_four(p, m0 + m));
  }
}

// The largest problems.  One persistent workgroup of eight waves per CU computes tiles of 256 latents x 256 tokens (a wave
// 128 x 64: 4 x 2 tiles of 32 x 32, 128 accumulators, two waves per SIMD).
//   * A stage is 256 columns: rows of 128 bytes, whole cache lines (pieces of 64-byte rows reach half the LDS-DMA rate), 64 KiB
//     per stage in a ring of two slots.  Chunk c of a row lies at c ^ (row / 2 % 8) ^ 4 (row / 64 % 2), so a fragment read
//     (32 rows, one chunk each) is free of conflicts.  The DMAs go through buffers: rows behind the last one read as zeros.
//   * A stage is four steps of eight matrix instructions.  The fragments of a step are read during the step before it, also
//     across the stages' border: the wait for the next stage and the barrier stand before a stage's LAST step, whose
//     fragments are in registers by then; behind it the slot is free, and the DMAs of the stage after the next one go out
//     between the matrix instructions.  A row's last stage may be half empty: what stands there is the next row's, and counts
//     2^-254 times (a code is never NaN).
//   * Scales come as 16 bytes of a row for two stages, in two buffers.
//   * The rows of W are dealt to the matrix instructions' rows so that a lane ends up with 64 consecutive latents of one token
//     (D: lane l holds column l % 32, rows 8 g + 4 (l / 32) + j).  Their 16-byte chunks are exchanged in registers, between the
//     four lanes of a quad and between neighbouring rows of 16 lanes: a store instruction then writes whole lines of 128
//     bytes, and the epilogue needs neither LDS nor a barrier.  The stores are issued behind the DMAs that the next tile waits
//     for, and drain while that tile runs.
constexpr int BM = 256, BN = 256, BK = 256;
constexpr int BSLOT = (BM + BN) * 128, BSCALE_OFF = 2 * BSLOT, BSCALE = (BM + BN) * 16;
constexpr int BBIAS_OFF = BSCALE_OFF + 2 * BSCALE, BIG_LDS = BBIAS_OFF + 3 * BM * 4;
static_assert(BIG_LDS <= 160 * 1024, "LDS");

typedef __attribute__((ext_vector_type(2))) int i32x2;
typedef int i32x2_a4 __attribute__((ext_vector_type(2), aligned(4)));

struct Frags {
  i32x4 a[4], b[2];
};

template <typename T, bool RELU>
__global__ __launch_bounds__(512) void mxfp4_big_kernel(const LinearArgs p) {
  __shared__ __attribute__((aligned(1024))) char lds[BIG_LDS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5, wm = wave >> 2, wn = wave & 3;
  const int rowb = p.kp / 2, sb = p.kp / 32, nst = (p.kp + BK - 1) / BK;
  const bool half = p.kp % BK != 0;  // the last stage has 128 columns
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds;

  // ---- tiles of this workgroup: its XCD (id % 8) owns a contiguous range of positions, a panel of latent tiles runs through
  //      all tokens, latents fastest: the rows that an XCD writes at a time are long and its operands stay in its L2
  const int nlt = (int)((p.M + BM - 1) / BM), ntt = (int)((p.N + BN - 1) / BN);
  const int ntiles = nlt * ntt;  // (host: < 2^31)
  const int xg = blockIdx.x & 7, nbx = ((int)gridDim.x - xg + 7) >> 3;
  const int q = ntiles >> 3, rest = ntiles & 7;
  const int xstart = xg * q + min(xg, rest), xstop = xstart + q + (xg < rest);
  int pos = xstart + (blockIdx.x >> 3);
  if (pos >= xstop) return;
  auto place = [&](int at, int64_t& m0, int64_t& n0) {
    const uint32_t full = (uint32_t)ntt * BPANEL;
    const uint32_t panel = (uint32_t)at / full, in = (uint32_t)at - panel * full;
    const uint32_t width = min((uint32_t)BPANEL, (uint32_t)nlt - panel * BPANEL);
    const uint32_t row = in / width;
    n0 = (int64_t)__builtin_amdgcn_readfirstlane(row) * BN;
    m0 = (int64_t)__builtin_amdgcn_readfirstlane(panel * BPANEL + in - row * width) * BM;
  };

  // ---- loader: runs two stages ahead of the multiplier.  What lies behind an array's end reads as zero (dword by dword).
  const bool bias_dma = p.bias && p.bias_dtype == CLT_F32;
  i32x4 wbuf, xbuf, sbuf_, bbuf;  // from the tile's first row: codes, this wave's scales (waves 0 .. 3: W, 4 .. 7: x), bias
  int lpos = pos, ls = 0, lslot = 0, lsbuf = 0, lbias = 0;  // the stage to be fetched next and where to
  const uint32_t chunk = ((lane & 7) ^ (lane >> 4) ^ (2 * wave & 4)) << 4;  // (row / 2 % 8 = lane / 16, + 4 in an odd piece)
  const uint32_t even = (uint32_t)(32 * wave + (lane >> 3)) * rowb + chunk, odd_ = even - chunk + (chunk ^ 64);
  const uint32_t srow = (uint32_t)((wave & 3) * 64 + lane) * sb;
  auto aim = [&]() {
    if (lpos >= xstop) {  // nothing more to fetch: every later piece reads zeros
      wbuf[2] = xbuf[2] = sbuf_[2] = bbuf[2] = 0;
      return;
    }
    int64_t m0, n0;
    place(lpos, m0, n0);
    wbuf = buffer_of(p.wc + m0 * rowb, (p.M - m0) * rowb);
    xbuf = buffer_of(p.xc + n0 * rowb, (p.N - n0) * rowb);
    sbuf_ = wave < 4 ? buffer_of(p.ws + m0 * sb, (p.M - m0) * sb) : buffer_of(p.xs + n0 * sb, (p.N - n0) * sb);
    bbuf = buffer_of(reinterpret_cast<const uint8_t*>(p.bias) + m0 * 4, bias_dma ? (p.M - m0) * 4 : 0);
  };
  auto load_piece = [&](int i) {  // 0 .. 3: W, 4 .. 7: x
    dma16_buffer(i < 4 ? wbuf : xbuf, ((i & 1) ? odd_ : even) + (uint32_t)(ls * 128 + (i & 3) * 8 * rowb),
                 lds0 + lslot * BSLOT + wave * 4096 + (i >> 2) * (BM * 128) + (i & 3) * 1024);
  };
  // (no branches in what stands between matrix instructions: the compiler would move those behind them)
  auto load_scales = [&]() {  // with every other stage; and with a tile's first stage its bias (64 latents a wave, twice)
    const int now = uni(~ls & 1), tile0 = uni(ls == 0 && bias_dma);
    dma16_masked(sbuf_, srow + 8 * ls, lds0 + BSCALE_OFF + lsbuf * BSCALE + wave * 1024, -now);
    dma4_masked(bbuf, ((wave & 3) * 64 + lane) * 4, lds0 + BBIAS_OFF + lbias * (BM * 4) + (wave & 3) * 256, -tile0);
    lsbuf ^= now;
    lbias = lbias + tile0 == 3 ? 0 : lbias + tile0;
  };
  auto advance = [&]() {
    lslot ^= 1;
    if (++ls == nst) {
      ls = 0;
      lpos += nbx;
      aim();
    }
  };

  // ---- multiplier
  // this lane's row of W (+ 16 i in row tile i) and its byte in step 0; step t is at byte ^ 32 t
  const int wrow = wm * 128 + (r32 >> 2 & 1) * 64 + (r32 >> 3) * 4 + (r32 & 3), xrow = wn * 64 + r32;
  const uint32_t wat = wrow * 128 + ((h ^ (wrow >> 1 & 7) ^ (wrow >> 4 & 4)) << 4);
  const uint32_t xat = BM * 128 + xrow * 128 + ((h ^ (xrow >> 1 & 7) ^ (xrow >> 4 & 4)) << 4);
  f32x16 acc[4][2];
  Frags F0, F1;
  i32x2 raw[6], sc[6];  // scales of four row tiles of W and two of x: as read, and with this lane's blocks in bytes 0 and 2
  auto read_frag = [&](Frags& f, int e, const char* base, int t) {  // in the order of their use
    const char* a = base + (wat ^ (32 * t));
    const char* b = base + (xat ^ (32 * t));
    if (e == 0) f.b[0] = *reinterpret_cast<const i32x4*>(b);
    if (e == 1) f.a[0] = *reinterpret_cast<const i32x4*>(a);
    if (e == 2) f.b[1] = *reinterpret_cast<const i32x4*>(b + 4096);
    if (e >= 3) f.a[e - 2] = *reinterpret_cast<const i32x4*>(a + (e - 2) * 2048);
  };
  auto read_scales = [&](int s, int buf) {
    const char* base = lds + BSCALE_OFF + buf * BSCALE + 8 * (s & 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = *reinterpret_cast<const i32x2*>(base + (wrow + 16 * i) * 16);
#pragma unroll
    for (int i = 0; i < 2; ++i) raw[4 + i] = *reinterpret_cast<const i32x2*>(base + (BM + xrow + 32 * i) * 16);
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  // Step t of a stage: eight matrix instructions on `cur` (to: acc = instead of acc +=, a tile's first); between them the
  // fragments of the next step come in and, if `piece` >= 0, four pieces go out.
  auto step = [&](auto t_, auto first_, auto piece_, const Frags& cur, Frags& nxt, const char* base, int tn) {
    constexpr int t = decltype(t_)::value, piece = decltype(piece_)::value;
    constexpr bool first = decltype(first_)::value;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f32x16& c = acc[e >> 1][e & 1];
      c = mfma4s<t & 1>(cur.a[e >> 1], cur.b[e & 1], first ? f32x16{} : c, sc[e >> 1][t >> 1], sc[4 + (e & 1)][t >> 1]);
      if (e < 6) read_frag(nxt, e, base, tn);
      if (piece >= 0 && (e & 1)) load_piece(piece + (e >> 1));
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto pin = [&]() {  // the sums are computed here, not further down
    asm volatile("" : "+v"(acc[0][0]), "+v"(acc[0][1]), "+v"(acc[1][0]), "+v"(acc[1][1]), "+v"(acc[2][0]), "+v"(acc[2][1]),
                 "+v"(acc[3][0]), "+v"(acc[3][1]));
  };
  using None = std::integral_constant<int, -1>;
  using P0 = std::integral_constant<int, 0>;
  using P4 = std::integral_constant<int, 4>;

  int64_t m0, n0;
  place(pos, m0, n0);
  aim();
#pragma unroll
  for (int k = 0; k < 2; ++k) {  // (the second stage is half on its way when the loop begins: see `stage`)
    load_scales();
#pragma unroll
    for (int i = 0; i < 8; ++i) load_piece(i);
    advance();
  }
  asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  int slot = 0, sbuf = 0;  // of the stage that is multiplied
  int tile = 0;            // modulo 3: the loader is up to two tiles ahead, so that three biases are there at a time
  read_scales(0, 0);
#pragma unroll
  for (int e = 0; e < 6; ++e) read_frag(F0, e, lds, 0);

  T* out = reinterpret_cast<T*>(p.out);
  constexpr int VEC = 16 / sizeof(T), NSTORE = 8 * sizeof(T);
  const int nl = wn * 64 + 4 * (lane >> 2 & 3);  // the token and the latent (in the tile) of this lane's first store
  const int ml = wm * 128 + 64 * h + ((lane >> 4 & 1) * 4 + (lane & 3)) * VEC;
  const uint32_t lane_out = (uint32_t)(nl * (int)p.ldo + ml) * (uint32_t)sizeof(T);
  float* bias = reinterpret_cast<float*>(lds + BBIAS_OFF);
  if (!bias_dma) {
    for (int i = threadIdx.x; i < 3 * BM; i += 512) bias[i] = 0.f;
  }

  for (;;) {
    auto stage = [&](int s, auto first_) {
      constexpr bool first = decltype(first_)::value;
      const bool final = s == nst - 1;
      const char* st = lds + slot * BSLOT;
      const char* sn = lds + (slot ^ 1) * BSLOT;
      const int s1 = final ? 0 : s + 1, sbuf1 = (s1 & 1) ? sbuf : sbuf ^ 1;
      const bool cut = half && final;
#pragma unroll
      for (int i = 0; i < 6; ++i) {
        sc[i][0] = (int)((uint32_t)raw[i][0] >> (8 * h));
        sc[i][1] = cut ? 0 : (int)((uint32_t)raw[i][1] >> (8 * h));
      }
      if constexpr (first) {  // (its successor's pieces went out in front of the stores)
        step(I0{}, std::true_type{}, None{}, F0, F1, st, 1);
      } else {
        step(I0{}, std::false_type{}, P4{}, F0, F1, st, 1);
        pin();
        advance();
      }
      step(I1{}, std::false_type{}, None{}, F1, F0, st, 2);
      step(I2{}, std::false_type{}, None{}, F0, F1, st, 3);
      pin();
      // The next stage is there, and every wave has what it needs of this one.  (In a tile's first stage nothing has been
      // issued behind the stores of the tile before; what stands in front of them is what is waited for.)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(first ? NSTORE : 0) : "memory");
      read_scales(s1, sbuf1);
      load_scales();
      step(I3{}, std::false_type{}, P0{}, F1, F0, sn, 0);
      pin();
      slot ^= 1;
      sbuf = sbuf1;
    };
    stage(0, std::true_type{});
#pragma unroll 1
    for (int s = 1; s < nst; ++s) stage(s, std::false_type{});
#pragma unroll
    for (int i = 4; i < 8; ++i) load_piece(i);
    advance();

    // ---- epilogue: bias, ReLU, one rounding.  acc[i][k][4 g + j]: token 32 k + l % 32, latent 64 h + 16 i + 4 g + j
    if (p.bias && !bias_dma) {
      __syncthreads();
      if (threadIdx.x < BM) {
        const int64_t m = m0 + threadIdx.x;
        bias[tile * BM + threadIdx.x] = m < p.M ? load_scalar(p.bias, p.bias_dtype, m) : 0.f;
      }
      __syncthreads();
    }
    const float* bt = bias + tile * BM + wm * 128 + 64 * h;
    const bool whole = m0 + BM <= p.M && n0 + BN <= p.N;
    char* tile_out = reinterpret_cast<char*>(out + n0 * p.ldo + m0);  // (host: 256 rows are less than 2 GiB)
    const int nleft = (int)min(p.N - n0, (int64_t)BN), mleft = (int)min(p.M - m0, (int64_t)BM);
    auto finish = [&](auto whole_, auto lines_) {
#pragma unroll
      for (int part = 0; part < (int)sizeof(T) / 2; ++part) {  // 128 bytes of every token: 64 or 32 latents of each half
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          u32x4 c[8];
#pragma unroll
          for (int e = 0; e < 16 / (int)sizeof(T) * 2; ++e) {  // groups of four latents
            const int i = part * 2 + e / 4, g = e % 4;
            const float4 b = *reinterpret_cast<const float4*>(bt + 16 * i + 4 * g);
            const f32x16& a = acc[i][k];
            float v[4] = {a[4 * g] + b.x, a[4 * g + 1] + b.y, a[4 * g + 2] + b.z, a[4 * g + 3] + b.w};
            if (RELU) {
#pragma unroll
              for (int q = 0; q < 4; ++q) v[q] = __builtin_elementwise_maximum(v[q], 0.f);
            }
            if constexpr (sizeof(T) == 2) {
              c[e / 2][e % 2 * 2] = pack2(v[0], v[1]);
              c[e / 2][e % 2 * 2 + 1] = pack2(v[2], v[3]);
            } else {
#pragma unroll
              for (int q = 0; q < 4; ++q) c[e][q] = __float_as_uint(v[q]);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
          lines_of(c);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int s = 0; s < 8; ++s) {
            const int n = 32 * k + 16 * (s >> 2) + (s & 3), m = part * 32;  // how far this line is from the lane's first one
            T* to = reinterpret_cast<T*>(tile_out + (uint32_t)(n * (int)p.ldo + m) * (uint32_t)sizeof(T) + lane_out);
            if (decltype(whole_)::value) {
              store_row16<decltype(lines_)::value>(to, c[s]);
            } else if (nl + n < nleft) {
              if (ml + m + VEC <= mleft) {
                store_row16<false>(to, c[s]);
              } else {
                T e[VEC];
                const u32x4 w = c[s];
                __builtin_memcpy(e, &w, 16);
#pragma unroll
                for (int q = 0; q < VEC; ++q)
                  if (ml + m + q < mleft) to[q] = e[q];
              }
            }
          }
        }
      }
    };
    if (whole && p.lines) finish(std::true_type{}, std::true_type{});
    else if (whole) finish(std::true_type{}, std::false_type{});
    else finish(std::false_type{}, std::false_type{});
    pos += nbx;
    if (pos >= xstop) break;
    place(pos, m0, n0);
    if (!whole) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (fewer stores than the next stage's wait counts on)
    tile = tile == 2 ? 0 : tile + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (no DMA is under way when the LDS goes to another workgroup)
}

}  // namespace
}  // namespace clt

using namespace clt;

static int64_t padded(int64_t K) { return (K + KPAD - 1) / KPAD * KPAD; }
static constexpr int64_t MAX_VALUES = (1ll << 35) - 2048;  // of a matrix with its padding (eight a thread, threads in 32 bits)
template <typename T>
static void launch_quantize(const T* x, int64_t ldx, int64_t R, int64_t K, uint8_t* codes, uint8_t* scales, hipStream_t st) {
  const int64_t lpr = padded(K) / 8, total = R * lpr;
  const bool flat = K == padded(K) && (ldx == K || R == 1);
  hipLaunchKernelGGL((flat ? mxfp4_quantize_kernel<T, true> : mxfp4_quantize_kernel<T, false>), dim3((unsigned)((total + 255) / 256)),
                     dim3(256), 0, st, x, ldx, K, total, lpr, (uint32_t*)codes, scales);
}
template <typename T>
static void launch_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t R, int64_t K, T* out, hipStream_t st) {
  const int64_t lpr = padded(K) / 8, total = R * lpr;
  hipLaunchKernelGGL((K == padded(K) ? mxfp4_dequantize_kernel<T, true> : mxfp4_dequantize_kernel<T, false>),
                     dim3((unsigned)((total + 255) / 256)), dim3(256), 0, st, (const uint32_t*)codes, scales, K, total, lpr, out);
}

extern "C" int clt_mxfp4_quantize(const void* x, int x_dtype, int64_t ldx, int64_t R, int64_t K, uint8_t* codes,
                                  uint8_t* scales, clt_stream_t stream) {
  CLT_CHECK_ARG(x && codes && scales, "clt_mxfp4_quantize: null pointer");
  CLT_CHECK_ARG(valid_dtype(x_dtype), "clt_mxfp4_quantize: dtype");
  CLT_CHECK_ARG(R > 0 && K > 0 && K < (1ll << 30) && R <= MAX_VALUES / padded(K) && ldx >= 0, "clt_mxfp4_quantize: bad sizes");
  CLT_CHECK_ARG(aligned16(codes) && !((uintptr_t)scales & 3) && !((uintptr_t)x & (dtype_size(x_dtype) - 1)),
                "clt_mxfp4_quantize: misaligned pointer");
  if (x_dtype == CLT_BF16) launch_quantize((const bf16_t*)x, ldx, R, K, codes, scales, (hipStream_t)stream);
  else launch_quantize((const float*)x, ldx, R, K, codes, scales, (hipStream_t)stream);
  CLT_CHECK_LAUNCH("clt_mxfp4_quantize");
  return CLT_OK;
}

extern "C" int clt_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t R, int64_t K, void* out,
                                    int out_dtype, clt_stream_t stream) {
  CLT_CHECK_ARG(codes && scales && out, "clt_mxfp4_dequantize: null pointer");
  CLT_CHECK_ARG(valid_dtype(out_dtype), "clt_mxfp4_dequantize: dtype");
  CLT_CHECK_ARG(R > 0 && K > 0 && K < (1ll << 30) && R <= MAX_VALUES / padded(K), "clt_mxfp4_dequantize: bad sizes");
  CLT_CHECK_ARG(aligned16(codes) && !((uintptr_t)scales & 3) && !((uintptr_t)out & (dtype_size(out_dtype) - 1)),
                "clt_mxfp4_dequantize: misaligned pointer");
  if (out_dtype == CLT_BF16) launch_dequantize(codes, scales, R, K, (bf16_t*)out, (hipStream_t)stream);
  else launch_dequantize(codes, scales, R, K, (float*)out, (hipStream_t)stream);
  CLT_CHECK_LAUNCH("clt_mxfp4_dequantize");
  return CLT_OK;
}

namespace {

constexpr int FEW_LDS = 64 * 1024;
int few_lds(int kp) { return 16 * (kp / 2 + 16 + kp / 32); }
bool few(int64_t N, int64_t K) { return N <= 16 && K < 16384 && few_lds((int)((K + KPAD - 1) / KPAD * KPAD)) <= FEW_LDS; }
// So few values of x that every workgroup of the product quantises them for itself (one launch / two, us; x 16384 latents: 1 x
// 768: 5.6 / 7.2, 8 x 1024: 7.1 / 7.1, 16 x 768: 7.4 / 7.0), in rows so short that reading W does not wait (1 x 4096: 17 / 10).
bool few_raw(int64_t N, int64_t K) { return N * K <= 8192 && K <= 1024 && few(N, K); }

int whole_lines(const void* out, int out_dtype, int64_t ldo) {
  return (((uintptr_t)out | (uintptr_t)(ldo * (int64_t)dtype_size(out_dtype))) & 127) == 0;
}

// Which kernel takes a problem of codes (tokens x latents x columns, bf16 output, us):
//   few / 64 x 64:      1 x 98304 x 64: 5.1 / 6.0     1 x 98304 x 768: 8.9 / 10.1     1 x 43579 x 768: 6.4 / 5.4
//   split / 64 x 64:    128 x 2048 x 4096: 4.8 / 7.6     128 x 2048 x 2048: 4.2 / 5.5    200 x 1500 x 2048: 5.6 / 5.4
//   64 x 64 / 128 x 128:    950 x 6151 x 768: 9.9 / 10.9    509 x 6151 x 4096: 21.0 / 18.4    64 x 98304 x 768: 11.4 / 14.7
//                           64 x 131072 x 4096: 80 / 70
//   256 x 256 / the others: 950 x 16384 x 768: 13.8 / 16.9   2048 x 6151 x 2048: 23.7 / 26.7   2048 x 10000 x 768: 27.3 / 23.0
//                           200 x 43579 x 4096: 34 / 42
enum Route { FEW, SPLIT, TILE64, TILE128, BIG };
int64_t tiles(int64_t M, int64_t N, int64_t side) { return (M + side - 1) / side * ((N + side - 1) / side); }
Route route_of(int64_t N, int64_t M, int64_t K, int out_dtype, int64_t ldo) {
  const int64_t t32 = tiles(M, N, 32), t64 = tiles(M, N, 64), t256 = tiles(M, N, 256);
  const int64_t stages = (padded(K) + 255) / 256, rounds = (t256 + 255) / 256;  // (of one tile a CU)
  if (few(N, K) && t64 > 1200) return FEW;
  if (stages >= 4 && t32 <= 32 * stages && t32 <= 512) return SPLIT;
  if (t256 >= 192 && M > 128 && N > 128 && (10 * t256 >= 7 * 256 * rounds || stages >= 10) &&
      256 * ldo * (int64_t)dtype_size(out_dtype) < (1ll << 31))
    return BIG;
  return t64 * (5 + stages) <= (N <= 64 ? 40000 : 15000) ? TILE64 : TILE128;
}

template <typename XT, typename T>
void launch_few(const LinearArgs& a, const XT* x, int64_t ldx, int64_t K, hipStream_t st) {
  const int64_t blocks = (a.M + 127) / 128;  // two groups of 16 rows and more a wave
  const dim3 grid((unsigned)(blocks < 1024 ? blocks : 1024));
  hipLaunchKernelGGL((mxfp4_few_kernel<XT, T>), grid, dim3(256), few_lds(a.kp), st, a, x, ldx, (int)K);
}

int check_linear(const char* name, const void* w_codes, const void* w_scales, const void* bias, int bias_dtype, int64_t N,
                 int64_t M, int64_t K, const void* out, int out_dtype, int64_t ldo) {
  CLT_CHECK_ARG(w_codes && w_scales && out, "%s: null pointer", name);
  CLT_CHECK_ARG(valid_dtype(out_dtype) && (!bias || valid_dtype(bias_dtype)), "%s: dtype", name);
  CLT_CHECK_ARG(N > 0 && M > 0 && K > 0 && ldo >= M, "%s: bad sizes", name);
  CLT_UNSUPPORTED(N < (1ll << 31) && M < (1ll << 31) && K < (1ll << 24), "%s: N and M below 2^31, K below 2^24", name);
  CLT_CHECK_ARG(aligned16(w_codes) && !((uintptr_t)w_scales & 3) && !((uintptr_t)out & (dtype_size(out_dtype) - 1)) &&
                    !(bias && ((uintptr_t)bias & (dtype_size(bias_dtype) - 1))),
                "%s: misaligned pointer", name);
  return CLT_OK;
}

}  // namespace

extern "C" int clt_mxfp4_linear(const uint8_t* x_codes, const uint8_t* x_scales, const uint8_t* w_codes,
                                const uint8_t* w_scales, const void* bias, int bias_dtype, int64_t N, int64_t M, int64_t K,
                                int relu, void* out, int out_dtype, int64_t ldo, clt_stream_t stream) {
  const int rc = check_linear("clt_mxfp4_linear", w_codes, w_scales, bias, bias_dtype, N, M, K, out, out_dtype, ldo);
  if (rc) return rc;
  CLT_CHECK_ARG(x_codes && x_scales, "clt_mxfp4_linear: null pointer");
  CLT_CHECK_ARG(aligned16(x_codes) && !((uintptr_t)x_scales & 3), "clt_mxfp4_linear: misaligned pointer");
  LinearArgs a{x_codes, x_scales, w_codes, w_scales, bias, out, N, M, ldo, (int)padded(K), bias_dtype, relu, whole_lines(out, out_dtype, ldo)};
  const auto st = (hipStream_t)stream;
  const bool b16 = out_dtype == CLT_BF16;
  CLT_UNSUPPORTED(tiles(M, N, 128) < (1ll << 24), "clt_mxfp4_linear: fewer than 2^24 tiles of 128 x 128");  // (threads of a launch: 32 bits)
  switch (route_of(N, M, K, out_dtype, ldo)) {
    case FEW:
      if (b16) launch_few<uint8_t, bf16_t>(a, nullptr, 0, K, st);
      else launch_few<uint8_t, float>(a, nullptr, 0, K, st);
      break;
    case SPLIT:
      hipLaunchKernelGGL((b16 ? mxfp4_split_kernel<bf16_t> : mxfp4_split_kernel<float>), dim3((unsigned)tiles(M, N, 32)), dim3(256), 0, st, a);
      break;
    case BIG: {
      const auto kernel = b16 ? (relu ? mxfp4_big_kernel<bf16_t, true> : mxfp4_big_kernel<bf16_t, false>)
                              : (relu ? mxfp4_big_kernel<float, true> : mxfp4_big_kernel<float, false>);
      hipLaunchKernelGGL(kernel, dim3(256), dim3(512), 0, st, a);
      break;
    }
    case TILE64:
      hipLaunchKernelGGL((b16 ? mxfp4_tile_kernel<bf16_t, 1> : mxfp4_tile_kernel<float, 1>), dim3((unsigned)tiles(M, N, 64)), dim3(256), 0, st, a);
      break;
    case TILE128:
      hipLaunchKernelGGL((b16 ? mxfp4_tile_kernel<bf16_t, 2> : mxfp4_tile_kernel<float, 2>), dim3((unsigned)tiles(M, N, 128)), dim3(256), 0, st, a);
      break;
  }
  CLT_CHECK_LAUNCH("clt_mxfp4_linear");
  return CLT_OK;
}

extern "C" const char* clt_mxfp4_linear_route(int64_t N, int64_t M, int64_t K, int out_dtype, int64_t ldo) {
  static const char* const names[] = {"few", "split", "64 x 64", "128 x 128", "256 x 256"};
  const bool taken = N > 0 && M > 0 && K > 0 && ldo >= M && valid_dtype(out_dtype) && N < (1ll << 31) && M < (1ll << 31) &&
                     K < (1ll << 24) && tiles(M, N, 128) < (1ll << 24);
  return taken ? names[route_of(N, M, K, out_dtype, ldo)] : "";
}

extern "C" size_t clt_mxfp4_linear_x_workspace_bytes(int64_t N, int64_t K) {
  if (N <= 0 || K <= 0 || few_raw(N, K)) return 0;
  return align_up((size_t)N * (padded(K) / 2), 16) + (size_t)N * (padded(K) / 32);
}

extern "C" int clt_mxfp4_linear_x(const void* x, int x_dtype, int64_t ldx, const uint8_t* w_codes, const uint8_t* w_scales,
                                  const void* bias, int bias_dtype, int64_t N, int64_t M, int64_t K, int relu, void* out,
                                  int out_dtype, int64_t ldo, void* workspace, size_t workspace_bytes, clt_stream_t stream) {
  const int rc = check_linear("clt_mxfp4_linear_x", w_codes, w_scales, bias, bias_dtype, N, M, K, out, out_dtype, ldo);
  if (rc) return rc;
  CLT_CHECK_ARG(x && valid_dtype(x_dtype) && ldx >= 0 && !((uintptr_t)x & (dtype_size(x_dtype) - 1)),
                "clt_mxfp4_linear_x: x is null or misaligned, or its dtype or stride is wrong");
  if (few_raw(N, K)) {
    const LinearArgs a{nullptr, nullptr, w_codes, w_scales, bias, out, N, M, ldo, (int)padded(K), bias_dtype, relu, whole_lines(out, out_dtype, ldo)};
    const hipStream_t st = (hipStream_t)stream;
    if (x_dtype == CLT_BF16) {
      if (out_dtype == CLT_BF16) launch_few<bf16_t, bf16_t>(a, (const bf16_t*)x, ldx, K, st);
      else launch_few<bf16_t, float>(a, (const bf16_t*)x, ldx, K, st);
    } else {
      if (out_dtype == CLT_BF16) launch_few<float, bf16_t>(a, (const float*)x, ldx, K, st);
      else launch_few<float, float>(a, (const float*)x, ldx, K, st);
    }
    CLT_CHECK_LAUNCH("clt_mxfp4_linear_x");
    return CLT_OK;
  }
  const size_t need = clt_mxfp4_linear_x_workspace_bytes(N, K);
  if (!workspace || workspace_bytes < need) {
    set_error("clt_mxfp4_linear_x: workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : 0, need);
    return CLT_ERR_WORKSPACE;
  }
  uint8_t* codes = (uint8_t*)workspace;
  uint8_t* scales = codes + align_up((size_t)N * (padded(K) / 2), 16);
  const int q = clt_mxfp4_quantize(x, x_dtype, ldx, N, K, codes, scales, stream);
  return q ? q : clt_mxfp4_linear(codes, scales, w_codes, w_scales, bias, bias_dtype, N, M, K, relu, out, out_dtype, ldo, stream);
}
