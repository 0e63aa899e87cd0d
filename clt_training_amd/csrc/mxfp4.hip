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


// Large problems.  A workgroup of four waves computes 256 latents x 128 tokens, a wave 128 x 64 of them (4 x 2 tiles of
// 32 x 32, 128 accumulators), so that two workgroups share a CU: the waits, the first loads and the stores of one run
// beside the matrix instructions of the other.
//
// Per stage of 128 columns both operands come as rows of 64 bytes by LDS-DMA (24 pieces of 16 rows = 1 KiB, six per wave)
// into a ring of three slots, two stages ahead; one barrier per stage.  A lane of a piece fetches the 16-byte chunk c =
// (lane % 4) ^ (row / 4 % 4) of its row: the fragment reads (lane l: row l % 32, chunk 2 t + l / 32) then touch every bank once.
// The scales of four stages are 16 bytes of a row: one DMA for 64 rows, then four registers per fragment row.
// The finished tile goes through the ring's LDS once, so that a store instruction writes rows of 256 bytes.
constexpr int TM = 256, TN = 128, KS = 128;
constexpr int STAGE_W = TM * 64, STAGE_BYTES = (TM + TN) * 64, NSLOT = 3;
constexpr int SCALE_OFF = NSLOT * STAGE_BYTES, TILE_LDS = SCALE_OFF + (TM + TN) * 16;
constexpr int PITCH = 272;                       // bytes between the token rows of the transposed tile (256 of data)
constexpr int BIAS_OFF = 4 * 32 * PITCH;
constexpr int PANEL = 16;                        // token tiles that share their operand rows in an XCD's L2
static_assert(BIAS_OFF + TM * 4 <= TILE_LDS && 2 * TILE_LDS <= 160 * 1024, "LDS");

typedef __attribute__((address_space(3))) void* lds_ptr_t;

// LDS[lds_dst + 16 * lane] = *(sbase + voff)
__device__ __forceinline__ void dma16(const uint8_t* sbase, uint32_t voff, uint32_t lds_dst) {
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %3\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %2\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(voff), "s"(sbase), "s"(lds_dst)
      : "memory");
}

template <int T>  // half of a stage: 64 columns
__device__ __forceinline__ f32x16 mfma4s(const i32x4& a, const i32x4& b, const f32x16& c, int sa, int sb) {
  const i32x8 A = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8 B = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, c, 4, 4, 2 * T, sa, 2 * T, sb);
}

template <typename T>
__global__ __launch_bounds__(256, 2) void mxfp4_tile_kernel(const LinearArgs p) {
  __shared__ __attribute__((aligned(1024))) char lds[TILE_LDS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5, wm = wave >> 1, wn = wave & 1;

  // ---- tile: an XCD (workgroup id % 8) owns a contiguous range of positions; a panel of token tiles runs through all latents
  const int64_t nlt = (p.M + TM - 1) / TM, ntt = (p.N + TN - 1) / TN, ntiles = nlt * ntt;
  const int64_t xg = blockIdx.x & 7, q = ntiles >> 3, rest = ntiles & 7;
  const int64_t pos = xg * q + min(xg, rest) + (blockIdx.x >> 3);
  const int64_t panel = pos / (nlt * PANEL), in = pos - panel * nlt * PANEL;
  const int64_t width = min((int64_t)PANEL, ntt - panel * PANEL);
  const int64_t m0 = in / width * TM, n0 = (panel * PANEL + in % width) * TN;

  // ---- loader: this wave's pieces of a stage (four of W, two of x), rows past the end read the last one again
  const int rowb = p.kp / 2, sb = p.kp / 32, nst = p.kp / KS;
  const uint8_t* wbase = p.wc + m0 * rowb;
  const uint8_t* xbase = p.xc + n0 * rowb;
  const int wleft = (int)min((int64_t)TM, p.M - m0) - 1, xleft = (int)min((int64_t)TN, p.N - n0) - 1;
  uint32_t woff[4], xoff[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (4 * wave + i) * 16 + (lane >> 2);
    woff[i] = (uint32_t)min(row, wleft) * rowb + (((lane & 3) ^ ((row >> 2) & 3)) << 4);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = (2 * wave + i) * 16 + (lane >> 2);
    xoff[i] = (uint32_t)min(row, xleft) * rowb + (((lane & 3) ^ ((row >> 2) & 3)) << 4);
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds;
  auto load_stage = [&](int s, int slot) {
    const uint32_t d = lds0 + slot * STAGE_BYTES;
#pragma unroll
    for (int i = 0; i < 4; ++i) dma16(wbase + (int64_t)s * 64, woff[i], d + (4 * wave + i) * 1024);
#pragma unroll
    for (int i = 0; i < 2; ++i) dma16(xbase + (int64_t)s * 64, xoff[i], d + STAGE_W + (2 * wave + i) * 1024);
  };
  // The scales of a row end behind 16 bytes of the last chunk: what follows is the next row's.  Only behind the last row
  // there is nothing; there the 16 bytes are taken from further left (`back`) and moved into place when they are read.
  const uint8_t* wsc = p.ws + m0 * sb;
  const uint8_t* xsc = p.xs + n0 * sb;
  const int64_t wend = (p.M - m0) * sb - 16, xend = (p.N - n0) * sb - 16;  // (last position that 16 bytes may be read from)
  auto load_scales = [&](int c) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int piece = wave + 4 * i;  // 0 .. 3: W, 4 .. 5: x
      if (piece >= 6) break;
      const bool w = piece < 4;
      const int row = min((w ? piece : piece - 4) * 64 + lane, w ? wleft : xleft);
      const int64_t off = min((int64_t)row * sb + 16 * c, w ? wend : xend);
      // (off may be negative: the base lies inside the array, 16 bytes before its end are inside it too)
      const uint8_t* base = w ? wsc : xsc;
      const uint8_t* low = base + min((int64_t)0, w ? wend : xend);
      dma16(low, (uint32_t)(base + off - low), lds0 + SCALE_OFF + piece * 1024);
    }
  };
  auto read_scales = [&](int row, int c, int left, int64_t end, int lds_row) {
    i32x4 v = *reinterpret_cast<const i32x4*>(lds + SCALE_OFF + lds_row * 16);
    const int64_t over = (int64_t)min(row, left) * sb + 16 * c - end;
    const int back = over > 0 ? (int)over >> 2 : 0;  // registers
    if (__builtin_amdgcn_ballot_w64(back != 0)) {
      i32x4 u;
      u[0] = back == 0 ? v[0] : back == 1 ? v[1] : back == 2 ? v[2] : v[3];
      u[1] = back == 0 ? v[1] : back == 1 ? v[2] : v[3];
      u[2] = back == 0 ? v[2] : v[3];
      u[3] = v[3];
      v = u;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (int)((uint32_t)v[j] >> (8 * h));  // bytes 0 and 2: this lane's blocks of the two halves
    return v;
  };

  f32x16 acc[4][2] = {};
  i32x4 sw[4], sx[2];
  uint32_t fa[2], fb[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint32_t o = r32 * 64 + (((2 * t + h) ^ ((r32 >> 2) & 3)) << 4);
    fa[t] = o + wm * 128 * 64;
    fb[t] = o + STAGE_W + wn * 64 * 64;
  }

  load_scales(0);
  load_stage(0, 0);
  if (nst > 1) load_stage(1, 1);
  int slot = 0;
  for (int s0 = 0; s0 < nst; s0 += 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int s = s0 + j;
      if (s >= nst) break;
      // stage s is there when at most the six pieces of stage s + 1 are on their way
      if (s + 1 < nst) asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (s + 2 < nst) {
        if (j == 2) load_scales((s + 2) >> 2);
        load_stage(s + 2, slot == 0 ? 2 : slot - 1);  // the slot of stage s - 1: every wave is past it
      }
      if (j == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sw[i] = read_scales(wm * 128 + i * 32 + r32, s0 >> 2, wleft, wend, wm * 128 + i * 32 + r32);
#pragma unroll
        for (int i = 0; i < 2; ++i) sx[i] = read_scales(wn * 64 + i * 32 + r32, s0 >> 2, xleft, xend, TM + wn * 64 + i * 32 + r32);
      }
      const char* st = lds + slot * STAGE_BYTES;
      i32x4 A[2][4], B[2][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) A[t][i] = *reinterpret_cast<const i32x4*>(st + fa[t] + i * 2048);
#pragma unroll
        for (int i = 0; i < 2; ++i) B[t][i] = *reinterpret_cast<const i32x4*>(st + fb[t] + i * 2048);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) acc[i][k] = mfma4s<0>(A[0][i], B[0][k], acc[i][k], sw[i][j], sx[k][j]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) acc[i][k] = mfma4s<1>(A[1][i], B[1][k], acc[i][k], sw[i][j], sx[k][j]);
      slot = slot == 2 ? 0 : slot + 1;
    }
  }

  // ---- epilogue: bias, ReLU, one rounding; lane l of D holds token l % 32, latents 8 (i / 4) + 4 h + i % 4
  __syncthreads();  // (the ring is free)
  float* bias = reinterpret_cast<float*>(lds + BIAS_OFF);
  {
    const int64_t m = m0 + threadIdx.x;
    bias[threadIdx.x] = p.bias && m < p.M ? load_scalar(p.bias, p.bias_dtype, m) : 0.f;
  }
  __syncthreads();
  char* mine = lds + wave * 32 * PITCH;
  constexpr int LAT = 256 / sizeof(T);            // latents in a row of the transposed tile
  constexpr int RT = LAT / 32, VEC = 16 / sizeof(T);
  T* out = reinterpret_cast<T*>(p.out);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int part = 0; part < 4 / RT; ++part) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int lat = (part * RT + i) * 32 + 8 * g + 4 * h;
          const float4 b = *reinterpret_cast<const float4*>(bias + wm * 128 + lat);
          float v[4] = {acc[part * RT + i][k][4 * g] + b.x, acc[part * RT + i][k][4 * g + 1] + b.y,
                        acc[part * RT + i][k][4 * g + 2] + b.z, acc[part * RT + i][k][4 * g + 3] + b.w};
          if (p.relu) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];
          }
          char* to = mine + r32 * PITCH + (i * 32 + 8 * g + 4 * h) * sizeof(T);
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
      const int64_t m = m0 + wm * 128 + part * LAT + (lane & 15) * VEC;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int tok = 4 * i + (lane >> 4);
        const uint4 w = *reinterpret_cast<const uint4*>(mine + tok * PITCH + (lane & 15) * 16);
        const int64_t n = n0 + wn * 64 + k * 32 + tok;
        if (n >= p.N) continue;
        T* to = out + n * p.ldo + m;
        struct __attribute__((packed, aligned(sizeof(T)))) Row {
          uint4 w;
        };
        if (m + VEC <= p.M) {
          reinterpret_cast<Row*>(to)->w = w;
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
  const int64_t tiles = (M + TM - 1) / TM * ((N + TN - 1) / TN);
  if (N >= 16 && M >= 16 && tiles >= 64 && tiles < (1ll << 31)) {
    if (out_dtype == CLT_BF16)
      hipLaunchKernelGGL(mxfp4_tile_kernel<bf16_t>, dim3((unsigned)tiles), dim3(256), 0, (hipStream_t)stream, a);
    else
      hipLaunchKernelGGL(mxfp4_tile_kernel<float>, dim3((unsigned)tiles), dim3(256), 0, (hipStream_t)stream, a);
    CLT_CHECK_LAUNCH("clt_mxfp4_linear");
    return CLT_OK;
  }
  const dim3 grid((unsigned)((M + 31) / 32), (unsigned)((N + 31) / 32));
  if (out_dtype == CLT_BF16)
    hipLaunchKernelGGL(mxfp4_linear_kernel<bf16_t>, grid, dim3(64), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(mxfp4_linear_kernel<float>, grid, dim3(64), 0, (hipStream_t)stream, a);
  CLT_CHECK_LAUNCH("clt_mxfp4_linear");
  return CLT_OK;
}
