// The microscaled 4-bit format (NVFP4) and its conversions.
//
// A matrix [rows, cols], cols a multiple of 16, is held as codes (two to a byte, the even column in the low nibble), one e4m3 scale for
// every 16 columns of a row, and one binary32 scale g for all: value = e2m1(code) * e4m3(scale) * g. e2m1 has the magnitudes 0, 1/2, 1,
// 3/2, 2, 3, 4, 6 and a sign; e2m1 * e4m3 has at most 6 significant bits and lies within 2^-10 .. 2688, so it is exact in binary16 and in binary32.
//
// Quantisation: s = e4m3(a / (6 g)) with a the block's largest magnitude, code = e2m1(x / (s g)); both quotients are the real ones, rounded once to
// nearest, ties to even, and saturate (448, 6). So the codes are a property of the input and not of the arithmetic: any correct program finds the same.
// The kernel rounds binary32 quotients a little too small and a little too large (by 2^-21; their error is below 2^-22) with the conversion
// instructions; where both give the same code it is the real quotient's, otherwise the code is found by comparing x with the exact products
// border * s * g in binary64 (31 bits).
#pragma once
#include "common.cuh"

namespace lm {

constexpr int kFp4Block = 16;                // columns that share a scale
constexpr float kFp4Largest = 2688.0f;       // 6 * 448
constexpr uint32_t kE4m3Nan = 0x7Fu;

// Eight codes of a word (ascending nibbles) as binary16 pairs.
__device__ __forceinline__ void e2m1_to_f16(uint32_t w, uint32_t (&r)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(w));
}
// The codes nearest to two binary32 (ties to even, saturating): the first in the low nibble.
__device__ __forceinline__ uint32_t f32_to_e2m1(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\tmov.b32 %0, {t, 0, 0, 0};\n\t}" : "=r"(r) : "f"(lo), "f"(hi));
  return r;
}
// The e4m3 values nearest to two binary32: the first in the low byte.
__device__ __forceinline__ uint32_t f32_to_e4m3(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(lo), "f"(hi));
  return r;
}
// Two e4m3 as a binary16 pair.
__device__ __forceinline__ uint32_t e4m3_to_f16(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(two)));
  return r;
}
__device__ __forceinline__ float f16_lo(uint32_t h) { float f; asm("{\n\t.reg .f16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.f32.f16 %0, a;\n\t}" : "=f"(f) : "r"(h)); return f; }
__device__ __forceinline__ float f16_hi(uint32_t h) { float f; asm("{\n\t.reg .f16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.f32.f16 %0, b;\n\t}" : "=f"(f) : "r"(h)); return f; }
__device__ __forceinline__ float e4m3_value(uint32_t code) { return f16_lo(e4m3_to_f16(code & 0xFFu)); }
__device__ __forceinline__ float e2m1_value(uint32_t magnitude) {            // codes 0 .. 7
  return magnitude < 4u ? 0.5f * static_cast<float>(magnitude) : (magnitude & 1u ? 1.5f : 1.0f) * (magnitude < 6u ? 2.0f : 4.0f);
}

// The code of the e4m3 value nearest to a / (6 g): the number of midpoints between neighbours that lie below (at a tie: where the lower code is odd).
__device__ __noinline__ uint32_t exact_scale(float a, float g) {
  const double ad = static_cast<double>(a), g6 = 6.0 * static_cast<double>(g);
  uint32_t lo = 0u, hi = 126u;                                              // 126: 448
  while (lo < hi) {
    const uint32_t mid = (lo + hi) >> 1;
    const double border = 0.5 * (static_cast<double>(e4m3_value(mid)) + static_cast<double>(e4m3_value(mid + 1u))) * g6;   // (exact: 7 bits times 24)
    if (ad > border || (ad == border && (mid & 1u))) lo = mid + 1u; else hi = mid;
  }
  return lo;
}
// ... of the e2m1 magnitude nearest to ax / unit.
__device__ __noinline__ uint32_t exact_code(float ax, double unit) {
  const double ad = static_cast<double>(ax);
  uint32_t lo = 0u, hi = 7u;
  while (lo < hi) {
    const uint32_t mid = (lo + hi) >> 1;
    const double border = 0.5 * (static_cast<double>(e2m1_value(mid)) + static_cast<double>(e2m1_value(mid + 1u))) * unit;
    if (ad > border || (ad == border && (mid & 1u))) lo = mid + 1u; else hi = mid;
  }
  return lo;
}

struct QuantDev {
  const void* x; int dtype; long long rows; int cols; int64_t row_stride;
  float* scale; uint32_t* amax; int find;    // find: *scale is formed from *amax (and written), otherwise it is given
  uint8_t* codes; int64_t codes_stride;
  uint8_t* scales; int64_t scales_stride;
};

__device__ __forceinline__ float quant_scale(const QuantDev& P) {
  if (!P.find) return __ldg(P.scale);
  const float g = __fdiv_rn(__uint_as_float(*P.amax), kFp4Largest);
  return g >= 0x1p-126f ? g : 1.0f;                                         // (nothing but zeros, or next to nothing)
}

// The 16 columns from `block * 16` on of a row.
template <bool F32>
__device__ __forceinline__ void load16(const QuantDev& P, long long row, int block, bool aligned, float (&v)[16]) {
  if (F32) {
    const float* p = static_cast<const float*>(P.x) + row * P.row_stride + block * kFp4Block;
    if (aligned) {
#pragma unroll
      for (int q = 0; q < 4; q++) { const float4 f = __ldcs(reinterpret_cast<const float4*>(p) + q); v[4 * q] = f.x; v[4 * q + 1] = f.y; v[4 * q + 2] = f.z; v[4 * q + 3] = f.w; }
    } else {
#pragma unroll
      for (int e = 0; e < 16; e++) v[e] = __ldg(p + e);
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(P.x) + row * P.row_stride + block * kFp4Block;
    if (aligned) {
#pragma unroll
      for (int q = 0; q < 2; q++) {
        const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p) + q);
        v[8 * q] = bf16_lo(u.x); v[8 * q + 1] = bf16_hi(u.x); v[8 * q + 2] = bf16_lo(u.y); v[8 * q + 3] = bf16_hi(u.y);
        v[8 * q + 4] = bf16_lo(u.z); v[8 * q + 5] = bf16_hi(u.z); v[8 * q + 6] = bf16_lo(u.w); v[8 * q + 7] = bf16_hi(u.w);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; e++) v[e] = __uint_as_float(static_cast<uint32_t>(__ldg(p + e)) << 16);
    }
  }
}

constexpr int kQuantThreads = 256;

// The largest finite magnitude, as bits (which order like the values), into *amax (zero before).
template <bool F32>
static __global__ void __launch_bounds__(kQuantThreads) nvfp4_amax_kernel(QuantDev P) {
  const int blocks = P.cols / kFp4Block;
  const long long total = P.rows * blocks;
  const bool aligned = ((reinterpret_cast<uintptr_t>(P.x) | static_cast<uintptr_t>(P.row_stride * (F32 ? 4 : 2))) & 15u) == 0;
  uint32_t best = 0u;
  for (long long i = static_cast<long long>(blockIdx.x) * kQuantThreads + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * kQuantThreads) {
    float v[16];
    load16<F32>(P, i / blocks, static_cast<int>(i % blocks), aligned, v);
#pragma unroll
    for (int e = 0; e < 16; e++) { const uint32_t b = __float_as_uint(v[e]) & 0x7FFFFFFFu; if (b < 0x7F800000u) best = max(best, b); }
  }
  best = warp_max_u32(best);
  if ((threadIdx.x & 31) == 0 && best) atomicMax(P.amax, best);
}

template <bool F32>
static __global__ void __launch_bounds__(kQuantThreads) nvfp4_quantize_kernel(QuantDev P) {
  const int blocks = P.cols / kFp4Block;
  const long long total = P.rows * blocks;
  const bool aligned = ((reinterpret_cast<uintptr_t>(P.x) | static_cast<uintptr_t>(P.row_stride * (F32 ? 4 : 2))) & 15u) == 0;
  const bool aligned_codes = ((reinterpret_cast<uintptr_t>(P.codes) | static_cast<uintptr_t>(P.codes_stride)) & 7u) == 0;
  const float g = quant_scale(P);
  const bool usable = g >= 0x1p-126f && g < INFINITY;                       // (a scale that is no positive normal number: every block's scale is NaN)
  const bool plain = g >= 0x1p-100f && g <= 0x1p100f;                       // binary32 quotients are as close as said above
  const float inv6 = __fdiv_rn(1.0f, __fmul_rn(6.0f, g));
  const float kLess = 1.0f - 0x1p-21f, kMore = 1.0f + 0x1p-21f;
  for (long long i = static_cast<long long>(blockIdx.x) * kQuantThreads + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * kQuantThreads) {
    const long long row = i / blocks;
    const int block = static_cast<int>(i % blocks);
    float v[16];
    load16<F32>(P, row, block, aligned, v);
    uint32_t amax = 0u;
#pragma unroll
    for (int e = 0; e < 16; e++) amax = max(amax, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    uint32_t s;
    uint2 codes = make_uint2(0u, 0u);
    if (!usable || amax >= 0x7F800000u) s = kE4m3Nan;                        // an infinity or a NaN in the block
    else {
      const float a = __uint_as_float(amax), t = __fmul_rn(a, inv6);
      const uint32_t two = f32_to_e4m3(__fmul_rn(t, kLess), __fmul_rn(t, kMore));
      s = two & 0xFFu;
      if (!plain || s != two >> 8) s = exact_scale(a, g);
      const float sv = e4m3_value(s);
      bool again = !plain;
      if (s == 0u) {
#pragma unroll
        for (int e = 0; e < 8; e++) { codes.x |= (__float_as_uint(v[e]) >> 31) << (4 * e + 3); codes.y |= (__float_as_uint(v[e + 8]) >> 31) << (4 * e + 3); }
        again = false;
      } else if (plain) {
        const float inv = __fdiv_rn(1.0f, __fmul_rn(sv, g));
        uint2 more = make_uint2(0u, 0u);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float q0 = __fmul_rn(v[2 * e], inv), q1 = __fmul_rn(v[2 * e + 1], inv), q2 = __fmul_rn(v[2 * e + 8], inv), q3 = __fmul_rn(v[2 * e + 9], inv);
          codes.x |= f32_to_e2m1(__fmul_rn(q0, kLess), __fmul_rn(q1, kLess)) << (8 * e); more.x |= f32_to_e2m1(__fmul_rn(q0, kMore), __fmul_rn(q1, kMore)) << (8 * e);
          codes.y |= f32_to_e2m1(__fmul_rn(q2, kLess), __fmul_rn(q3, kLess)) << (8 * e); more.y |= f32_to_e2m1(__fmul_rn(q2, kMore), __fmul_rn(q3, kMore)) << (8 * e);
        }
        again = codes.x != more.x || codes.y != more.y;
      }
      if (again) {
        const double unit = static_cast<double>(sv) * static_cast<double>(g);
        codes = make_uint2(0u, 0u);
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const uint32_t c = exact_code(fabsf(v[e]), unit) | (__float_as_uint(v[e]) >> 31 << 3);
          if (e < 8) codes.x |= c << (4 * e); else codes.y |= c << (4 * (e - 8));
        }
      }
    }
    uint8_t* out = P.codes + row * P.codes_stride + block * 8;
    if (aligned_codes) *reinterpret_cast<uint2*>(out) = codes;
    else {
#pragma unroll
      for (int e = 0; e < 8; e++) out[e] = static_cast<uint8_t>((e < 4 ? codes.x : codes.y) >> (8 * (e & 3)));
    }
    P.scales[row * P.scales_stride + block] = static_cast<uint8_t>(s);
  }
  if (P.find && blockIdx.x == 0 && threadIdx.x == 0) *P.scale = g;
}

struct DequantDev {
  const uint8_t* codes; int64_t codes_stride; const uint8_t* scales; int64_t scales_stride; const float* scale;
  long long rows; int cols; float* out; int64_t out_stride;
};

// One thread: half a block, 8 values (32 bytes) from one word of codes.
static __global__ void __launch_bounds__(kQuantThreads) nvfp4_dequantize_kernel(DequantDev P) {
  const int words = P.cols / 8;
  const long long total = P.rows * words;
  const float g = __ldg(P.scale);
  const bool aligned = ((reinterpret_cast<uintptr_t>(P.codes) | static_cast<uintptr_t>(P.codes_stride)) & 3u) == 0;
  const bool aligned_out = ((reinterpret_cast<uintptr_t>(P.out) | static_cast<uintptr_t>(P.out_stride * 4)) & 15u) == 0;
  for (long long i = static_cast<long long>(blockIdx.x) * kQuantThreads + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * kQuantThreads) {
    const long long row = i / words;
    const int word = static_cast<int>(i % words);
    const uint8_t* c = P.codes + row * P.codes_stride + word * 4;
    const uint32_t w = aligned ? __ldcs(reinterpret_cast<const uint32_t*>(c))
                               : static_cast<uint32_t>(c[0]) | static_cast<uint32_t>(c[1]) << 8 | static_cast<uint32_t>(c[2]) << 16 | static_cast<uint32_t>(c[3]) << 24;
    const float s = e4m3_value(P.scales[row * P.scales_stride + (word >> 1)]);
    uint32_t h[4];
    e2m1_to_f16(w, h);
    float v[8];
#pragma unroll
    for (int q = 0; q < 4; q++) { v[2 * q] = __fmul_rn(__fmul_rn(f16_lo(h[q]), s), g); v[2 * q + 1] = __fmul_rn(__fmul_rn(f16_hi(h[q]), s), g); }
    float* o = P.out + row * P.out_stride + word * 8;
    if (aligned_out) {
      __stcs(reinterpret_cast<float4*>(o), make_float4(v[0], v[1], v[2], v[3]));
      __stcs(reinterpret_cast<float4*>(o) + 1, make_float4(v[4], v[5], v[6], v[7]));
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] = v[e];
    }
  }
}

}  // namespace lm
