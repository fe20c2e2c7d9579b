// The microscaled 4-bit format (NVFP4) and its conversions.
//
// A matrix [rows, cols], cols a multiple of 16, is held as codes (two to a byte, the even column in the low nibble), one e4m3 scale for
// every 16 columns of a row, and one binary32 scale g for all: value = e2m1(code) * e4m3(scale) * g. e2m1 has the magnitudes 0, 1/2, 1,
// 3/2, 2, 3, 4, 6 and a sign; e2m1 * e4m3 has at most 6 significant bits and lies within 2^-10 .. 2688, so it is exact in binary16 and in binary32.
//
// Quantisation: s = e4m3(a / (6 g)) with a the block's largest magnitude, code = e2m1(x / (s g)); both quotients are the real ones, rounded once to
// nearest, ties to even, and saturate (448, 6). So the codes are a property of the input and not of the arithmetic: any correct program finds the same.
// The kernel forms quotients in binary32 with a reciprocal that is a little too small and one that is a little too large, by 2^-21 = 8 * 2^-24: the product s * g, the reciprocal (__fdividef: two units in the
// last place), its shift and the product with x are off by (1 + 4 + 1 + 1) * 2^-24 at most, so the real quotient lies between. Both are rounded with the conversion instructions; where both give the same code it is the real quotient's, otherwise one fused multiply-add tells on which side of x the exact product border * s * g (31 bits)
// lies. (That is not rare: with BF16 inputs and a scale formed from one of them, quotients fall on borders but for the scale's own rounding; comparing in binary64 then took 1.6 of 1.8 ms for
// 151,936 x 4096.) Scales beyond 2^-100 .. 2^100: all by comparisons in binary64.
// Bound by HBM, each a pass over the matrix, a thread a block of 16. 151,936 x 4096 in BF16 (L2 cold): quantised under a given scale 277 to 289 us (1.6 GB, 5.5 to 5.8 TB/s), the scale found first 480 to 490 (L2
// does not keep the matrix between the passes: 2.8 GB), the values written as binary32 500 (2.8 GB, 5.7 TB/s). In FP32 442 (2.8 GB, 6.4 TB/s) and 802 (5.3 GB, 6.6 TB/s).
#pragma once
#include "common.cuh"

namespace lm {

constexpr int kFp4Block = 16;                // columns that share a scale
constexpr float kFp4Largest = 2688.0f;       // 6 * 448
constexpr uint32_t kE4m3Nan = 0x7Fu;

// Eight codes of a word (ascending nibbles) as binary16 pairs. All four results have to be used: with the last two dropped, nvcc 12.9 took the first two from the wrong bytes.
__device__ __forceinline__ void e2m1_to_f16(uint32_t w, uint32_t (&r)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(w));
}
// ... four codes, of the lower two bytes.
__device__ __forceinline__ void e2m1_to_f16_low(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b8 a, b;\n\tmov.b16 {a, b}, %2;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "h"(static_cast<uint16_t>(w)));
}
// The codes nearest to eight binary32 (ties to even, saturating), ascending nibbles.
__device__ __forceinline__ uint32_t f32_to_e2m1(const float2 (&v)[4]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\tcvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\tmov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r) : "f"(v[0].x), "f"(v[0].y), "f"(v[1].x), "f"(v[1].y), "f"(v[2].x), "f"(v[2].y), "f"(v[3].x), "f"(v[3].y));
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

// 16 columns of a row as they lie in memory, and as binary32.
template <bool F32> struct Sixteen {
  uint32_t w[F32 ? 16 : 8];
  __device__ __forceinline__ void load(const QuantDev& P, long long row, int block, bool aligned) {
    const unsigned char* p = static_cast<const unsigned char*>(P.x) + (row * P.row_stride + block * kFp4Block) * (F32 ? 4 : 2);
    if (aligned) {
#pragma unroll
      for (int q = 0; q < (F32 ? 4 : 2); q++) { const uint4 u = *(reinterpret_cast<const uint4*>(p) + q); w[4 * q] = u.x; w[4 * q + 1] = u.y; w[4 * q + 2] = u.z; w[4 * q + 3] = u.w; }
    } else if (F32) {
#pragma unroll
      for (int e = 0; e < 16; e++) w[e % (F32 ? 16 : 8)] = reinterpret_cast<const uint32_t*>(p)[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) { const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + 2 * e; w[e] = static_cast<uint32_t>(h[0]) | static_cast<uint32_t>(h[1]) << 16; }
    }
  }
  __device__ __forceinline__ float2 pair(int i) const {                      // columns 2 i, 2 i + 1
    return F32 ? make_float2(__uint_as_float(w[(2 * i) % (F32 ? 16 : 8)]), __uint_as_float(w[(2 * i + 1) % (F32 ? 16 : 8)])) : make_float2(bf16_lo(w[i % 8]), bf16_hi(w[i % 8]));
  }
  __device__ __forceinline__ uint32_t top() const {                          // the largest magnitude's bits, infinities and NaN included
    uint32_t m = 0u;
    if (F32) {
#pragma unroll
      for (int e = 0; e < 16; e++) m = max(m, w[e % (F32 ? 16 : 8)] & 0x7FFFFFFFu);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) m = __vmaxu2(m, w[e] & 0x7FFF7FFFu);
      m = max(m << 16, m & 0x7FFF0000u);
    }
    return m;
  }
  __device__ __forceinline__ uint32_t signs(int half) const {                // the sign bits of 8 columns as those of codes
    uint32_t r = 0u;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint32_t bit = F32 ? w[(8 * half + e) % (F32 ? 16 : 8)] >> 31 : (w[(4 * half + e / 2) % 8] >> (e & 1 ? 31 : 15)) & 1u;
      r |= bit << (4 * e + 3);
    }
    return r;
  }
};

constexpr int kQuantThreads = 256;
// A thread's items one after the other, `step` apart, as row and place in the row (no division on the way).
struct Stride2 {
  long long row, drow; int at, dat, per_row;
  __device__ __forceinline__ Stride2(long long first, long long step, int per_row_) : row(first / per_row_), drow(step / per_row_), at(static_cast<int>(first % per_row_)), dat(static_cast<int>(step % per_row_)), per_row(per_row_) {}
  __device__ __forceinline__ void next() { row += drow; at += dat; if (at >= per_row) { at -= per_row; row++; } }
};

// The largest finite magnitude, as bits (which order like the values), into *amax (zero before).
template <bool F32>
static __global__ void __launch_bounds__(kQuantThreads) nvfp4_amax_kernel(QuantDev P) {
  const bool aligned = ((reinterpret_cast<uintptr_t>(P.x) | static_cast<uintptr_t>(P.row_stride * (F32 ? 4 : 2))) & 15u) == 0;
  constexpr int kTogether = F32 ? 2 : 4;
  uint32_t best = 0u;
  Stride2 i(static_cast<long long>(blockIdx.x) * kQuantThreads + threadIdx.x, static_cast<long long>(gridDim.x) * kQuantThreads, P.cols / kFp4Block);
  while (i.row < P.rows) {
    Sixteen<F32> v[kTogether];
#pragma unroll
    for (int u = 0; u < kTogether; u++) {
      if (i.row < P.rows) v[u].load(P, i.row, i.at, aligned);
      else {
#pragma unroll
        for (int e = 0; e < (F32 ? 16 : 8); e++) v[u].w[e] = 0u;
      }
      i.next();
    }
#pragma unroll
    for (int u = 0; u < kTogether; u++) {
      const uint32_t m = v[u].top();
      if (m < 0x7F800000u) best = max(best, m);
      else {                                                                // something infinite or NaN: the others
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float2 p = v[u].pair(e);
          const uint32_t a = __float_as_uint(p.x) & 0x7FFFFFFFu, b = __float_as_uint(p.y) & 0x7FFFFFFFu;
          if (a < 0x7F800000u) best = max(best, a);
          if (b < 0x7F800000u) best = max(best, b);
        }
      }
    }
  }
  best = warp_max_u32(best);
  if ((threadIdx.x & 31) == 0 && best) atomicMax(P.amax, best);
}

template <bool F32>
static __global__ void __launch_bounds__(kQuantThreads) nvfp4_quantize_kernel(QuantDev P) {
  const bool aligned = ((reinterpret_cast<uintptr_t>(P.x) | static_cast<uintptr_t>(P.row_stride * (F32 ? 4 : 2))) & 15u) == 0;
  const bool aligned_codes = ((reinterpret_cast<uintptr_t>(P.codes) | static_cast<uintptr_t>(P.codes_stride)) & 7u) == 0;
  const float g = quant_scale(P);
  const bool usable = g >= 0x1p-126f && g < INFINITY;                       // (a scale that is no positive normal number: every block's scale is NaN)
  const bool plain = g >= 0x1p-100f && g <= 0x1p100f;                       // binary32 quotients are as close as said above
  const float kLess = 1.0f - 0x1p-21f, kMore = 1.0f + 0x1p-21f;
  const float inv6 = __fdiv_rn(1.0f, __fmul_rn(6.0f, g)), inv6_less = __fmul_rn(inv6, kLess), inv6_more = __fmul_rn(inv6, kMore);
  auto one = [&](const Sixteen<F32>& v, long long row, int block) {
    const uint32_t top = v.top();
    uint32_t s = kE4m3Nan;
    uint2 codes = make_uint2(0u, 0u);
    if (usable && top < 0x7F800000u) {                                      // (an infinity or a NaN in the block: its scale is NaN)
      const float a = __uint_as_float(top);
      const uint32_t two = f32_to_e4m3(__fmul_rn(a, inv6_less), __fmul_rn(a, inv6_more));
      s = two & 0xFFu;
      if (!plain) s = exact_scale(a, g);
      else if (s != two >> 8) {                                             // next to the border between two scales
        const float d = __fmaf_rn(-3.0f * (e4m3_value(s) + e4m3_value(s + 1u)), g, a);     // (the sum and its triple are exact: 8 bits)
        if (d > 0.0f || (d == 0.0f && (s & 1u))) s++;
      }
      const float sv = e4m3_value(s);
      bool again = !plain;
      if (s == 0u) { codes = make_uint2(v.signs(0), v.signs(1)); again = false; }
      else if (plain) {
        const float inv = __fdividef(1.0f, __fmul_rn(sv, g)), less = __fmul_rn(inv, kLess), more = __fmul_rn(inv, kMore);
        uint2 up;
        float2 q[4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
          for (int e = 0; e < 4; e++) q[e] = __fmul2_rn(v.pair(4 * h + e), make_float2(less, less));
          (h ? codes.y : codes.x) = f32_to_e2m1(q);
#pragma unroll
          for (int e = 0; e < 4; e++) q[e] = __fmul2_rn(v.pair(4 * h + e), make_float2(more, more));
          (h ? up.y : up.x) = f32_to_e2m1(q);
        }
        // codes next to a border: both candidates are neighbours
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint32_t& c = h ? codes.y : codes.x;
          uint32_t differ = c ^ (h ? up.y : up.x);
          while (differ) {
            const int e = (__ffs(static_cast<int>(differ)) - 1) >> 2;       // column 8 h + e
            const uint32_t m = (c >> (4 * e)) & 7u;                         // the lower magnitude
            const int64_t at = row * P.row_stride + block * kFp4Block + 8 * h + e;
            const float x = F32 ? static_cast<const float*>(P.x)[at] : __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(P.x)[at]) << 16);
            const float d = __fmaf_rn(-0.5f * (e2m1_value(m) + e2m1_value(m + 1u)) * sv, g, fabsf(x));
            if (d > 0.0f || (d == 0.0f && (m & 1u))) c += 1u << (4 * e);
            differ &= ~(15u << (4 * e));
          }
        }
      }
      if (again) {
        const double unit = static_cast<double>(sv) * static_cast<double>(g);
        codes = make_uint2(v.signs(0), v.signs(1));
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float2 p = v.pair(e);
          const uint32_t c = exact_code(fabsf(p.x), unit) | exact_code(fabsf(p.y), unit) << 4;
          if (e < 4) codes.x |= c << (8 * e); else codes.y |= c << (8 * (e - 4));
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
  };
  constexpr int kTogether = F32 ? 1 : 2;
  Stride2 i(static_cast<long long>(blockIdx.x) * kQuantThreads + threadIdx.x, static_cast<long long>(gridDim.x) * kQuantThreads, P.cols / kFp4Block);
  while (i.row < P.rows) {
    Sixteen<F32> v[kTogether];
    long long row[kTogether];
    int at[kTogether];
#pragma unroll
    for (int u = 0; u < kTogether; u++) {
      row[u] = i.row; at[u] = i.at;
      if (i.row < P.rows) v[u].load(P, i.row, i.at, aligned);
      i.next();
    }
#pragma unroll
    for (int u = 0; u < kTogether; u++) if (row[u] < P.rows) one(v[u], row[u], at[u]);
  }
  if (P.find && blockIdx.x == 0 && threadIdx.x == 0) *P.scale = g;
}

struct DequantDev {
  const uint8_t* codes; int64_t codes_stride; const uint8_t* scales; int64_t scales_stride; const float* scale;
  long long rows; int cols; float* out; int64_t out_stride;
};

// One thread: 4 values (a warp writes 512 bytes in a row) from two bytes of codes, several of these at a time.
static __global__ void __launch_bounds__(kQuantThreads) nvfp4_dequantize_kernel(DequantDev P) {
  constexpr int kTogether = 8;
  const float g = __ldg(P.scale);
  const bool aligned = ((reinterpret_cast<uintptr_t>(P.codes) | static_cast<uintptr_t>(P.codes_stride)) & 1u) == 0;
  const bool aligned_out = ((reinterpret_cast<uintptr_t>(P.out) | static_cast<uintptr_t>(P.out_stride * 4)) & 15u) == 0;
  Stride2 i(static_cast<long long>(blockIdx.x) * kQuantThreads + threadIdx.x, static_cast<long long>(gridDim.x) * kQuantThreads, P.cols / 4), o = i;
  while (i.row < P.rows) {
    uint32_t c[kTogether], s[kTogether];
#pragma unroll
    for (int u = 0; u < kTogether; u++) {
      c[u] = s[u] = 0u;
      if (i.row < P.rows) {
        const uint8_t* p = P.codes + i.row * P.codes_stride + i.at * 2;
        c[u] = aligned ? *reinterpret_cast<const uint16_t*>(p) : static_cast<uint32_t>(p[0]) | static_cast<uint32_t>(p[1]) << 8;
        s[u] = P.scales[i.row * P.scales_stride + (i.at >> 2)];
      }
      i.next();
    }
#pragma unroll
    for (int u = 0; u < kTogether; u++) {
      if (o.row < P.rows) {
        uint32_t h[2];
        e2m1_to_f16_low(c[u], h[0], h[1]);
        const uint32_t sc = __byte_perm(e4m3_to_f16(s[u]), 0u, 0x1010);
        asm("mul.rn.f16x2 %0, %0, %2;\n\tmul.rn.f16x2 %1, %1, %2;" : "+r"(h[0]), "+r"(h[1]) : "r"(sc));      // (exact)
        const float4 v = make_float4(__fmul_rn(f16_lo(h[0]), g), __fmul_rn(f16_hi(h[0]), g), __fmul_rn(f16_lo(h[1]), g), __fmul_rn(f16_hi(h[1]), g));
        float* out = P.out + o.row * P.out_stride + o.at * 4;
        if (aligned_out) __stcs(reinterpret_cast<float4*>(out), v);
        else { out[0] = v.x; out[1] = v.y; out[2] = v.z; out[3] = v.w; }
      }
      o.next();
    }
  }
}

}  // namespace lm
