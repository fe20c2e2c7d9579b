// The vocabulary projection of a decode step with a 4-bit weight (nvfp4.cuh): logits[t, v] = bf16(g * sum_k x[t, k] * e2m1(c[v, k]) * e4m3(s[v, k / 16])),
// FP32 accumulation, for up to 8 NT rows (NT of 1 to 4), the final RMSNorm fused on the input as in lm_head.cuh (the norm's output is rounded to BF16 by definition).
//
// The weight is read once: 0.5625 bytes an element instead of 2 (350 MB for 151,936 x 4096: 53 us at the measured copy rate), so an SM has to take in
// some 43 weights a clock. A code becomes binary16 by the conversion instruction (two codes each), times its block's scale by one packed multiplication:
// exact, since e2m1 * e4m3 has 6 significant bits. The products and sums are those of mma.sync m16n8k16 (binary16 in, FP32 accumulate), 16 vocabulary rows to a
// warp; measured alone, conversion, scale and mma together take in 57 weights a clock and SM, bit operations in the place of the conversion 34. (The operands go from registers to the
// mma: on tcgen05 they pass through shared or tensor memory, which costs more than the products of so few rows: lm_head_nvfp4_batch.cuh.) A warp's loads run ahead in registers.
//
// x is BF16 and the mma wants binary16 on both sides. A row of x is multiplied by the power of two that brings its largest magnitude to 2^14 .. 2^15 (taken out
// again behind the sum); BF16 values down to 2^-31 of the largest are then exact in binary16, subnormals included. Where some x is not (or is infinite or NaN),
// every block sees it and takes the rows the slow way, in FP64 on the CUDA cores, whose range holds every product.
//
// A row's sum is (q0 + q1) + (q2 + q3) over four quarters of the hidden dimension, each in order: the same additions whether a warp walks the whole row or, for the tiles left over after
// the last full round, four warps take a quarter each.
#pragma once
#include "common.cuh"
#include "nvfp4.cuh"

namespace lm {

constexpr int kH4Threads = 512;
constexpr int kH4Warps = kH4Threads / 32;
constexpr int kH4Rows = 8;                   // rows of x to an mma (its n dimension)
constexpr int kH4MaxNT = 4;
constexpr int kH4Tile = 16;                  // vocabulary rows per warp tile (the m dimension)
constexpr int kH4Step = 256;                 // columns per step: 32 bytes of codes per thread and row, a whole 128-byte line per row and quad
constexpr int kH4MaxHidden = 12736;
constexpr int kH4MaxSteps = (kH4MaxHidden + kH4Step - 1) / kH4Step;

struct Head4Dev {
  const uint16_t* x; int64_t x_stride; int rows;
  const uint8_t* codes; int64_t codes_stride; const uint8_t* scales; int64_t scales_stride; const float* scale;
  int hidden; int vocab;
  const uint16_t* gamma; float eps; int one_plus;
  uint16_t* logits; int64_t logits_stride;
};

// A row of x in shared memory: per step of 256 columns 512 bytes, in them the 16-byte chunk c of quad thread t (columns 64 t + 8 c ..) at 16 (4 c + t), so that the four
// threads of a quad read 64 bytes in a row; rows 64 bytes out of step with each other's banks.
__host__ __device__ inline int head4_steps(int hidden) { return (hidden + kH4Step - 1) / kH4Step; }
__host__ __device__ inline int head4_row_bytes(int hidden) { return head4_steps(hidden) * 512 + 64; }
__host__ __device__ inline size_t head4_smem_bytes(int hidden, int nt) { return static_cast<size_t>(kH4Rows * nt) * head4_row_bytes(hidden); }
__device__ __forceinline__ int head4_x_offset(int k) { return (k >> 8) * 512 + ((((k >> 3) & 7) << 2) + ((k >> 6) & 3)) * 16 + (k & 7) * 2; }

__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t f16x2_mul(uint32_t a, uint32_t b) { uint32_t r; asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint16_t f32_to_f16(float f) { uint16_t r; asm("cvt.rn.f16.f32 %0, %1;" : "=h"(r) : "f"(f)); return r; }
__device__ __forceinline__ uint16_t f32_to_bf16(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }

// 2^shift in two factors (each a normal binary32 for every shift that occurs), and a BF16 value times that as binary16; false where it is not exact (a product that vanishes in
// binary32 included). The first product is exact, the second one rounds at most where it falls below the normal numbers.
struct Scale4 { float a, b; };
__device__ __forceinline__ Scale4 scale_of(int shift) {
  const int h = shift / 2;
  return Scale4{__int_as_float((127 + h) << 23), __int_as_float((127 + shift - h) << 23)};
}
__device__ __forceinline__ bool scaled_f16(float x, Scale4 s, uint16_t* h) {
  const float f = __fmul_rn(__fmul_rn(x, s.a), s.b);
  *h = f32_to_f16(f);
  return f16_lo(*h) == f && (f != 0.0f || x == 0.0f);
}
// The power of two that brings a row whose largest magnitude has these BF16 bits to 2^14 .. 2^15.
__device__ __forceinline__ int shift_of(uint32_t top) { return top == 0u ? 0 : 141 - static_cast<int>(max(top >> 7, 1u)); }
__device__ __forceinline__ uint32_t top_of(const uint32_t (&w)[4]) {         // the largest magnitude of eight BF16
  uint32_t m = 0u;
#pragma unroll
  for (int e = 0; e < 4; e++) m = max(m, max(w[e] & 0x7FFFu, (w[e] >> 16) & 0x7FFFu));
  return m;
}
// Eight BF16 from any address.
__device__ __forceinline__ void load8(const uint16_t* p, uint32_t (&w)[4]) {
  if ((reinterpret_cast<uintptr_t>(p) & 15u) == 0) { const uint4 q = *reinterpret_cast<const uint4*>(p); w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w; }
  else {
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = static_cast<uint32_t>(p[2 * e]) | static_cast<uint32_t>(p[2 * e + 1]) << 16;
  }
}
// Eight elements of a row normalised: bf16(x * inv_rms * scale).
__device__ __forceinline__ void normalise8(uint32_t (&w)[4], const uint32_t (&gamma)[4], float inv_rms, int one_plus) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float g0 = bf16_lo(gamma[e]), g1 = bf16_hi(gamma[e]);
    const float lo = __fmul_rn(__fmul_rn(bf16_lo(w[e]), inv_rms), one_plus ? __fadd_rn(1.0f, g0) : g0), hi = __fmul_rn(__fmul_rn(bf16_hi(w[e]), inv_rms), one_plus ? __fadd_rn(1.0f, g1) : g1);
    w[e] = static_cast<uint32_t>(f32_to_bf16(lo)) | static_cast<uint32_t>(f32_to_bf16(hi)) << 16;
  }
}
__device__ __forceinline__ float squares8(const uint32_t (&w)[4]) {
  float ss = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; e++) { ss = __fmaf_rn(bf16_lo(w[e]), bf16_lo(w[e]), ss); ss = __fmaf_rn(bf16_hi(w[e]), bf16_hi(w[e]), ss); }
  return ss;
}
__device__ __forceinline__ bool scaled8(uint32_t (&w)[4], Scale4 s) {         // in place, BF16 to binary16; false where one is not exact
  bool exact = true;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    uint16_t lo, hi;
    exact &= scaled_f16(bf16_lo(w[e]), s, &lo); exact &= scaled_f16(bf16_hi(w[e]), s, &hi);
    w[e] = static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 16;
  }
  return exact;
}
// The sum of a logit times g and 2^-n (n: what x was multiplied by), in binary64 so that no intermediate leaves the range.
__device__ __forceinline__ float head4_finish(double sum, float g, int n) {
  return __double2float_rn(sum * static_cast<double>(g) * __hiloint2double((1023 - n) << 20, 0));
}

// 16 vocabulary rows' codes and scales of a step, a thread's part: 64 columns of rows g and g + 8.
struct Piece4 { uint4 a[2], b[2]; uint32_t fa, fb; };

// kAhead: steps whose loads are in registers or on the way.
template <int NT, int kAhead>
static __global__ void __launch_bounds__(kH4Threads, 1) lm_head_nvfp4_kernel(Head4Dev P) {
  constexpr int kRows = kH4Rows * NT;
  extern __shared__ __align__(16) unsigned char smem_raw[];                 // [kRows][row_bytes]
  __shared__ union {
    struct { float sum[kRows * kH4MaxSteps]; uint32_t top[kRows * kH4MaxSteps]; } x;       // while x is prepared
    float part[4][3][32][4 * NT];                                           // later: quarters of the tiles left over
  } s_u;
  float* s_sum = s_u.x.sum;
  uint32_t* s_top = s_u.x.top;
  __shared__ float s_factor[kRows];                                         // 1 / rms, then g * 2^-shift
  __shared__ int s_shift[kRows];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int H = P.hidden, row_bytes = head4_row_bytes(H), steps = head4_steps(H);
  const int gq = lane >> 2, t = lane & 3;
  // A round: a tile to a warp. What is left over after the full rounds takes another one, or (two quarters of a round or less) four warps to a tile.
  const int n_tiles = (P.vocab + kH4Tile - 1) / kH4Tile, all_warps = gridDim.x * kH4Warps, left = n_tiles % all_warps, full = left > all_warps / 2 ? n_tiles : n_tiles - left;
  after_predecessor();
  const float g = __ldg(P.scale);
  auto fetch = [&](Piece4& p, int tile, int s) {
    const int v0 = tile * kH4Tile + gq, k = s * kH4Step + 64 * t;
    if (k < H) {                                                            // (H is a multiple of 64: all of a thread's 64 columns or none)
      const int64_t ra = min(v0, P.vocab - 1), rb = min(v0 + 8, P.vocab - 1);          // (rows beyond the vocabulary: loaded again, never stored)
      const uint8_t *ca = P.codes + ra * P.codes_stride + (k >> 1), *cb = P.codes + rb * P.codes_stride + (k >> 1);
      p.a[0] = __ldcs(reinterpret_cast<const uint4*>(ca)); p.a[1] = __ldcs(reinterpret_cast<const uint4*>(ca) + 1);
      p.b[0] = __ldcs(reinterpret_cast<const uint4*>(cb)); p.b[1] = __ldcs(reinterpret_cast<const uint4*>(cb) + 1);
      p.fa = __ldg(reinterpret_cast<const uint32_t*>(P.scales + ra * P.scales_stride + (k >> 4))); p.fb = __ldg(reinterpret_cast<const uint32_t*>(P.scales + rb * P.scales_stride + (k >> 4)));
    } else { p.a[0] = p.a[1] = p.b[0] = p.b[1] = make_uint4(0u, 0u, 0u, 0u); p.fa = p.fb = 0u; }
  };
  // ---- the first steps' loads; they arrive while x is prepared
  Piece4 ring[kAhead];
  int load_tile = blockIdx.x * kH4Warps + warp, load_step = 0;
  auto fetch_next = [&](Piece4& p) {
    if (load_tile >= full) return;
    fetch(p, load_tile, load_step);
    if (++load_step == steps) { load_step = 0; load_tile += all_warps; }
  };
#pragma unroll
  for (int d = 0; d < kAhead - 1; d++) fetch_next(ring[d]);
  // ---- the rows of x: normalised if a norm is fused, scaled, binary16. `per` warps to a row, 256 columns at a time, a lane a chunk of 8. (Rows of the mma beyond P.rows hold whatever
  // is there: they reach no other row's sums.)
  int per = kH4Warps;
  while (per > 1 && per * P.rows > kH4Warps) per >>= 1;
  const int my_row = warp / per, my_part = warp % per, row_step = kH4Warps / per;
  constexpr int kTogether = 4;                                              // chunks a lane has under way
  auto chunk = [&](int row, int s) -> uint4* { return reinterpret_cast<uint4*>(smem_raw + row * row_bytes + s * 512 + ((((lane & 7) << 2) + (lane >> 3)) << 4)); };
  // f(row, s, w): the chunk's eight elements, changed or not; the chunks of a batch are asked for together
  auto each = [&](auto get, auto f) {
    for (int row = my_row; row < P.rows; row += row_step) {
      for (int base = my_part; base < steps; base += kTogether * per) {
        uint32_t w[kTogether][4];
#pragma unroll
        for (int u = 0; u < kTogether; u++) if (base + u * per < steps) get(row, base + u * per, w[u]);
#pragma unroll
        for (int u = 0; u < kTogether; u++) if (base + u * per < steps) f(row, base + u * per, w[u]);
      }
    }
  };
  auto from_memory = [&](int row, int s, uint32_t (&w)[4]) {
    const int k = s * kH4Step + lane * 8;
    w[0] = w[1] = w[2] = w[3] = 0u;
    if (k < H) load8(P.x + row * P.x_stride + k, w);
  };
  auto from_shared = [&](int row, int s, uint32_t (&w)[4]) { const uint4 q = *chunk(row, s); w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w; };
  auto to_shared = [&](int row, int s, const uint32_t (&w)[4]) { *chunk(row, s) = make_uint4(w[0], w[1], w[2], w[3]); };
  auto mean_square = [&](int row) {
    float ss = 0.0f;
    for (int s = 0; s < steps; s++) ss += s_sum[row * kH4MaxSteps + s];
    return __frsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(H)), P.eps));
  };
  each(from_memory, [&](int row, int s, uint32_t (&w)[4]) {
    to_shared(row, s, w);
    if (P.gamma) {
      float ss = squares8(w);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
      if (lane == 0) s_sum[row * kH4MaxSteps + s] = ss;
    } else { const uint32_t m = warp_max_u32(top_of(w)); if (lane == 0) s_top[row * kH4MaxSteps + s] = m; }
  });
  if (P.gamma) {
    __syncthreads();
    float inv_rms = 0.0f;
    int known = -1;
    each(from_shared, [&](int row, int s, uint32_t (&w)[4]) {
      if (row != known) { inv_rms = mean_square(row); known = row; }
      const int k = s * kH4Step + lane * 8;
      if (k < H) {
        uint32_t gamma[4];
        load8(P.gamma + k, gamma);
        normalise8(w, gamma, inv_rms, P.one_plus);
        to_shared(row, s, w);
      }
      const uint32_t m = warp_max_u32(top_of(w));
      if (lane == 0) s_top[row * kH4MaxSteps + s] = m;
    });
  }
  __syncthreads();
  bool plain = true, bad = false;                                           // plain: every g * 2^-shift is a normal binary32, with room for the sum
  if (tid < P.rows) {
    uint32_t m = 0u;
    for (int s = 0; s < steps; s++) m = max(m, s_top[tid * kH4MaxSteps + s]);
    bad = m >= 0x7F80u;                                                     // an infinity or a NaN
    const int shift = shift_of(m);
    const double f = static_cast<double>(g) * __hiloint2double((1023 - shift) << 20, 0);
    plain = fabs(f) >= 0x1p-100 && fabs(f) <= 0x1p80;
    s_shift[tid] = shift; s_factor[tid] = static_cast<float>(f);
  }
  plain = __syncthreads_and(plain);
  each(from_shared, [&](int row, int s, uint32_t (&w)[4]) { bad |= !scaled8(w, scale_of(s_shift[row])); to_shared(row, s, w); });
  if (__syncthreads_or(bad)) {
    // some x is no binary16 after the scaling: FP64 on the values themselves
    for (int v = blockIdx.x * kH4Warps + warp; v < P.vocab; v += all_warps) {
      for (int r = 0; r < P.rows; r++) {
        const float inv_rms = P.gamma ? mean_square(r) : 1.0f;
        double sum = 0.0;
        for (int k = lane * 8; k < H; k += 256) {
          uint32_t x[4], h[4];
          load8(P.x + r * P.x_stride + k, x);
          if (P.gamma) {
            uint32_t gamma[4];
            load8(P.gamma + k, gamma);
            normalise8(x, gamma, inv_rms, P.one_plus);
          }
          e2m1_to_f16(*reinterpret_cast<const uint32_t*>(P.codes + static_cast<int64_t>(v) * P.codes_stride + (k >> 1)), h);
          const float sc = e4m3_value(P.scales[static_cast<int64_t>(v) * P.scales_stride + (k >> 4)]);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            sum += static_cast<double>(bf16_lo(x[e])) * static_cast<double>(f16_lo(h[e]) * sc);
            sum += static_cast<double>(bf16_hi(x[e])) * static_cast<double>(f16_hi(h[e]) * sc);
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
        if (lane == 0) P.logits[r * P.logits_stride + v] = f32_to_bf16(head4_finish(sum, g, 0));
      }
    }
    return;
  }
  // ---- products
  const unsigned char* xrow = smem_raw + gq * row_bytes + t * 16;           // row gq of every eight of x, this thread's chunks
  auto multiply = [&](const Piece4& p, int s, float (&c)[NT][4]) {
    const uint32_t wa[8] = {p.a[0].x, p.a[0].y, p.a[0].z, p.a[0].w, p.a[1].x, p.a[1].y, p.a[1].z, p.a[1].w};
    const uint32_t wb[8] = {p.b[0].x, p.b[0].y, p.b[0].z, p.b[0].w, p.b[1].x, p.b[1].y, p.b[1].z, p.b[1].w};
#pragma unroll
    for (int h = 0; h < 2; h++) {                                           // two scales each
      const uint32_t pa = e4m3_to_f16(p.fa >> (16 * h)), pb = e4m3_to_f16(p.fb >> (16 * h));
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int j = 4 * h + q;
        const uint32_t sa = __byte_perm(pa, 0u, q < 2 ? 0x1010 : 0x3232), sb = __byte_perm(pb, 0u, q < 2 ? 0x1010 : 0x3232);
        uint32_t ha[4], hb[4];
        e2m1_to_f16(wa[j], ha);
        e2m1_to_f16(wb[j], hb);
#pragma unroll
        for (int e = 0; e < 4; e++) { ha[e] = f16x2_mul(ha[e], sa); hb[e] = f16x2_mul(hb[e], sb); }
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const uint4 x = *reinterpret_cast<const uint4*>(xrow + n * kH4Rows * row_bytes + s * 512 + j * 64);
          mma_f16_16816(c[n], ha[0], hb[0], ha[1], hb[1], x.x, x.y);
          mma_f16_16816(c[n], ha[2], hb[2], ha[3], hb[3], x.z, x.w);
        }
      }
    }
  };
  auto store = [&](int tile, const float (&c)[NT][4]) {
    const int v = tile * kH4Tile + gq;
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int r = n * kH4Rows + 2 * t + (e & 1), vv = v + (e >> 1) * 8;
        if (r < P.rows && vv < P.vocab) P.logits[r * P.logits_stride + vv] = f32_to_bf16(plain ? __fmul_rn(c[n][e], s_factor[r]) : head4_finish(c[n][e], g, s_shift[r]));
      }
    }
  };
  float c[NT][4], lo[NT][4], hi[NT][4];                                     // a quarter's sum; the first two quarters'; the third's
#pragma unroll
  for (int n = 0; n < NT; n++) {
#pragma unroll
    for (int e = 0; e < 4; e++) c[n][e] = lo[n][e] = hi[n][e] = 0.0f;
  }
  int s = 0, q = 0, bound = steps / 4;                                      // (a quarter: steps q * steps / 4 .. (q + 1) * steps / 4)
  for (int tile = blockIdx.x * kH4Warps + warp; tile < full;) {
#pragma unroll
    for (int d = 0; d < kAhead; d++) {
      if (tile >= full) break;
      fetch_next(ring[(d + kAhead - 1) % kAhead]);
      while (s == bound) {                                                  // the end of a quarter
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            if (q < 2) lo[n][e] = q == 0 ? c[n][e] : __fadd_rn(lo[n][e], c[n][e]); else hi[n][e] = c[n][e];
            c[n][e] = 0.0f;
          }
        }
        q++;
        bound = (q + 1) * steps / 4;
      }
      multiply(ring[d], s, c);
      if (++s == steps) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
          for (int e = 0; e < 4; e++) { c[n][e] = __fadd_rn(lo[n][e], __fadd_rn(hi[n][e], c[n][e])); lo[n][e] = hi[n][e] = 0.0f; }
        }
        store(tile, c);
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
          for (int e = 0; e < 4; e++) c[n][e] = 0.0f;
        }
        s = 0; q = 0; bound = steps / 4;
        tile += all_warps;
      }
    }
  }
  // ---- the tiles left over: four warps to a tile, a quarter each
  const int group = warp >> 2, part = warp & 3, s0 = part * steps / 4, s1 = (part + 1) * steps / 4;
  for (int tile = full + blockIdx.x + group * gridDim.x; tile < n_tiles; tile += 4 * gridDim.x) {
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int e = 0; e < 4; e++) c[n][e] = 0.0f;
    }
    for (int b = s0; b < s1; b += kAhead) {
#pragma unroll
      for (int d = 0; d < kAhead; d++) if (b + d < s1) fetch(ring[d], tile, b + d);
#pragma unroll
      for (int d = 0; d < kAhead; d++) if (b + d < s1) multiply(ring[d], b + d, c);
    }
    if (part > 0) {
#pragma unroll
      for (int n = 0; n < NT; n++) *reinterpret_cast<float4*>(&s_u.part[group][part - 1][lane][4 * n]) = make_float4(c[n][0], c[n][1], c[n][2], c[n][3]);
    }
    asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory");
    if (part == 0) {
#pragma unroll
      for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int e = 0; e < 4; e++)
          c[n][e] = __fadd_rn(__fadd_rn(c[n][e], s_u.part[group][0][lane][4 * n + e]), __fadd_rn(s_u.part[group][1][lane][4 * n + e], s_u.part[group][2][lane][4 * n + e]));
      }
      store(tile, c);
    }
    asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory");
  }
}

}  // namespace lm
