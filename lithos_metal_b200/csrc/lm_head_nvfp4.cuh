// The vocabulary projection of a decode step with a 4-bit weight (nvfp4.cuh): logits[t, v] = bf16(g * sum_k x[t, k] * e2m1(c[v, k]) * e4m3(s[v, k / 16])),
// FP32 accumulation, for up to 8 rows, the final RMSNorm fused on the input as in lm_head.cuh (the norm's output is rounded to BF16 by definition).
//
// The weight is read once: 0.5625 bytes an element instead of 2 (350 MB for 151,936 x 4096: 53 us at the measured copy rate), so an SM has to take in
// some 43 weights a clock. A code becomes binary16 by the conversion instruction (two codes each), times its block's scale by one packed multiplication:
// exact, since e2m1 * e4m3 has 6 significant bits. The products and sums are those of mma.sync m16n8k16 (binary16 in, FP32 accumulate), 16 vocabulary rows to a
// warp; measured alone, conversion, scale and mma together take in 57 weights a clock and SM, bit operations in the place of the conversion 34.
//
// x is BF16 and the mma wants binary16 on both sides. A row of x is multiplied by the power of two that brings its largest magnitude to 2^14 .. 2^15 (taken out
// again behind the sum); BF16 values down to 2^-31 of the largest are then exact in binary16, subnormals included. Where some x is not (or is infinite or NaN),
// every block sees it and takes the rows the slow way, in FP64 on the CUDA cores, whose range holds every product.
#pragma once
#include "common.cuh"
#include "nvfp4.cuh"

namespace lm {

constexpr int kH4Threads = 256;
constexpr int kH4Warps = kH4Threads / 32;
constexpr int kH4Rows = 8;                   // rows of x (the n dimension of the mma)
constexpr int kH4Tile = 16;                  // vocabulary rows per warp tile (the m dimension)
constexpr int kH4Step = 256;                 // columns per step: 32 bytes of codes per thread and row, a whole 128-byte line per row and quad
constexpr int kH4Unroll = 4;                 // steps whose loads are in flight together: a batch
constexpr int kH4MaxBatches = 13;            // batches of the longest row that fits (12,736 columns)
constexpr int kH4MaxHidden = 12736;

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
__host__ __device__ inline size_t head4_smem_bytes(int hidden) { return static_cast<size_t>(kH4Rows) * head4_row_bytes(hidden); }
__device__ __forceinline__ int head4_x_offset(int k) { return (k >> 8) * 512 + ((((k >> 3) & 7) << 2) + ((k >> 6) & 3)) * 16 + (k & 7) * 2; }

__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t f16x2_mul(uint32_t a, uint32_t b) { uint32_t r; asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint16_t f32_to_f16(float f) { uint16_t r; asm("cvt.rn.f16.f32 %0, %1;" : "=h"(r) : "f"(f)); return r; }
__device__ __forceinline__ uint16_t f32_to_bf16(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }

// A BF16 value times 2^shift as binary16; false where that is not exact (a product that vanishes in binary32 included).
__device__ __forceinline__ bool scaled_f16(uint16_t bf16, int shift, uint16_t* h) {
  const float f = ldexpf(__uint_as_float(static_cast<uint32_t>(bf16) << 16), shift);
  *h = f32_to_f16(f);
  return f16_lo(*h) == f && (f != 0.0f || (bf16 & 0x7FFFu) == 0u);
}
// The sum of a logit times g and 2^-n (n: what x was multiplied by), in binary64 so that no intermediate leaves the range.
__device__ __forceinline__ float head4_finish(double sum, float g, int n) {
  return __double2float_rn(sum * static_cast<double>(g) * __hiloint2double((1023 - n) << 20, 0));
}

static __global__ void __launch_bounds__(kH4Threads, 2) lm_head_nvfp4_kernel(Head4Dev P) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ float s_part[kH4Rows][kH4Warps];
  __shared__ uint32_t s_max[kH4Rows][kH4Warps];
  __shared__ float part[kH4MaxBatches][32][4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int H = P.hidden, row_bytes = head4_row_bytes(H), steps = head4_steps(H), padded = steps * kH4Step;
  after_predecessor();
  // ---- the rows of x: normalised if a norm is fused, scaled, binary16
  float inv_rms[kH4Rows];
  if (P.gamma) {
    float ss[kH4Rows];
#pragma unroll
    for (int r = 0; r < kH4Rows; r++) ss[r] = 0.0f;
    for (int k = tid; k < H; k += kH4Threads) {
#pragma unroll
      for (int r = 0; r < kH4Rows; r++) if (r < P.rows) { const float v = __uint_as_float(static_cast<uint32_t>(P.x[r * P.x_stride + k]) << 16); ss[r] = __fmaf_rn(v, v, ss[r]); }
    }
#pragma unroll
    for (int r = 0; r < kH4Rows; r++) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss[r] += __shfl_xor_sync(kFull, ss[r], o);
      if (lane == 0) s_part[r][warp] = ss[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kH4Rows; r++) {
      float s = 0.0f;
#pragma unroll
      for (int q = 0; q < kH4Warps; q++) s += s_part[r][q];
      inv_rms[r] = __frsqrt_rn(__fadd_rn(__fdiv_rn(s, static_cast<float>(H)), P.eps));
    }
  }
  // column k of the rows, as the BF16 values that are multiplied
  auto column = [&](int k, uint16_t (&x)[kH4Rows]) {
#pragma unroll
    for (int r = 0; r < kH4Rows; r++) x[r] = (r < P.rows && k < H) ? P.x[r * P.x_stride + k] : static_cast<uint16_t>(0u);
    if (P.gamma && k < H) {
      const float gm = __uint_as_float(static_cast<uint32_t>(P.gamma[k]) << 16), scale = P.one_plus ? __fadd_rn(1.0f, gm) : gm;
#pragma unroll
      for (int r = 0; r < kH4Rows; r++) if (r < P.rows) x[r] = f32_to_bf16(__fmul_rn(__fmul_rn(__uint_as_float(static_cast<uint32_t>(x[r]) << 16), inv_rms[r]), scale));
    }
  };
  uint32_t top[kH4Rows];
#pragma unroll
  for (int r = 0; r < kH4Rows; r++) top[r] = 0u;
  for (int k = tid; k < padded; k += kH4Threads) {
    uint16_t x[kH4Rows];
    column(k, x);
#pragma unroll
    for (int r = 0; r < kH4Rows; r++) { top[r] = max(top[r], static_cast<uint32_t>(x[r]) & 0x7FFFu); *reinterpret_cast<uint16_t*>(smem_raw + r * row_bytes + head4_x_offset(k)) = x[r]; }
  }
#pragma unroll
  for (int r = 0; r < kH4Rows; r++) { const uint32_t m = warp_max_u32(top[r]); if (lane == 0) s_max[r][warp] = m; }
  __syncthreads();
  int shift[kH4Rows];                                                       // x is multiplied by 2^shift
  bool bad = false;
#pragma unroll
  for (int r = 0; r < kH4Rows; r++) {
    uint32_t m = 0u;
#pragma unroll
    for (int q = 0; q < kH4Warps; q++) m = max(m, s_max[r][q]);
    bad |= m >= 0x7F80u;                                                    // an infinity or a NaN
    shift[r] = m == 0u ? 0 : 141 - static_cast<int>(max(m >> 7, 1u));       // (exponent of the largest to 14)
  }
  for (int k = tid; k < padded && !bad; k += kH4Threads) {
#pragma unroll
    for (int r = 0; r < kH4Rows; r++) {
      uint16_t* p = reinterpret_cast<uint16_t*>(smem_raw + r * row_bytes + head4_x_offset(k));
      uint16_t h;
      bad |= !scaled_f16(*p, shift[r], &h);
      *p = h;
    }
  }
  const bool slow = __syncthreads_or(bad);
  const float g = __ldg(P.scale);
  auto put = [&](int r, int v, double sum, int n) { if (r < P.rows && v < P.vocab) P.logits[r * P.logits_stride + v] = f32_to_bf16(head4_finish(sum, g, n)); };
  if (slow) {                                                               // some x is no binary16 after the scaling: BF16 in shared memory, FP64 arithmetic
    for (int k = tid; k < padded; k += kH4Threads) {
      uint16_t x[kH4Rows];
      column(k, x);
#pragma unroll
      for (int r = 0; r < kH4Rows; r++) *reinterpret_cast<uint16_t*>(smem_raw + r * row_bytes + head4_x_offset(k)) = x[r];
    }
    __syncthreads();
    for (int v = blockIdx.x * kH4Warps + warp; v < P.vocab; v += gridDim.x * kH4Warps) {
      double sum[kH4Rows];
#pragma unroll
      for (int r = 0; r < kH4Rows; r++) sum[r] = 0.0;
      for (int w = lane; w < H / 8; w += 32) {
        uint32_t h[4];
        e2m1_to_f16(*reinterpret_cast<const uint32_t*>(P.codes + static_cast<int64_t>(v) * P.codes_stride + w * 4), h);
        const float s = e4m3_value(P.scales[static_cast<int64_t>(v) * P.scales_stride + (w >> 1)]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const double w0 = f16_lo(h[e]) * s, w1 = f16_hi(h[e]) * s;
#pragma unroll
          for (int r = 0; r < kH4Rows; r++) {
            const uint32_t x = *reinterpret_cast<const uint32_t*>(smem_raw + r * row_bytes + head4_x_offset(8 * w + 2 * e));
            sum[r] += static_cast<double>(bf16_lo(x)) * w0;
            sum[r] += static_cast<double>(bf16_hi(x)) * w1;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < kH4Rows; r++) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum[r] += __shfl_xor_sync(kFull, sum[r], o);
        if (lane == 0) put(r, v, sum[r], 0);
      }
    }
    return;
  }
  // ---- the tiles. A tile's sums are formed batch by batch (kH4Unroll steps into a fresh accumulator, then added to the total), the batches in order: the same
  // additions whether one warp walks the whole row or, for the tiles left over after the last full round, the warps of a block take a batch each.
  const int gq = lane >> 2, t = lane & 3;
  const int n_tiles = (P.vocab + kH4Tile - 1) / kH4Tile;
  const int batches = (steps + kH4Unroll - 1) / kH4Unroll;
  const unsigned char* xrow = smem_raw + gq * row_bytes + t * 16;           // row gq of x, this thread's chunks
  auto batch_sum = [&](int tile, int batch, float (&c)[4]) {
    const int v0 = tile * kH4Tile;
    const int64_t ra = min(v0 + gq, P.vocab - 1), rb = min(v0 + gq + 8, P.vocab - 1);      // (rows beyond the vocabulary: loaded again, never stored)
    const int k0 = batch * kH4Unroll * kH4Step + 64 * t;
    const uint8_t *ca = P.codes + ra * P.codes_stride + (k0 >> 1), *cb = P.codes + rb * P.codes_stride + (k0 >> 1);
    const uint8_t *sa = P.scales + ra * P.scales_stride + (k0 >> 4), *sb = P.scales + rb * P.scales_stride + (k0 >> 4);
    uint4 a[kH4Unroll][2], b[kH4Unroll][2];
    uint32_t fa[kH4Unroll], fb[kH4Unroll];
#pragma unroll
    for (int u = 0; u < kH4Unroll; u++) {
      if (k0 + u * kH4Step < H) {                                           // (H is a multiple of 64: all of a thread's 64 columns or none)
        a[u][0] = __ldcs(reinterpret_cast<const uint4*>(ca + u * 128)); a[u][1] = __ldcs(reinterpret_cast<const uint4*>(ca + u * 128) + 1);
        b[u][0] = __ldcs(reinterpret_cast<const uint4*>(cb + u * 128)); b[u][1] = __ldcs(reinterpret_cast<const uint4*>(cb + u * 128) + 1);
        fa[u] = __ldg(reinterpret_cast<const uint32_t*>(sa + u * 16)); fb[u] = __ldg(reinterpret_cast<const uint32_t*>(sb + u * 16));
      } else { a[u][0] = a[u][1] = b[u][0] = b[u][1] = make_uint4(0u, 0u, 0u, 0u); fa[u] = fb[u] = 0u; }
    }
    c[0] = c[1] = c[2] = c[3] = 0.0f;
#pragma unroll
    for (int u = 0; u < kH4Unroll; u++) {
      const int s = batch * kH4Unroll + u;
      if (s >= steps) break;
      const uint32_t wa[8] = {a[u][0].x, a[u][0].y, a[u][0].z, a[u][0].w, a[u][1].x, a[u][1].y, a[u][1].z, a[u][1].w};
      const uint32_t wb[8] = {b[u][0].x, b[u][0].y, b[u][0].z, b[u][0].w, b[u][1].x, b[u][1].y, b[u][1].z, b[u][1].w};
#pragma unroll
      for (int p = 0; p < 2; p++) {                                         // two scales each
        const uint32_t pa = e4m3_to_f16(fa[u] >> (16 * p)), pb = e4m3_to_f16(fb[u] >> (16 * p));
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const int j = 4 * p + q;
          const uint32_t sca = __byte_perm(pa, 0u, q < 2 ? 0x1010 : 0x3232), scb = __byte_perm(pb, 0u, q < 2 ? 0x1010 : 0x3232);
          uint32_t ha[4], hb[4];
          e2m1_to_f16(wa[j], ha);
          e2m1_to_f16(wb[j], hb);
#pragma unroll
          for (int e = 0; e < 4; e++) { ha[e] = f16x2_mul(ha[e], sca); hb[e] = f16x2_mul(hb[e], scb); }
          const uint4 x = *reinterpret_cast<const uint4*>(xrow + s * 512 + j * 64);
          mma_f16_16816(c, ha[0], hb[0], ha[1], hb[1], x.x, x.y);
          mma_f16_16816(c, ha[2], hb[2], ha[3], hb[3], x.z, x.w);
        }
      }
    }
  };
  auto store = [&](int tile, const float (&c)[4]) {
    const int v = tile * kH4Tile + gq;
#pragma unroll
    for (int r = 0; r < kH4Rows; r++) {
      if (r >> 1 == t) { put(r, v, c[r & 1], shift[r]); put(r, v + 8, c[2 + (r & 1)], shift[r]); }
    }
  };
  const int all_warps = gridDim.x * kH4Warps;
  const int full = n_tiles / all_warps * all_warps;
  for (int tile = blockIdx.x * kH4Warps + warp; tile < full; tile += all_warps) {
    float total[4] = {0.0f, 0.0f, 0.0f, 0.0f}, c[4];
    for (int batch = 0; batch < batches; batch++) {
      batch_sum(tile, batch, c);
#pragma unroll
      for (int e = 0; e < 4; e++) total[e] = __fadd_rn(total[e], c[e]);
    }
    store(tile, total);
  }
  for (int tile = full + blockIdx.x; tile < n_tiles; tile += gridDim.x) {
    for (int batch = warp; batch < batches; batch += kH4Warps) {
      float c[4];
      batch_sum(tile, batch, c);
#pragma unroll
      for (int e = 0; e < 4; e++) part[batch][lane][e] = c[e];
    }
    __syncthreads();
    if (warp == 0) {
      float total[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int batch = 0; batch < batches; batch++) {
#pragma unroll
        for (int e = 0; e < 4; e++) total[e] = __fadd_rn(total[e], part[batch][lane][e]);
      }
      store(tile, total);
    }
    __syncthreads();
  }
}

}  // namespace lm
