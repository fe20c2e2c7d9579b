// The vocabulary projection of a decode step with a 4-bit weight (nvfp4.cuh): logits[t, v] = bf16(g * sum_k x[t, k] * e2m1(c[v, k]) * e4m3(s[v, k / 16])),
// FP32 accumulation, for up to 8 NT rows (NT of 1 or 2), the final RMSNorm fused on the input as in lm_head.cuh (the norm's output is rounded to BF16 by definition).
//
// The weight is read once: 0.5625 bytes an element instead of 2 (350 MB for 151,936 x 4096: 53 us at the measured copy rate), so an SM has to take in
// some 43 weights a clock. A code becomes binary16 by the conversion instruction (two codes each), times its block's scale by one packed multiplication:
// exact, since e2m1 * e4m3 has 6 significant bits. The products and sums are those of mma.sync m16n8k16 (binary16 in, FP32 accumulate), 16 vocabulary rows to a
// warp; measured alone, conversion, scale and mma together take in 57 weights a clock and SM, bit operations in the place of the conversion 34. (The operands go from registers to the
// mma: on tcgen05 they pass through shared or tensor memory, which costs more than the products of so few rows: lm_head_nvfp4_batch.cuh.) A warp's loads run ahead in registers.
//
// The conversion instructions know binary16 only (for BF16, which would hold e2m1 * e4m3 as well, every pair of weights would take another conversion), x is BF16, and the mma wants one type on both sides. A row of x is multiplied by the power of two that brings its largest magnitude to 2^14 .. 2^15 (taken out
// again behind the sum); BF16 values down to 2^-31 of the largest are then exact in binary16, subnormals included. A row where some x is not (or is infinite or NaN) is
// done over at the end, in FP64 on the CUDA cores, whose range holds every product: a row reads the whole weight again for itself, 0.65 ms for 151,936 x 4096, one row after the other (8 rows, 83 us: 731 with one
// row done over, 5.2 ms with all; 256 rows, all of them NaN or with an element below 2^-31 of their largest: 126 ms). All this is nvfp4_rows_kernel's work, once per call; this kernel's blocks copy its result. (Every block
// preparing x for itself took 13 us of a call of 8 rows of 4096.)
//
// Measured, calls back to back (with L2 full of lines that have to be written first, some 10 us more at 151,936 x 4096): 8 rows of 151,936 x 4096 72 us, 4.9 TB/s = 0.75 of the copy rate: issue slots (0.54 of the cycles; conversions, scales and mma wait for each other) and loads share the blame; 1 row 71;
// 8 rows of 50,257 x 4096 32 us, 1 row of 32,768 x 2048 14, of 4,099 x 4096 9 (two launches, and memory's latency in each). Blocks that prepared one or two rows themselves, without the first launch:
// 71.8, 13.7 and 8.4, for 100 bytes of spilled registers: not kept.
//
// A row's sum is (q0 + q1) + (q2 + q3) over four quarters of the hidden dimension, each in order: the same additions whether a warp walks the whole row or, for the tiles left over after
// the last full round, four warps take a quarter each.
#pragma once
#include "common.cuh"
#include "nvfp4.cuh"

#include <climits>

namespace lm {

constexpr int kH4Threads = 512;
constexpr int kH4Warps = kH4Threads / 32;
constexpr int kH4Rows = 8;                   // rows of x to an mma (its n dimension)
constexpr int kH4MaxNT = 2;
constexpr int kH4Tile = 16;                  // vocabulary rows per warp tile (the m dimension)
constexpr int kH4Step = 256;                 // columns per step: 32 bytes of codes per thread and row, a whole 128-byte line per row and quad
constexpr int kH4MaxHidden = 12736;

struct Head4Dev {
  int rows;
  const uint8_t* codes; int64_t codes_stride; const uint8_t* scales; int64_t scales_stride; const float* scale;
  int hidden; int vocab;
  const uint8_t* xt; const uint16_t* xb; const int* shift; const int* bad;
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

// ---- the rows of x, once per call: normalised if a norm is fused, scaled, binary16 --------------------------------------------------------------------

// Workspace: x in binary16, for few rows as they lie in shared memory (head4_x_offset), otherwise by pieces of 64 columns, [group of 256 rows][hidden / 64][rows of the group, padded to 16]
// [128 bytes, swizzled]; x in BF16 [rows][hidden]; shift and bad [padded rows].
constexpr int kX4Threads = 256;
constexpr int kX4Group = 256;
constexpr uint32_t kWait4Limit = 1u << 20;
__host__ __device__ inline int x4_padded(int64_t rows) { return static_cast<int>((rows + 15) / 16 * 16); }
__host__ inline size_t x4_xt_bytes(int64_t rows, int64_t hidden) { return (static_cast<size_t>(x4_padded(rows)) * head4_row_bytes(static_cast<int>(hidden)) + 255) / 256 * 256; }
__host__ inline size_t x4_xb_bytes(int64_t rows, int64_t hidden) { return (static_cast<size_t>(rows) * hidden * 2 + 255) / 256 * 256; }
__host__ inline size_t x4_workspace_bytes(int64_t rows, int64_t hidden) { return x4_xt_bytes(rows, hidden) + x4_xb_bytes(rows, hidden) + static_cast<size_t>(x4_padded(rows)) * 8; }

struct Rows4Dev {
  const uint16_t* x; int64_t x_stride; int rows; int hidden;
  const uint16_t* gamma; float eps; int one_plus;
  int few;                                  // the layout of the mma.sync kernel
  uint8_t* xt; uint16_t* xb; int* shift; int* bad;
};

// One block: one (padded) row, a thread up to kX4Chunks chunks of 8 columns.
constexpr int kX4Chunks = (kH4MaxHidden / 8 + kX4Threads - 1) / kX4Threads;
static __global__ void __launch_bounds__(kX4Threads) nvfp4_rows_kernel(Rows4Dev P) {
  __shared__ float s_sum[kX4Threads / 32];
  __shared__ uint32_t s_top[kX4Threads / 32];
  after_predecessor();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x, chunks = P.hidden / 8;
  // where the 16 bytes of 8 columns go
  const int group = row / kX4Group, in_group = row % kX4Group, n = min(kX4Group, x4_padded(P.rows) - group * kX4Group);
  unsigned char* out = P.few ? P.xt + static_cast<size_t>(row) * head4_row_bytes(P.hidden) : P.xt + static_cast<size_t>(group) * kX4Group * P.hidden * 2;
  auto place = [&](int c) {
    return reinterpret_cast<uint4*>(P.few ? out + head4_x_offset(8 * c) : out + (static_cast<size_t>(c >> 3) * n + in_group) * 128 + (((c & 7) ^ (in_group & 7)) << 4));
  };
  if (row >= P.rows) {
    for (int c = tid; c < chunks; c += kX4Threads) *place(c) = make_uint4(0u, 0u, 0u, 0u);
    if (tid == 0) { P.shift[row] = 0; P.bad[row] = 0; }
    return;
  }
  uint32_t w[kX4Chunks][4];
  float ss = 0.0f;
#pragma unroll
  for (int u = 0; u < kX4Chunks; u++) {
    w[u][0] = w[u][1] = w[u][2] = w[u][3] = 0u;
    if (tid + u * kX4Threads < chunks) load8(P.x + row * P.x_stride + 8 * (tid + u * kX4Threads), w[u]);
  }
  if (P.gamma) {
#pragma unroll
    for (int u = 0; u < kX4Chunks; u++) ss += squares8(w[u]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
    if (lane == 0) s_sum[warp] = ss;
    __syncthreads();
    ss = 0.0f;
#pragma unroll
    for (int q = 0; q < kX4Threads / 32; q++) ss += s_sum[q];
    const float inv_rms = __frsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(P.hidden)), P.eps));
#pragma unroll
    for (int u = 0; u < kX4Chunks; u++) {
      if (tid + u * kX4Threads < chunks) {
        uint32_t gamma[4];
        load8(P.gamma + 8 * (tid + u * kX4Threads), gamma);
        normalise8(w[u], gamma, inv_rms, P.one_plus);
      }
    }
  }
  uint32_t top = 0u;
#pragma unroll
  for (int u = 0; u < kX4Chunks; u++) top = max(top, top_of(w[u]));
  top = warp_max_u32(top);
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kX4Threads / 32; q++) top = max(top, s_top[q]);
  const int shift = shift_of(top);
  bool bad = top >= 0x7F80u;
#pragma unroll
  for (int u = 0; u < kX4Chunks; u++) {
    if (tid + u * kX4Threads < chunks) {
      *reinterpret_cast<uint4*>(P.xb + static_cast<size_t>(row) * P.hidden + 8 * (tid + u * kX4Threads)) = make_uint4(w[u][0], w[u][1], w[u][2], w[u][3]);
      bad |= !scaled8(w[u], scale_of(shift));
    }
  }
  bad = __syncthreads_or(bad);
#pragma unroll
  for (int u = 0; u < kX4Chunks; u++)
    if (tid + u * kX4Threads < chunks) *place(tid + u * kX4Threads) = bad ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(w[u][0], w[u][1], w[u][2], w[u][3]);
  if (P.few && tid < head4_steps(P.hidden) * 32 - chunks) *place(chunks + tid) = make_uint4(0u, 0u, 0u, 0u);     // (the last step's columns beyond the row)
  if (tid == 0) { P.shift[row] = shift; P.bad[row] = bad ? 1 : 0; }
}

// ---- barriers and copies -------------------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void barrier_arrive(uint32_t bar, uint32_t count = 1u) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0u;
}
// False when the limit ran out here or the block has given up. (Out of line: the usual wait is over at the first or second look, and the roles' loops have to stay short.)
__device__ __noinline__ bool barrier_wait_long(uint32_t bar, uint32_t parity, volatile uint32_t* given_up) {
  for (uint32_t i = 0; i < kWait4Limit; i++) {
    if (barrier_try(bar, parity)) return true;
    if ((i & 15u) == 15u && *given_up) return false;
  }
  *given_up = 1u;
  return false;
}
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, volatile uint32_t* given_up) {
  return barrier_try(bar, parity) || barrier_wait_long(bar, parity, given_up);
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
constexpr int kBad4 = INT_MIN;               // in the place of a shift: the row is done over

// The sum of a logit in FP64, by a warp: x [hidden] in BF16, a row's codes and scales.
__device__ __noinline__ double exact_sum(const uint16_t* x, const uint8_t* codes, const uint8_t* scales, int hidden, int lane) {
  double sum = 0.0;
  for (int k = lane * 8; k < hidden; k += 256) {
    uint32_t xw[4], h[4];
    load8(x + k, xw);
    e2m1_to_f16(*reinterpret_cast<const uint32_t*>(codes + (k >> 1)), h);
    const float sc = e4m3_value(scales[k >> 4]);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      sum += static_cast<double>(bf16_lo(xw[e])) * static_cast<double>(f16_lo(h[e]) * sc);
      sum += static_cast<double>(bf16_hi(xw[e])) * static_cast<double>(f16_hi(h[e]) * sc);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
  return sum;
}

// 16 vocabulary rows' codes and scales of a step, a thread's part: 64 columns of rows g and g + 8.
struct Piece4 { uint4 a[2], b[2]; uint32_t fa, fb; };

// kAhead: steps whose loads are in registers or on the way.
template <int NT, int kAhead>
static __global__ void __launch_bounds__(kH4Threads, 1) lm_head_nvfp4_kernel(Head4Dev P) {
  constexpr int kRows = kH4Rows * NT;
  extern __shared__ __align__(16) unsigned char smem_raw[];                 // [kRows][row_bytes]
  __shared__ float4 s_part[4][3][32][NT];                                   // quarters of the tiles left over
  __shared__ float s_factor[kRows];                                         // g * 2^-shift
  __shared__ int s_shift[kRows];
  __shared__ uint64_t s_bar;
  __shared__ uint32_t s_gave_up;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int H = P.hidden, row_bytes = head4_row_bytes(H), steps = head4_steps(H);
  const int gq = lane >> 2, t = lane & 3;
  // A round: a tile to a warp. What is left over after the full rounds takes another one, or (two quarters of a round or less) four warps to a tile.
  const int n_tiles = (P.vocab + kH4Tile - 1) / kH4Tile, all_warps = gridDim.x * kH4Warps, left = n_tiles % all_warps, full = left > all_warps / 2 ? n_tiles : n_tiles - left;
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
  // ---- the first steps' loads; they arrive while x is prepared. (The launch in front is the preparation of x, which begins to let this one in when all before it is complete: the weight
  // may be read at once.)
  Piece4 ring[kAhead];
  int load_tile = blockIdx.x * kH4Warps + warp, load_step = 0;
  auto fetch_next = [&](Piece4& p) {
    if (load_tile >= full) return;
    fetch(p, load_tile, load_step);
    if (++load_step == steps) { load_step = 0; load_tile += all_warps; }
  };
#pragma unroll
  for (int d = 0; d < kAhead - 1; d++) fetch_next(ring[d]);
  // ---- x
  if (tid == 0) {
    barrier_init(smem_address(&s_bar), 1);
    s_gave_up = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  after_predecessor();
  bool plain = true;                                                        // every g * 2^-shift is a normal binary32, with room for the sum
  if (tid == 0) {
    barrier_expect(smem_address(&s_bar), static_cast<uint32_t>(P.rows * row_bytes));
    bulk_copy(smem_address(smem_raw), P.xt, static_cast<uint32_t>(P.rows * row_bytes), smem_address(&s_bar));       // (rows of the mma beyond P.rows reach no other row's sums)
  }
  bool any_bad = false;
  if (tid < P.rows) {
    const int shift = P.shift[tid];
    const double f = static_cast<double>(g) * __hiloint2double((1023 - shift) << 20, 0);
    plain = fabs(f) >= 0x1p-100 && fabs(f) <= 0x1p80;
    any_bad = P.bad[tid] != 0;
    s_shift[tid] = any_bad ? kBad4 : shift; s_factor[tid] = static_cast<float>(f);
  }
  plain = __syncthreads_and(plain);
  any_bad = __syncthreads_or(any_bad);
  barrier_wait(smem_address(&s_bar), 0u, &s_gave_up);
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
        if (r < P.rows && vv < P.vocab && s_shift[r] != kBad4) P.logits[r * P.logits_stride + vv] = f32_to_bf16(plain ? __fmul_rn(c[n][e], s_factor[r]) : head4_finish(c[n][e], g, s_shift[r]));
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
      for (int n = 0; n < NT; n++) s_part[group][part - 1][lane][n] = make_float4(c[n][0], c[n][1], c[n][2], c[n][3]);
    }
    asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory");
    if (part == 0) {
#pragma unroll
      for (int n = 0; n < NT; n++) {
        const float4 p = s_part[group][0][lane][n], q = s_part[group][1][lane][n], r = s_part[group][2][lane][n];
        c[n][0] = __fadd_rn(__fadd_rn(c[n][0], p.x), __fadd_rn(q.x, r.x)); c[n][1] = __fadd_rn(__fadd_rn(c[n][1], p.y), __fadd_rn(q.y, r.y));
        c[n][2] = __fadd_rn(__fadd_rn(c[n][2], p.z), __fadd_rn(q.z, r.z)); c[n][3] = __fadd_rn(__fadd_rn(c[n][3], p.w), __fadd_rn(q.w, r.w));
      }
      store(tile, c);
    }
    asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory");
  }
  // ---- rows whose x is no binary16 after the scaling, or x that never came
  __syncthreads();
  for (int r = 0; r < P.rows && (any_bad || s_gave_up); r++) {
    if (s_shift[r] != kBad4 && !s_gave_up) continue;
    for (int v = blockIdx.x * kH4Warps + warp; v < P.vocab; v += all_warps) {
      const float z = s_gave_up ? __int_as_float(0x7FC00000) : head4_finish(exact_sum(P.xb + static_cast<size_t>(r) * H, P.codes + v * P.codes_stride, P.scales + v * P.scales_stride, H, lane), g, 0);
      if (lane == 0) P.logits[r * P.logits_stride + v] = f32_to_bf16(z);
    }
  }
}

}  // namespace lm
