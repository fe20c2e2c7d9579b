// The vocabulary projection with a 4-bit weight for more rows than a decode step has (9 and up): logits = x * W^T on tcgen05, 128 vocabulary rows (M) by up to
// 256 rows of x (N) to an accumulator, FP32 in tensor memory.
//
// W arrives as codes and leaves shared memory as binary16: 16 warps take a tile's codes from global memory (several tiles ahead, in registers), multiply by the block scales
// (exact, nvfp4.cuh) and store the operand in the 128-byte swizzle; one thread issues the products. x is prepared once per call by nvfp4_rows_kernel: normalised if a norm is
// fused, scaled by a power of two per row, rounded to binary16 (exact; rows where it is not are done over, in FP64, at the end), laid out so that the columns of a step are
// one contiguous piece: an untiled bulk copy brings it.
//
// A block owns a contiguous range of tiles and walks the hidden dimension once for as many of them as tensor memory holds accumulators (512 columns: 2 tiles of 256 rows, 16 of
// 32): x then crosses from L2 once for all of these. The order of a logit's additions is that of the hidden dimension, whatever the tile or the block.
// Every wait has a limit; a block whose wait ran out writes NaN.
#pragma once
#include "common.cuh"
#include "lm_head_nvfp4.cuh"
#include "nvfp4.cuh"

namespace lm {

constexpr int kB4Tile = 128;                 // vocabulary rows per tile (M)
constexpr int kB4MaxN = 256;                 // rows of x per launch
constexpr int kB4Cols = 128;                 // columns per step
constexpr int kB4Stages = 3;                 // tiles of W in shared memory
constexpr int kB4StageBytes = kB4Tile * kB4Cols * 2;
constexpr int kB4DequantWarps = 16, kB4DoneWarps = 4;
constexpr int kB4MmaWarp = kB4DequantWarps, kB4CopyWarp = kB4MmaWarp + 1, kB4FirstDoneWarp = kB4CopyWarp + 1;
constexpr int kB4Threads = 32 * (kB4FirstDoneWarp + kB4DoneWarps);
constexpr int kB4Ahead = 6;                  // tiles whose codes are in flight
constexpr int kB4MaxXStages = 4;
constexpr int kB4RowsThreads = 256;
constexpr uint32_t kB4WaitLimit = 1u << 20;
constexpr int kB4SmemLimit = 232448;

struct Batch4Dev {
  const uint8_t* codes; int64_t codes_stride; const uint8_t* scales; int64_t scales_stride; const float* scale;
  int hidden; int vocab; int rows; int n;    // n: rows padded to a multiple of 16
  const uint8_t* xt; const uint16_t* xb; const int* shift; const int* bad;
  uint16_t* logits; int64_t logits_stride;
  int per_pass; int column_stride; int x_stages;
};

// Workspace: x in binary16 by steps of 64 columns, [group][hidden / 64][rows of the group, padded][128 bytes, swizzled]; x in BF16 [rows][hidden]; shift and bad [padded rows].
__host__ __device__ inline int batch4_padded(int64_t rows) { return static_cast<int>((rows + 15) / 16 * 16); }
__host__ inline size_t batch4_xt_bytes(int64_t rows, int64_t hidden) { return static_cast<size_t>(batch4_padded(rows)) * hidden * 2; }
__host__ inline size_t batch4_xb_bytes(int64_t rows, int64_t hidden) { return (static_cast<size_t>(rows) * hidden * 2 + 255) / 256 * 256; }
__host__ inline size_t batch4_workspace_bytes(int64_t rows, int64_t hidden) {
  return batch4_xt_bytes(rows, hidden) + batch4_xb_bytes(rows, hidden) + 2 * (static_cast<size_t>(batch4_padded(rows)) * 4 + 255) / 256 * 256 + 512;
}
__host__ __device__ inline int batch4_x_stage_bytes(int n) { return n * kB4Cols * 2; }
__host__ inline size_t batch4_smem_bytes(int n, int x_stages) { return 1024 + kB4Stages * kB4StageBytes + static_cast<size_t>(x_stages) * batch4_x_stage_bytes(n) + kB4MaxN * 4 + 256; }

struct Rows4Dev {
  const uint16_t* x; int64_t x_stride; int rows; int hidden;
  const uint16_t* gamma; float eps; int one_plus;
  uint8_t* xt; uint16_t* xb; int* shift; int* bad;
};

// One block: one (padded) row.
static __global__ void __launch_bounds__(kB4RowsThreads) nvfp4_rows_kernel(Rows4Dev P) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  uint16_t* xs = reinterpret_cast<uint16_t*>(smem_raw);                     // [hidden]
  __shared__ float s_sum[kB4RowsThreads / 32];
  __shared__ uint32_t s_max[kB4RowsThreads / 32];
  after_predecessor();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x, H = P.hidden;
  const int group = row / kB4MaxN, in_group = row % kB4MaxN;
  const int n = min(kB4MaxN, batch4_padded(P.rows) - group * kB4MaxN);
  unsigned char* out = P.xt + static_cast<size_t>(group) * kB4MaxN * H * 2;
  auto place = [&](int chunk) { return out + (static_cast<size_t>(chunk >> 3) * n + in_group) * 128 + (((chunk & 7) ^ (in_group & 7)) << 4); };   // 8 columns: 16 bytes
  if (row >= P.rows) {
    for (int c = tid; c < H / 8; c += kB4RowsThreads) *reinterpret_cast<uint4*>(place(c)) = make_uint4(0u, 0u, 0u, 0u);
    if (tid == 0) { P.shift[row] = 0; P.bad[row] = 0; }
    return;
  }
  const uint16_t* x = P.x + row * P.x_stride;
  const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15u) == 0;
  float ss = 0.0f;
  for (int c = tid; c < H / 8; c += kB4RowsThreads) {
    uint4 q;
    if (aligned) q = *reinterpret_cast<const uint4*>(x + 8 * c);
    else {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; e++) w[e] = static_cast<uint32_t>(x[8 * c + 2 * e]) | static_cast<uint32_t>(x[8 * c + 2 * e + 1]) << 16;
      q = make_uint4(w[0], w[1], w[2], w[3]);
    }
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; e++) { ss = __fmaf_rn(bf16_lo(w[e]), bf16_lo(w[e]), ss); ss = __fmaf_rn(bf16_hi(w[e]), bf16_hi(w[e]), ss); }
    *reinterpret_cast<uint4*>(xs + 8 * c) = q;
  }
  float inv_rms = 1.0f;
  if (P.gamma) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
    if (lane == 0) s_sum[warp] = ss;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int q = 0; q < kB4RowsThreads / 32; q++) s += s_sum[q];
    inv_rms = __frsqrt_rn(__fadd_rn(__fdiv_rn(s, static_cast<float>(H)), P.eps));
  }
  uint32_t top = 0u;
  for (int c = tid; c < H / 8; c += kB4RowsThreads) {                        // (a thread's own columns: no barrier)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      uint16_t v = xs[8 * c + e];
      if (P.gamma) {
        const float gm = __uint_as_float(static_cast<uint32_t>(P.gamma[8 * c + e]) << 16);
        v = f32_to_bf16(__fmul_rn(__fmul_rn(__uint_as_float(static_cast<uint32_t>(v) << 16), inv_rms), P.one_plus ? __fadd_rn(1.0f, gm) : gm));
        xs[8 * c + e] = v;
      }
      top = max(top, static_cast<uint32_t>(v) & 0x7FFFu);
    }
  }
  top = warp_max_u32(top);
  if (lane == 0) s_max[warp] = top;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kB4RowsThreads / 32; q++) top = max(top, s_max[q]);
  const int shift = top == 0u ? 0 : 141 - static_cast<int>(max(top >> 7, 1u));
  bool bad = top >= 0x7F80u;
  for (int c = tid; c < H / 8; c += kB4RowsThreads) {
#pragma unroll
    for (int e = 0; e < 8; e++) { uint16_t h; bad |= !scaled_f16(xs[8 * c + e], shift, &h); }
  }
  bad = __syncthreads_or(bad);
  for (int c = tid; c < H / 8; c += kB4RowsThreads) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      uint16_t lo, hi;
      scaled_f16(xs[8 * c + 2 * e], shift, &lo); scaled_f16(xs[8 * c + 2 * e + 1], shift, &hi);
      w[e] = bad ? 0u : static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 16;
    }
    *reinterpret_cast<uint4*>(place(c)) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(P.xb + static_cast<size_t>(row) * H + 8 * c) = *reinterpret_cast<const uint4*>(xs + 8 * c);
  }
  if (tid == 0) { P.shift[row] = shift; P.bad[row] = bad ? 1 : 0; }
}

// ---- barriers, copies and products --------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void barrier_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0u;
}
// False when the limit ran out here or the block has given up.
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, volatile uint32_t* given_up) {
  for (uint32_t i = 0; i < kB4WaitLimit; i++) {
    if (barrier_try(bar, parity)) return true;
    if ((i & 15u) == 15u && *given_up) return false;
  }
  *given_up = 1u;
  return false;
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void products_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// An operand in shared memory, rows of 128 bytes (64 binary16, the hidden dimension running along them) in the 128-byte swizzle: groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand(uint32_t address) {
  return static_cast<uint64_t>((address >> 4) & 0x3FFFu) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void product_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t form, bool add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(form), "r"(add ? 1u : 0u) : "memory");
}
__device__ __forceinline__ void accumulators32(uint32_t address, uint32_t (&v)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
                 "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
                 "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31]) : "r"(address));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// The tiles and steps of a block in the order they are taken: passes of per_pass tiles, in a pass the steps, in a step the tiles.
struct Walk4 {
  int first, last, end, per_pass, steps;     // the pass' tiles [first, last)
  int tile, step;
  __device__ __forceinline__ Walk4(int begin, int end_, int per_pass_, int steps_)
      : first(begin), last(min(begin + per_pass_, end_)), end(end_), per_pass(per_pass_), steps(steps_), tile(begin), step(0) {}
  __device__ __forceinline__ bool more() const { return first < end; }
  __device__ __forceinline__ void next() {
    if (++tile < last) return;
    tile = first;
    if (++step < steps) return;
    step = 0; first = last; last = min(first + per_pass, end); tile = first;
  }
};

static __global__ void __launch_bounds__(kB4Threads, 1) lm_head_nvfp4_batch_kernel(Batch4Dev P) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_address(smem_raw) & 1023u)) & 1023u);
  unsigned char* ws = smem;                                                 // W: kB4Stages tiles
  unsigned char* xs = ws + kB4Stages * kB4StageBytes;                        // x: x_stages steps
  const int x_bytes = batch4_x_stage_bytes(P.n);
  float* factor = reinterpret_cast<float*>(xs + P.x_stages * x_bytes);        // [n] g * 2^-shift
  uint64_t* bars = reinterpret_cast<uint64_t*>(factor + kB4MaxN);
  uint32_t* words = reinterpret_cast<uint32_t*>(bars + 2 * kB4Stages + 2 * kB4MaxXStages + 3);     // [0] tensor memory, [1] given up
  volatile uint32_t* given_up = words + 1;
  const uint32_t w_full = smem_address(bars), w_empty = w_full + 8 * kB4Stages, x_full = w_empty + 8 * kB4Stages, x_empty = x_full + 8 * kB4MaxXStages, acc_full = x_empty + 8 * kB4MaxXStages,
                 acc_empty = acc_full + 8, drained = acc_empty + 8;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int H = P.hidden, steps = (H + kB4Cols - 1) / kB4Cols;
  const int n_tiles = (P.vocab + kB4Tile - 1) / kB4Tile;
  const int begin = static_cast<int>(static_cast<long long>(blockIdx.x) * n_tiles / gridDim.x), end = static_cast<int>(static_cast<long long>(blockIdx.x + 1) * n_tiles / gridDim.x);
  if (warp == kB4MmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_address(words)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int s = 0; s < kB4Stages; s++) { barrier_init(w_full + 8 * s, kB4DequantWarps); barrier_init(w_empty + 8 * s, 1); }
    for (int s = 0; s < kB4MaxXStages; s++) { barrier_init(x_full + 8 * s, 1); barrier_init(x_empty + 8 * s, 1); }
    barrier_init(acc_full, 1); barrier_init(acc_empty, kB4DoneWarps); barrier_init(drained, 1);
    words[1] = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  after_predecessor();
  const float g = __ldg(P.scale);
  bool plain = true;                                                        // every g * 2^-shift is a normal binary32, with room for the sum
  for (int r = tid; r < P.n; r += kB4Threads) {
    const double f = static_cast<double>(g) * __hiloint2double((1023 - P.shift[r]) << 20, 0);
    plain &= fabs(f) >= 0x1p-100 && fabs(f) <= 0x1p80;
    factor[r] = static_cast<float>(f);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  plain = __syncthreads_and(plain);
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = words[0];

  if (warp < kB4DequantWarps) {
    // ---- W: a warp has 8 rows of a tile, 4 lanes to a row, 32 columns each (16 bytes of codes, two scales)
    const int r8 = lane >> 2, q = lane & 3, row = 8 * warp + r8;
    // (the four 16-byte chunks of a lane in an order that keeps 8 lanes -- 2 rows, 2 halves of 64 columns -- on different banks)
    const bool swap = q >= 2;
    const uint32_t base = static_cast<uint32_t>((q >> 1) * (kB4Tile * 128) + row * 128);
    uint32_t offset[4];
#pragma unroll
    for (int i = 0; i < 4; i++) offset[i] = base + static_cast<uint32_t>((((q & 1) * 4 + (swap ? i ^ 2 : i)) ^ r8) << 4);
    uint4 c[kB4Ahead];
    uint32_t s[kB4Ahead];
    Walk4 load(begin, end, P.per_pass, steps), use = load;
    auto fetch = [&](uint4& cc, uint32_t& ss) {
      cc = make_uint4(0u, 0u, 0u, 0u); ss = 0u;
      if (load.more()) {
        const int64_t v = min(load.tile * kB4Tile + row, P.vocab - 1);       // (rows beyond the vocabulary: the last one again, never stored)
        const int k = load.step * kB4Cols + q * 32;
        if (k < H) {
          cc = __ldcs(reinterpret_cast<const uint4*>(P.codes + v * P.codes_stride + (k >> 1)));
          ss = __ldg(reinterpret_cast<const uint16_t*>(P.scales + v * P.scales_stride + (k >> 4)));
        }
        load.next();
      }
    };
#pragma unroll
    for (int u = 0; u < kB4Ahead; u++) fetch(c[u], s[u]);
    int stage = 0; uint32_t phase = 0u;
    bool go = true;
    while (go && use.more()) {
#pragma unroll
      for (int u = 0; u < kB4Ahead; u++) {
        if (!go || !use.more()) break;
        const uint4 cc = c[u];
        const uint32_t pair = e4m3_to_f16(s[u]);
        const bool half = use.step * kB4Cols + q * 32 < H;                   // (the last step may have 64 columns only)
        fetch(c[u], s[u]);
        const uint32_t s0 = __byte_perm(pair, 0u, swap ? 0x3232 : 0x1010), s1 = __byte_perm(pair, 0u, swap ? 0x1010 : 0x3232);
        const uint32_t w[4] = {swap ? cc.z : cc.x, swap ? cc.w : cc.y, swap ? cc.x : cc.z, swap ? cc.y : cc.w};
        uint4 h[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          uint32_t v[4];
          e2m1_to_f16(w[i], v);
          const uint32_t sc = i < 2 ? s0 : s1;
          h[i] = make_uint4(f16x2_mul(v[0], sc), f16x2_mul(v[1], sc), f16x2_mul(v[2], sc), f16x2_mul(v[3], sc));
        }
        go = barrier_wait(w_empty + 8 * stage, phase ^ 1u, given_up);
        if (go && half) {
          unsigned char* out = ws + stage * kB4StageBytes;
#pragma unroll
          for (int i = 0; i < 4; i++) *reinterpret_cast<uint4*>(out + offset[i]) = h[i];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) barrier_arrive(w_full + 8 * stage);
        if (++stage == kB4Stages) { stage = 0; phase ^= 1u; }
        use.next();
        go = __all_sync(kFull, go);
      }
    }
  } else if (warp == kB4MmaWarp) {
    if (lane == 0) {
      const uint32_t form = (1u << 4) | (static_cast<uint32_t>(P.n >> 3) << 17) | (static_cast<uint32_t>(kB4Tile >> 4) << 24);   // binary16 operands, FP32 accumulators
      int ws_ = 0, xs_ = 0; uint32_t wp = 0u, xp = 0u, ap = 1u;
      bool go = true;
      for (Walk4 at(begin, end, P.per_pass, steps); go && at.more(); at.next()) {
        if (at.tile == at.first) {
          if (at.step == 0) { go = barrier_wait(acc_empty, ap, given_up); ap ^= 1u; }     // (the first pass finds them empty)
          go = go && barrier_wait(x_full + 8 * xs_, xp, given_up);
        }
        go = go && barrier_wait(w_full + 8 * ws_, wp, given_up);
        if (!go) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem + static_cast<uint32_t>((at.tile - at.first) * P.column_stride);
        const int halves = H - at.step * kB4Cols > 64 ? 2 : 1;
        for (int half = 0; half < halves; half++) {
          const uint64_t a = operand(smem_address(ws) + ws_ * kB4StageBytes + half * (kB4Tile * 128)), b = operand(smem_address(xs) + xs_ * x_bytes + half * P.n * 128);
#pragma unroll
          for (int k = 0; k < 4; k++) product_f16(d, a + 2 * k, b + 2 * k, form, at.step + half + k > 0);
        }
        products_commit(w_empty + 8 * ws_);
        if (++ws_ == kB4Stages) { ws_ = 0; wp ^= 1u; }
        if (at.tile == at.last - 1) {
          products_commit(x_empty + 8 * xs_);
          if (++xs_ == P.x_stages) { xs_ = 0; xp ^= 1u; }
          if (at.step == steps - 1) products_commit(acc_full);
        }
      }
      if (!go) {                                                            // what is under way ends before the block does
        products_commit(drained);
        for (uint32_t i = 0; i < kB4WaitLimit && !barrier_try(drained, 0u); i++) {}
      }
    }
  } else if (warp == kB4CopyWarp) {
    if (lane == 0) {
      int stage = 0, issued = 0; uint32_t phase = 0u;
      bool go = true;
      for (int first = begin; go && first < end; first += P.per_pass) {
        for (int step = 0; step < steps; step++) {
          go = barrier_wait(x_empty + 8 * stage, phase ^ 1u, given_up);
          if (!go) break;
          const uint32_t bytes = static_cast<uint32_t>(min(2, (H - step * kB4Cols) / 64) * P.n * 128);
          barrier_expect(x_full + 8 * stage, bytes);
          bulk_copy(smem_address(xs) + stage * x_bytes, P.xt + static_cast<size_t>(step) * x_bytes, bytes, x_full + 8 * stage);
          issued++;
          if (++stage == P.x_stages) { stage = 0; phase ^= 1u; }
        }
      }
      if (!go)                                                              // the copies under way
        for (int k = 0; k < P.x_stages && k < issued; k++) {
          if (stage == 0) { stage = P.x_stages; phase ^= 1u; }
          stage--;
          for (uint32_t i = 0; i < kB4WaitLimit && !barrier_try(x_full + 8 * stage, phase); i++) {}
        }
    }
  } else {
    // ---- finished accumulators: a warp has 32 vocabulary rows of every tile; a column is a row of logits
    const int part = warp & 3;
    bool go = true;
    uint32_t phase = 0u;
    for (int first = begin; go && first < end; first += P.per_pass, phase ^= 1u) {
      const int last = min(first + P.per_pass, end);
      go = __all_sync(kFull, barrier_wait(acc_full, phase, given_up));
      if (!go) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      for (int tile = first; tile < last; tile++) {
        const int v = tile * kB4Tile + part * 32 + lane;
        for (int r0 = 0; r0 < P.n; r0 += 32) {
          uint32_t a[32];
          accumulators32(tmem + (static_cast<uint32_t>(part * 32) << 16) + static_cast<uint32_t>((tile - first) * P.column_stride + r0), a);
          if (v < P.vocab) {
#pragma unroll
            for (int j = 0; j < 32; j++) {
              const int r = r0 + j;
              if (r >= P.rows) break;
              const float z = plain ? __fmul_rn(__uint_as_float(a[j]), factor[r]) : head4_finish(__uint_as_float(a[j]), g, P.shift[r]);
              P.logits[r * P.logits_stride + v] = f32_to_bf16(z);
            }
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) barrier_arrive(acc_empty);
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == kB4MmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  const int v0 = begin * kB4Tile, v1 = min(end * kB4Tile, P.vocab);
  if (*given_up) {
    for (int r = 0; r < P.rows; r++)
      for (int v = v0 + tid; v < v1; v += kB4Threads) P.logits[r * P.logits_stride + v] = 0x7FFFu;
    return;
  }
  // ---- rows whose x is no binary16 after the scaling: FP64
  for (int r = 0; r < P.rows; r++) {
    if (!P.bad[r]) continue;
    const uint16_t* x = P.xb + static_cast<size_t>(r) * H;
    for (int v = v0 + warp; v < v1; v += kB4Threads / 32) {
      double sum = 0.0;
      for (int w = lane; w < H / 8; w += 32) {
        uint32_t h[4];
        e2m1_to_f16(*reinterpret_cast<const uint32_t*>(P.codes + static_cast<int64_t>(v) * P.codes_stride + w * 4), h);
        const float s = e4m3_value(P.scales[static_cast<int64_t>(v) * P.scales_stride + (w >> 1)]);
        const uint4 xq = *reinterpret_cast<const uint4*>(x + 8 * w);
        const uint32_t xw[4] = {xq.x, xq.y, xq.z, xq.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          sum += static_cast<double>(bf16_lo(xw[e])) * static_cast<double>(f16_lo(h[e]) * s);
          sum += static_cast<double>(bf16_hi(xw[e])) * static_cast<double>(f16_hi(h[e]) * s);
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
      if (lane == 0) P.logits[r * P.logits_stride + v] = f32_to_bf16(head4_finish(sum, g, 0));
    }
  }
}

}  // namespace lm
