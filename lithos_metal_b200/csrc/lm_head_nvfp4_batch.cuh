// The vocabulary projection with a 4-bit weight for more rows than a decode step has (17 and up; 9 where shared memory does not hold two eights of long rows): logits = x * W^T on tcgen05, 128 vocabulary rows (M) by up to
// 256 rows of x (N) to an accumulator, FP32 in tensor memory.
//
// W arrives in shared memory as codes and goes to tensor memory as binary16: 16 warps turn codes into binary16, multiply by the block scales (exact, nvfp4.cuh) and store the A
// operand there, a lane a row; one thread issues the products. (With A in shared memory a tile's 32 KB were written and read there once more: 218 us with 16 rows, 384 with 256, bound by
// shared memory's bandwidth.) x is prepared once per call by nvfp4_rows_kernel: normalised if a norm is
// fused, scaled by a power of two per row, rounded to binary16 (exact; rows where it is not are done over, in FP64, at the end), laid out so that the columns of a step are
// one contiguous piece: an untiled bulk copy brings it.
//
// A block owns a contiguous range of tiles and walks the hidden dimension once for as many of them as tensor memory holds accumulators beside four operands (256 columns: a tile of
// 256 rows, 8 of 32): x then crosses from L2 once for all of these. The order of a logit's additions is that of the hidden dimension, whatever the tile or the block.
// Measured, 151,936 x 4096, calls back to back: 17 rows 95 us, 64 109, 128 148, 256 240 (1330 TFLOP/s, 0.79 of the measured library rate; tensor pipe 0.74 busy at 1.6 GHz); beyond that a launch for every 256
// rows, each of which converts the weight again: 512 rows 518, 1024 1036, 4096 4430. Up to 64 rows a tile's step of 256 columns takes 0.75 us whatever the rows, and no unit is full: with 32 rows (100,000 x 4096)
// the tensor pipe is busy for 19 % of the clocks (some 15 of them to a product of 128 x 16 of W), issue slots 41 %, DRAM 3.2 TB/s. What is left is the turn of a pair: codes, conversion, store to tensor memory, products,
// commit, and only then the next conversion. More of these under way in another split of the same room were slower: a third set of operands in tensor memory 32 rows 98 -> 105 us, 64 110 -> 130 (half the accumulators),
// 24 converting warps instead of 16 98 -> 114. With 256 rows what comes in per SM bounds it, 128 KB of x from L2 a step, 42 bytes a
// clock, and, between two tiles, the accumulators' way out, for which tensor memory has no second set.
// Every wait has a limit; a block whose wait ran out writes NaN.
#pragma once
#include "common.cuh"
#include "lm_head_nvfp4.cuh"
#include "nvfp4.cuh"

#include <cuda.h>

namespace lm {

constexpr int kB4Tile = 128;                 // vocabulary rows per tile (M)
constexpr int kB4MaxN = kX4Group;            // rows of x per launch
constexpr int kB4StepCols = 256;             // columns of a tile's codes that come together: 128 bytes a row, and 16 of scales
constexpr int kB4Cols = 128;                 // columns of an operand: two a step
constexpr int kB4XCols = 64;                 // columns of x that come together
constexpr int kB4Pairs = 2;                  // steps of a tile in the making, and as many in tensor memory: 8 warps each, 4 to an operand
constexpr int kB4CodeBytes = kB4Tile * kB4StepCols / 2, kB4SlotBytes = kB4CodeBytes + kB4Tile * kB4StepCols / kFp4Block;
constexpr int kB4MaxCodeSlots = 8, kB4MaxXStages = 8;
constexpr int kB4OperandColumns = kB4Cols / 2;                              // of tensor memory
constexpr int kB4SumColumns = 512 - 2 * kB4Pairs * kB4OperandColumns;        // ... for the accumulators
constexpr int kB4MaxSums = kB4SumColumns / 32;
constexpr int kB4DequantWarps = 8 * kB4Pairs, kB4DoneWarps = 4;
constexpr int kB4MmaWarp = kB4DequantWarps, kB4CopyWarp = kB4MmaWarp + 1, kB4CodeWarp = kB4CopyWarp + 1, kB4FirstDoneWarp = kB4CodeWarp + 1;
constexpr int kB4Threads = 32 * (kB4FirstDoneWarp + kB4DoneWarps);
constexpr int kB4SmemLimit = 232448;

struct Batch4Dev {
  const uint8_t* codes; int64_t codes_stride; const uint8_t* scales; int64_t scales_stride; const float* scale;
  int hidden; int vocab; int rows; int n;    // n: rows padded to a multiple of 16
  const uint8_t* xt; const uint16_t* xb; const int* shift; const int* bad;
  uint16_t* logits; int64_t logits_stride;
  int per_pass; int column_stride; int code_slots; int x_stages;
  int each; int left; int left_blocks; int left_n;    // tiles that every block has; tiles left over; blocks to each of these; rows of x to such a block
};

__host__ __device__ inline int batch4_x_stage_bytes(int n) { return n * kB4XCols * 2; }
__host__ inline size_t batch4_smem_bytes(int n, int code_slots, int x_stages) {
  return 1024 + static_cast<size_t>(code_slots) * kB4SlotBytes + static_cast<size_t>(x_stages) * batch4_x_stage_bytes(n) + kB4MaxN * 4 + 512;
}

// ---- copies and products -------------------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ bool elected() {                                 // true in one lane of a warp that is together, always the same
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0u;
}
// A box of 128 rows: 128 bytes of codes in the 128-byte swizzle, or 16 bytes of scales (columns a multiple of that; what lies beyond the matrix arrives as zeros).
__device__ __forceinline__ void tile_copy(uint32_t dst, const CUtensorMap* map, int column, int row, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(column), "r"(row), "r"(bar) : "memory");
}
__device__ __forceinline__ void products_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// An operand in shared memory, rows of 128 bytes (64 binary16, the hidden dimension running along them) in the 128-byte swizzle: groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand(uint32_t address) {
  return static_cast<uint64_t>((address >> 4) & 0x3FFFu) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void product_f16(uint32_t d, uint32_t a, uint64_t b, uint32_t form, uint32_t add) {     // a: in tensor memory
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(form), "r"(add) : "memory");
}
__device__ __forceinline__ void operand16(uint32_t address, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(address), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
               "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void accumulators32(uint32_t address, uint32_t (&v)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
                 "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
                 "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31]) : "r"(address));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t picked(const uint32_t (&v)[32], int j) {
  uint32_t r = v[0];
#pragma unroll
  for (int i = 1; i < 32; i++) r = i == j ? v[i] : r;
  return r;
}

// Every block has as many tiles as every other; the few left over are shared by the rows of x (a block that did one with all rows made the others wait: 256 rows of 151,936 x 4096 256 us, 244 so; of 32,768 x 2048 72 and 45).
struct Pass4 { int first, count, n, r0; };    // tiles first .. first + count, rows r0 .. r0 + n of x
struct Passes4 {
  int begin, end, per_pass, main, n, tiles; Pass4 left;
  __device__ __forceinline__ explicit Passes4(const Batch4Dev& P) {
    begin = blockIdx.x * P.each; end = begin + P.each; per_pass = P.per_pass; main = (P.each + per_pass - 1) / per_pass; n = P.n; tiles = P.each;
    left = Pass4{0, 0, 0, 0};
    if (static_cast<int>(blockIdx.x) < P.left * P.left_blocks) {
      const int r0 = blockIdx.x % P.left_blocks * P.left_n;
      if (r0 < P.n) { left = Pass4{static_cast<int>(gridDim.x) * P.each + static_cast<int>(blockIdx.x) / P.left_blocks, 1, min(P.left_n, P.n - r0), r0}; tiles++; }
    }
  }
  __device__ __forceinline__ bool get(int i, Pass4& p) const {
    if (i < main) { p.first = begin + i * per_pass; p.count = min(per_pass, end - p.first); p.n = n; p.r0 = 0; return true; }
    p = left;
    return i == main && left.count > 0;
  }
};

// A block takes its tiles in passes of per_pass, in a pass the steps of 256 columns, in a step the tiles. These (step, tile) are numbered through: number i has place i % code_slots for its
// codes and pair i % 2 of the operands in the making. code_slots is even: a place then belongs to one pair, whose warps have all seen one filling before they wait for the next. (With three
// places a pair could come to one whose codes for the other pair were still on their way, and a wait by parity takes the phase before the current one for the phase after it: it read codes
// that were arriving, and the barriers lost count.)
static __global__ void __launch_bounds__(kB4Threads, 1) lm_head_nvfp4_batch_kernel(const __grid_constant__ CUtensorMap code_map, const __grid_constant__ CUtensorMap scale_map, Batch4Dev P) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_address(smem_raw) & 1023u)) & 1023u);
  const int x_bytes = batch4_x_stage_bytes(P.n);
  unsigned char* cs = smem;                                                 // codes, in the 128-byte swizzle: code_slots tiles of a step
  unsigned char* xs = cs + P.code_slots * kB4CodeBytes;                      // x: x_stages times 64 columns
  unsigned char* ss = xs + P.x_stages * x_bytes;                             // scales: code_slots times [128 rows][16 bytes]
  float* factor = reinterpret_cast<float*>(ss + P.code_slots * (kB4SlotBytes - kB4CodeBytes));    // [n] g * 2^-shift
  uint64_t* bars = reinterpret_cast<uint64_t*>(factor + kB4MaxN);
  uint32_t* words = reinterpret_cast<uint32_t*>(bars + 2 * (kB4Pairs + kB4MaxXStages + kB4MaxSums + kB4MaxCodeSlots) + 1);     // [0] tensor memory, [1] given up, [2] rows to do over
  volatile uint32_t* given_up = words + 1;
  const uint32_t w_full = smem_address(bars), w_empty = w_full + 8 * kB4Pairs, x_full = w_empty + 8 * kB4Pairs, x_empty = x_full + 8 * kB4MaxXStages, acc_full = x_empty + 8 * kB4MaxXStages,
                 acc_empty = acc_full + 8 * kB4MaxSums, c_full = acc_empty + 8 * kB4MaxSums, c_empty = c_full + 8 * kB4MaxCodeSlots, drained = c_empty + 8 * kB4MaxCodeSlots;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int H = P.hidden, steps = (H + kB4StepCols - 1) / kB4StepCols;
  const Passes4 passes(P);
  Pass4 pass;
  if (warp == kB4MmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_address(words)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int s = 0; s < kB4Pairs; s++) { barrier_init(w_full + 8 * s, 8); barrier_init(w_empty + 8 * s, 1); }
    for (int s = 0; s < kB4MaxXStages; s++) { barrier_init(x_full + 8 * s, 1); barrier_init(x_empty + 8 * s, 1); }
    for (int s = 0; s < kB4MaxSums; s++) { barrier_init(acc_full + 8 * s, 1); barrier_init(acc_empty + 8 * s, kB4DoneWarps); }
    for (int s = 0; s < kB4MaxCodeSlots; s++) { barrier_init(c_full + 8 * s, 1); barrier_init(c_empty + 8 * s, 8); }
    barrier_init(drained, 1);
    words[1] = words[2] = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = words[0];

  if (warp < kB4DequantWarps) {
    // ---- W: 4 warps make an operand, a lane a row of it (a lane of tensor memory), 8 warps a tile's two. The codes' 16-byte pieces are swizzled: 8 lanes reading their rows' piece
    // meet different banks.
    const int pair = warp >> 3, half = (warp >> 2) & 1, quarter = warp & 3, in_tile = 32 * quarter + lane;
    const unsigned char *code_row = cs + in_tile * 128, *scale_row = ss + in_tile * 16 + half * 8;
    const uint32_t operand = tmem + kB4SumColumns + static_cast<uint32_t>((2 * pair + half) * kB4OperandColumns) + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t full = w_full + 8 * pair, empty = w_empty + 8 * pair;
    int piece[4];
#pragma unroll
    for (int i = 0; i < 4; i++) piece[i] = ((half * 4 + i) ^ (lane & 7)) << 4;
    uint32_t phase = 1u, slot_phase = 0u;
    int slot = pair;                                                        // (code_slots is even: slots of this pair's parity)
    for (int left = passes.tiles * steps - pair; left > 0; left -= 2) {        // (which tile and step: the copies know)
      barrier_wait(c_full + 8 * slot, slot_phase, given_up);                 // (where a wait has run out, what follows is harmless and the block writes NaN)
      uint4 cc[4];
#pragma unroll
      for (int i = 0; i < 4; i++) cc[i] = *reinterpret_cast<const uint4*>(code_row + slot * kB4CodeBytes + piece[i]);
      const uint2 sc = *reinterpret_cast<const uint2*>(scale_row + slot * (kB4SlotBytes - kB4CodeBytes));
      barrier_wait(empty, phase, given_up);
      phase ^= 1u;
      __syncwarp();
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
      for (int i = 0; i < 4; i++) {                                          // 32 columns
        const uint32_t two = e4m3_to_f16((i < 2 ? sc.x : sc.y) >> (16 * (i & 1)));
        const uint32_t w[4] = {cc[i].x, cc[i].y, cc[i].z, cc[i].w};
        uint32_t v[16];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          uint32_t h[4];
          e2m1_to_f16(w[j], h);
          const uint32_t s = __byte_perm(two, 0u, j < 2 ? 0x1010 : 0x3232);
#pragma unroll
          for (int e = 0; e < 4; e++) v[4 * j + e] = f16x2_mul(h[e], s);
        }
        operand16(operand + i * 16, v);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      // (The place is handed back when its codes have been converted, not when their loads have been issued: with shared memory busy these were overtaken by the copy that followed.)
      if (lane == 0) { barrier_arrive(c_empty + 8 * slot); barrier_arrive(full); }
      slot += 2;
      if (slot >= P.code_slots) { slot -= P.code_slots; slot_phase ^= 1u; }
    }
  } else if (warp == kB4MmaWarp) {
    // (the whole warp walks, and one lane issues: its operands are then uniform values. A single lane's walk took 1300 clocks a tile.)
    const bool one = elected();
    int x0 = 0;
    uint32_t a = tmem + kB4SumColumns, w_bar = w_full, wp = 0u, xp = 0u, ap = 1u;
    const uint32_t other_a = a ^ (a + 2 * kB4OperandColumns), other_bar = w_full ^ (w_full + 8);    // (the two pairs in turn)
    const auto one_tile = [&](uint32_t form) {                              // x piece by piece
      barrier_wait(acc_empty, ap, given_up);                               // (the first pass finds it empty)
      for (int k0 = 0; k0 < H; k0 += kB4StepCols) {
        const int quarters = min(4, (H - k0) / kB4XCols);
        barrier_wait(w_bar, wp, given_up);
#pragma unroll
        for (int q = 0; q < 4; q++) {
          if (q < quarters) {
            const uint32_t x_bar = x_full + 8 * x0;
            barrier_wait(x_bar, xp, given_up);
            __syncwarp();
            if (one) {
              const uint64_t b = operand(smem_address(xs) + x0 * x_bytes);
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
              for (int k = 0; k < 4; k++) product_f16(tmem, a + 32 * q + 8 * k, b + 2 * k, form, q + k > 0 ? 1u : static_cast<uint32_t>(k0));
              products_commit(x_bar + 8 * kB4MaxXStages);                  // (x_empty)
            }
            if (++x0 == P.x_stages) { x0 = 0; xp ^= 1u; }
          }
        }
        if (one) products_commit(w_bar + 8 * kB4Pairs);                    // (w_empty)
        __syncwarp();
        a ^= other_a; w_bar ^= other_bar;
        wp ^= w_bar == w_full ? 1u : 0u;
      }
      if (one) products_commit(acc_full);
      __syncwarp();
    };
    const auto form_of = [](int n) { return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kB4Tile >> 4) << 24); };    // binary16 operands, FP32 accumulators
    const uint32_t form = form_of(P.n);
    for (int first = passes.begin; first < passes.end; first += P.per_pass, ap ^= 1u) {
      const int count = min(P.per_pass, passes.end - first);
      if (count == 1) { one_tile(form); continue; }
      for (int k0 = 0; k0 < H; k0 += kB4StepCols) {
        const int quarters = min(4, (H - k0) / kB4XCols);
        const bool last = k0 + kB4StepCols >= H;
        uint64_t b[4];                                                       // the step's places of x
        uint32_t x_bar[4], x_par[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const int x = x0 + q < P.x_stages ? x0 + q : x0 + q - P.x_stages;
          b[q] = operand(smem_address(xs) + x * x_bytes); x_bar[q] = x_full + 8 * x; x_par[q] = x0 + q < P.x_stages ? xp : xp ^ 1u;
        }
        uint32_t d = tmem;
        for (int sum = 0; sum < count; sum++, d += static_cast<uint32_t>(P.column_stride)) {
          if (k0 == 0) barrier_wait(acc_empty + 8 * sum, ap, given_up);                    // (the first pass finds them empty)
          barrier_wait(w_bar, wp, given_up);
          if (sum == 0 || sum == count - 1 || quarters < 4) {                // x arrives, or leaves
#pragma unroll
            for (int q = 0; q < 4; q++) {
              if (q < quarters) {
                if (sum == 0) barrier_wait(x_bar[q], x_par[q], given_up);
                __syncwarp();
                if (one) {
                  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                  for (int k = 0; k < 4; k++) product_f16(d, a + 32 * q + 8 * k, b[q] + 2 * k, form, q + k > 0 ? 1u : static_cast<uint32_t>(k0));
                  if (sum == count - 1) products_commit(x_bar[q] + 8 * kB4MaxXStages);     // (x_empty)
                }
              }
            }
          } else if (one) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int q = 0; q < 4; q++) {
#pragma unroll
              for (int k = 0; k < 4; k++) product_f16(d, a + 32 * q + 8 * k, b[q] + 2 * k, form, q + k > 0 ? 1u : static_cast<uint32_t>(k0));
            }
          }
          if (one) {
            products_commit(w_bar + 8 * kB4Pairs);                           // (w_empty)
            if (last) products_commit(acc_full + 8 * sum);
          }
          __syncwarp();
          a ^= other_a; w_bar ^= other_bar;
          wp ^= w_bar == w_full ? 1u : 0u;
        }
        x0 += quarters;
        if (x0 >= P.x_stages) { x0 -= P.x_stages; xp ^= 1u; }
      }
    }
    if (passes.left.count > 0) one_tile(form_of(passes.left.n));
    if (*given_up && one) {                                                 // what is under way ends before the block does
      products_commit(drained);
      for (uint32_t i = 0; i < kWait4Limit && !barrier_try(drained, 0u); i++) {}
    }
  } else if (warp == kB4CopyWarp) {
    after_predecessor();                                                    // (the weight's copies do not wait for the preparation of x: see lm_head_nvfp4_kernel)
    if (lane == 0) {
      int stage = 0, issued = 0; uint32_t phase = 0u;
      bool go = true;
      for (int i = 0; go && passes.get(i, pass); i++) {
        const uint32_t bytes = static_cast<uint32_t>(pass.n * kB4XCols * 2);
        for (int k = 0; k < H / kB4XCols; k++) {
          go = barrier_wait(x_empty + 8 * stage, phase ^ 1u, given_up);
          if (!go) break;
          barrier_expect(x_full + 8 * stage, bytes);
          bulk_copy(smem_address(xs) + stage * x_bytes, P.xt + static_cast<size_t>(k) * x_bytes + pass.r0 * (kB4XCols * 2), bytes, x_full + 8 * stage);
          issued++;
          if (++stage == P.x_stages) { stage = 0; phase ^= 1u; }
        }
      }
      if (!go)                                                              // the copies under way
        for (int k = 0; k < P.x_stages && k < issued; k++) {
          if (stage == 0) { stage = P.x_stages; phase ^= 1u; }
          stage--;
          for (uint32_t i = 0; i < kWait4Limit && !barrier_try(x_full + 8 * stage, phase); i++) {}
        }
    }
  } else if (warp == kB4CodeWarp) {
    if (lane == 0) {
      bool go = true;
      int issued = 0, slot = 0;
      uint32_t phase = 0u;
      for (int i = 0; go && passes.get(i, pass); i++) {
        for (int step = 0; go && step < steps; step++) {
          for (int tile = pass.first; tile < pass.first + pass.count; tile++) {
            const uint32_t bar = c_full + 8 * slot;
            go = barrier_wait(c_empty + 8 * slot, phase ^ 1u, given_up);
            if (!go) break;
            barrier_expect(bar, kB4SlotBytes);
            tile_copy(smem_address(cs) + slot * kB4CodeBytes, &code_map, step * (kB4StepCols / 2), tile * kB4Tile, bar);
            tile_copy(smem_address(ss) + slot * (kB4SlotBytes - kB4CodeBytes), &scale_map, step * (kB4StepCols / kFp4Block), tile * kB4Tile, bar);
            issued++;
            if (++slot == P.code_slots) { slot = 0; phase ^= 1u; }
          }
        }
      }
      if (!go)                                                              // the copies under way
        for (int k = 0; k < P.code_slots && k < issued; k++) {
          if (slot == 0) { slot = P.code_slots; phase ^= 1u; }
          slot--;
          for (uint32_t i = 0; i < kWait4Limit && !barrier_try(c_full + 8 * slot, phase); i++) {}
        }
    }
  } else {
    // ---- finished accumulators: a warp has 32 vocabulary rows of every tile; a column is a row of logits
    after_predecessor();
    const int part = warp & 3;
    const uint32_t row_bytes = static_cast<uint32_t>(P.logits_stride * 2);
    const float g = __ldg(P.scale);
    bool go = true, plain = true, bad = false;                              // plain: every g * 2^-shift is a normal binary32, with room for the sum
    for (int r = lane; r < P.n; r += 32) {                                  // (each of these warps looks at all rows and writes down a quarter of them)
      const double f = static_cast<double>(g) * __hiloint2double((1023 - P.shift[r]) << 20, 0);
      plain &= fabs(f) >= 0x1p-100 && fabs(f) <= 0x1p80;
      if ((r >> 5) % kB4DoneWarps == warp - kB4FirstDoneWarp) factor[r] = static_cast<float>(f);
      bad |= P.bad[r] != 0;
    }
    if (bad) words[2] = 1u;
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kB4DoneWarps) : "memory");    // factors are read by other lanes and warps than wrote them: a vote does not order them
    plain = __all_sync(kFull, plain);
    uint32_t phase = 0u;
    for (int i = 0; go && passes.get(i, pass); i++, phase ^= 1u) {
      for (int sum = 0; sum < pass.count; sum++) {
        const int tile = pass.first + sum;
        go = __all_sync(kFull, barrier_wait(acc_full + 8 * sum, phase, given_up));
        if (!go) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const int v = tile * kB4Tile + part * 32 + lane, rows = min(P.rows, pass.r0 + pass.n);
        for (int r0 = pass.r0 + 32 * ((warp - kB4FirstDoneWarp) >> 2); r0 < pass.r0 + pass.n; r0 += 8 * kB4DoneWarps) {
          uint32_t a[32];
          __syncwarp();                                                      // (a load by the whole warp, behind stores by some of its lanes)
          accumulators32(tmem + (static_cast<uint32_t>(part * 32) << 16) + static_cast<uint32_t>(sum * P.column_stride + r0 - pass.r0), a);
          uint16_t* out = P.logits + r0 * P.logits_stride + v;
          if (!plain) {
            for (int j = 0; j < 32; j++)
              if (v < P.vocab && r0 + j < rows) out[j * P.logits_stride] = f32_to_bf16(head4_finish(__uint_as_float(picked(a, j)), g, P.shift[r0 + j]));
          } else {
            const int there = v < P.vocab ? rows - r0 : 0;                  // rows of logits among the 32
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 f = *reinterpret_cast<const float4*>(factor + r0 + j);
              const float fj[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
              for (int e = 0; e < 4; e++)
                if (j + e < there) *reinterpret_cast<uint16_t*>(reinterpret_cast<unsigned char*>(out) + static_cast<uint64_t>(row_bytes) * static_cast<uint32_t>(j + e)) = f32_to_bf16(__fmul_rn(__uint_as_float(a[j + e]), fj[e]));
            }
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) barrier_arrive(acc_empty + 8 * sum);
      }
    }
  }
  __syncwarp();
  after_predecessor();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == kB4MmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  // ---- rows whose x is no binary16 after the scaling, or (a wait ran out) everything of this block's
  const bool all = *given_up != 0u;
  for (int r = 0; r < P.rows && (all || words[2]); r++) {                   // (256 looks one after the other took 10 us and more)
    if (!all && !P.bad[r]) continue;
    const uint16_t* x = P.xb + static_cast<size_t>(r) * H;
    for (int i = 0; passes.get(i, pass); i++) {
      if (r < pass.r0 || r >= pass.r0 + pass.n) continue;
      for (int v = pass.first * kB4Tile + warp; v < min((pass.first + pass.count) * kB4Tile, P.vocab); v += kB4Threads / 32) {
        const float z = all ? __int_as_float(0x7FC00000) : head4_finish(exact_sum(x, P.codes + v * P.codes_stride, P.scales + v * P.scales_stride, H, lane), __ldg(P.scale), 0);
        if (lane == 0) P.logits[r * P.logits_stride + v] = f32_to_bf16(z);
      }
    }
  }
}

}  // namespace lm
