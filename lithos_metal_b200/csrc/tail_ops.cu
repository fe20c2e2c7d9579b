// C ABI of the operators between the projection and the sampler: the microscaled 4-bit weight, the projection with it, and the logits' processing. As in
// lithos_b200.cu: argument checks, launch geometry, kernel launches; no allocation, no synchronisation.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "common.cuh"
#include "host.cuh"
#include "lm_head_nvfp4.cuh"
#include "lm_head_nvfp4_batch.cuh"
#include "logits.cuh"
#include "nvfp4.cuh"

using namespace lm;

namespace {

bool misaligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

// The sizes of a matrix in the 4-bit format (nvfp4.cuh).
int fp4_matrix_ok(int64_t rows, int64_t cols, const void* codes, int64_t codes_stride, const void* scales, int64_t scales_stride, const void* scale) {
  if (!codes || !scales || !scale || codes_stride < cols / 2 || scales_stride < cols / kFp4Block) return LM_E_INVALID;
  if (cols % kFp4Block != 0 || cols > 0x7FFFFFFF || rows > 0x7FFFFFFF) return LM_E_UNSUPPORTED;
  return LM_OK;
}

// Blocks of a grid-stride kernel over `items` threads' work.
unsigned stride_grid(long long items, int threads, int sms, int per_sm) {
  const long long want = (items + threads - 1) / threads, most = static_cast<long long>(sms) * per_sm;
  return static_cast<unsigned>(want < most ? want : most);
}

}  // namespace

extern "C" {

int lm_quantize_nvfp4(const lm_quantize_nvfp4_args* a) {
  if (!a || a->struct_size != sizeof(lm_quantize_nvfp4_args)) return LM_E_INVALID;
  if (a->rows < 0 || a->cols < 0 || (a->dtype != LM_DTYPE_BF16 && a->dtype != LM_DTYPE_F32)) return LM_E_INVALID;
  if (a->rows == 0 || a->cols == 0) return LM_OK;
  if (!a->x || a->row_stride < a->cols || (a->find_scale && !a->amax)) return LM_E_INVALID;
  int rc = fp4_matrix_ok(a->rows, a->cols, a->codes, a->codes_stride, a->scales, a->scales_stride, a->scale);
  if (rc != LM_OK) return rc;
  int sms = 0;
  rc = sm_count(&sms);
  if (rc != LM_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(a->stream);
  QuantDev P;
  P.x = a->x; P.dtype = a->dtype; P.rows = a->rows; P.cols = static_cast<int>(a->cols); P.row_stride = a->row_stride;
  P.scale = a->scale; P.amax = static_cast<uint32_t*>(a->amax); P.find = a->find_scale ? 1 : 0;
  P.codes = a->codes; P.codes_stride = a->codes_stride; P.scales = a->scales; P.scales_stride = a->scales_stride;
  const long long blocks = a->rows * (a->cols / kFp4Block);
  const unsigned grid = stride_grid(blocks, kQuantThreads, sms, 8);
  const bool f32 = a->dtype == LM_DTYPE_F32;
  if (P.find) {
    const cudaError_t e = cudaMemsetAsync(P.amax, 0, sizeof(uint32_t), st);
    if (e != cudaSuccess) return cuda_fail(e);
    rc = f32 ? launch_stream(false, nvfp4_amax_kernel<true>, dim3(grid), kQuantThreads, 0, 1, st, P)
             : launch_stream(false, nvfp4_amax_kernel<false>, dim3(grid), kQuantThreads, 0, 1, st, P);
    if (rc != LM_OK) return rc;
  }
  return f32 ? launch_stream(false, nvfp4_quantize_kernel<true>, dim3(grid), kQuantThreads, 0, 1, st, P)
             : launch_stream(false, nvfp4_quantize_kernel<false>, dim3(grid), kQuantThreads, 0, 1, st, P);
}

int lm_dequantize_nvfp4(const lm_dequantize_nvfp4_args* a) {
  if (!a || a->struct_size != sizeof(lm_dequantize_nvfp4_args)) return LM_E_INVALID;
  if (a->rows < 0 || a->cols < 0) return LM_E_INVALID;
  if (a->rows == 0 || a->cols == 0) return LM_OK;
  if (!a->out || a->out_stride < a->cols) return LM_E_INVALID;
  int rc = fp4_matrix_ok(a->rows, a->cols, a->codes, a->codes_stride, a->scales, a->scales_stride, a->scale);
  if (rc != LM_OK) return rc;
  int sms = 0;
  rc = sm_count(&sms);
  if (rc != LM_OK) return rc;
  DequantDev P{a->codes, a->codes_stride, a->scales, a->scales_stride, a->scale, a->rows, static_cast<int>(a->cols), a->out, a->out_stride};
  return launch_stream(false, nvfp4_dequantize_kernel, dim3(stride_grid(a->rows * (a->cols / 4), kQuantThreads, sms, 8)), kQuantThreads, 0, 1, static_cast<cudaStream_t>(a->stream), P);
}

// Whether the mma.sync kernel takes the call: 16 rows at most (its products grow by eights of rows, the other kernel's conversion of the weight is the same for all), and two eights only where
// shared memory holds them. Measured, mma.sync against tcgen05: 16 rows of 50,257 x 4096 38.9 and 47.2 us, of 20,011 x 1024 10.9 and 13.2, of 4,099 x 4096 11.6 and 18.2, of 151,936 x 4096
// 89.8 and 94.6, of 128,000 x 2048 44.8 and 43.7; 24 rows (with three eights) 50.7 and 47.2, 12.8 and 13.3, 13.0 and 18.1, 125.6 and 96.5, 55.5 and 44.6.
static bool head4_few_rows(int64_t rows, int64_t hidden) {
  const int64_t nt = (rows + kH4Rows - 1) / kH4Rows;
  return nt <= 1 || (nt <= kH4MaxNT && head4_smem_bytes(static_cast<int>(hidden), static_cast<int>(nt)) <= 200 * 1024);
}

size_t lm_head_nvfp4_workspace_bytes(int64_t rows, int64_t hidden_dim) {
  if (rows < 1 || hidden_dim < 1 || rows > LM_HEAD_NVFP4_MAX_ROWS || hidden_dim > kH4MaxHidden) return 0;
  return x4_workspace_bytes(rows, hidden_dim);
}

static int head_nvfp4_few(void (*kernel)(Head4Dev), const lm_head_nvfp4_args* a, const Rows4Dev& R, int nt, int sms) {
  Head4Dev P;
  P.rows = R.rows; P.codes = a->codes; P.codes_stride = a->codes_stride; P.scales = a->scales; P.scales_stride = a->scales_stride; P.scale = a->scale;
  P.hidden = R.hidden; P.vocab = static_cast<int>(a->vocab);
  P.xt = R.xt; P.xb = R.xb; P.shift = R.shift; P.bad = R.bad; P.logits = static_cast<uint16_t*>(a->logits); P.logits_stride = a->logits_stride;
  const size_t smem = head4_smem_bytes(P.hidden, nt);
  const int rc = ensure_dynamic_smem(static_cast<KernelSlot>(kSlotHeadNvfp4 + nt - 1), reinterpret_cast<const void*>(kernel), smem);
  if (rc != LM_OK) return rc;
  const int tiles = (P.vocab + kH4Tile - 1) / kH4Tile;
  return launch_stream(true, kernel, dim3(static_cast<unsigned>(tiles < sms ? tiles : sms)), kH4Threads, smem, 1, static_cast<cudaStream_t>(a->stream), P);
}

// A matrix of bytes that the copy engine reads in boxes of 128 rows by `width` bytes.
static int byte_map(const uint8_t* p, int64_t rows, int64_t bytes, int64_t stride, uint32_t width, CUtensorMapSwizzle swizzle, CUtensorMap* map) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<Encode> known{nullptr};
  Encode encode = known.load(std::memory_order_relaxed);
  if (!encode) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found);
    if (e != cudaSuccess) return cuda_fail(e);
    if (found != cudaDriverEntryPointSuccess || !f) return cuda_fail(cudaErrorSymbolNotFound);
    known.store(encode = reinterpret_cast<Encode>(f), std::memory_order_relaxed);
  }
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(bytes), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(stride)};
  const cuuint32_t box[2] = {width, kB4Tile}, steps[2] = {1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(p), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? LM_OK : cuda_fail(cudaErrorInvalidValue);
}

// More rows: a launch for every 256 of them.
static int head_nvfp4_batch(const lm_head_nvfp4_args* a, const Rows4Dev& R, int sms) {
  cudaStream_t st = static_cast<cudaStream_t>(a->stream);
  Batch4Dev P;
  P.codes = a->codes; P.codes_stride = a->codes_stride; P.scales = a->scales; P.scales_stride = a->scales_stride; P.scale = a->scale;
  P.hidden = R.hidden; P.vocab = static_cast<int>(a->vocab); P.logits_stride = a->logits_stride;
  int rc = ensure_dynamic_smem(kSlotHeadNvfp4Batch, reinterpret_cast<const void*>(lm_head_nvfp4_batch_kernel), kB4SmemLimit);
  if (rc != LM_OK) return rc;
  CUtensorMap code_map, scale_map;
  rc = byte_map(a->codes, P.vocab, P.hidden / 2, a->codes_stride, kB4StepCols / 2, CU_TENSOR_MAP_SWIZZLE_128B, &code_map);
  if (rc == LM_OK) rc = byte_map(a->scales, P.vocab, P.hidden / kFp4Block, a->scales_stride, kB4StepCols / kFp4Block, CU_TENSOR_MAP_SWIZZLE_NONE, &scale_map);
  if (rc != LM_OK) return rc;
  const int tiles = (P.vocab + kB4Tile - 1) / kB4Tile;
  for (int64_t r = 0; r < a->rows; r += kB4MaxN) {
    P.rows = static_cast<int>(a->rows - r < kB4MaxN ? a->rows - r : kB4MaxN);
    P.n = x4_padded(P.rows);
    P.xt = R.xt + static_cast<size_t>(r) * R.hidden * 2; P.xb = R.xb + static_cast<size_t>(r) * R.hidden; P.shift = R.shift + r; P.bad = R.bad + r;
    P.logits = static_cast<uint16_t*>(a->logits) + r * a->logits_stride;
    P.column_stride = P.n <= 32 ? 32 : P.n <= 64 ? 64 : P.n <= 128 ? 128 : 256;
    P.per_pass = kB4SumColumns / P.column_stride;
    // of x eight pieces in shared memory (a step's four and the next's, where tiles share them) or as many as fit beside two tiles of codes, and as many of these as fit then: an even number
    // (batch kernel: a place's codes are then always the same pair's)
    P.x_stages = static_cast<int>((kB4SmemLimit - batch4_smem_bytes(P.n, 2, 0)) / static_cast<size_t>(batch4_x_stage_bytes(P.n)));
    if (P.x_stages > kB4MaxXStages) P.x_stages = kB4MaxXStages;
    P.code_slots = kB4MaxCodeSlots;
    while (batch4_smem_bytes(P.n, P.code_slots, P.x_stages) > kB4SmemLimit) P.code_slots -= 2;
    // Left over, or all there are: as many blocks to each as there are blocks, or sixteens of rows.
    P.each = tiles / sms; P.left = tiles % sms;
    P.left_blocks = P.left == 0 ? 1 : sms / P.left < P.n / 16 ? sms / P.left : P.n / 16;
    P.left_n = ((P.n + P.left_blocks - 1) / P.left_blocks + 15) / 16 * 16;
    P.left_blocks = (P.n + P.left_n - 1) / P.left_n;
    const int grid = P.each > 0 ? sms : P.left * P.left_blocks;
    rc = launch_stream(true, lm_head_nvfp4_batch_kernel, dim3(static_cast<unsigned>(grid)), kB4Threads, batch4_smem_bytes(P.n, P.code_slots, P.x_stages), 1, st, code_map, scale_map, P);
    if (rc != LM_OK) return rc;
  }
  return LM_OK;
}

int lm_head_nvfp4(const lm_head_nvfp4_args* given) {
  if (!given || given->struct_size != sizeof(lm_head_nvfp4_args)) return LM_E_INVALID;
  lm_head_nvfp4_args one = *given;
  const lm_head_nvfp4_args* const a = &one;
  if (a->rows < 0 || a->vocab < 0 || a->hidden_dim < 1) return LM_E_INVALID;
  if (a->rows == 0 || a->vocab == 0) return LM_OK;
  // what lies between rows is of no account where there is one
  if (a->rows == 1 && a->hidden_stride >= a->hidden_dim && a->logits_stride >= a->vocab) { one.hidden_stride = a->hidden_dim; one.logits_stride = a->vocab; }
  if (a->vocab == 1 && a->codes_stride >= a->hidden_dim / 2 && a->scales_stride >= a->hidden_dim / kFp4Block) {
    one.codes_stride = (a->hidden_dim / 2 + 15) / 16 * 16; one.scales_stride = (a->hidden_dim / kFp4Block + 15) / 16 * 16;
  }
  if (!a->hidden || !a->logits || a->hidden_stride < a->hidden_dim || a->logits_stride < a->vocab) return LM_E_INVALID;
  int rc = fp4_matrix_ok(a->vocab, a->hidden_dim, a->codes, a->codes_stride, a->scales, a->scales_stride, a->scale);
  if (rc != LM_OK) return rc;
  if (a->rows > LM_HEAD_NVFP4_MAX_ROWS || a->vocab > LM_MAX_VOCAB || (a->hidden_dim % 64) != 0 || a->hidden_dim > kH4MaxHidden) return LM_E_UNSUPPORTED;
  if (a->codes_stride > 0x7FFFFFFF || a->scales_stride > 0x7FFFFFFF || a->logits_stride > 0x3FFFFFFF) return LM_E_UNSUPPORTED;
  if (misaligned(a->codes, 16) || (a->codes_stride % 16) != 0 || misaligned(a->scales, 16) || (a->scales_stride % 16) != 0) return LM_E_UNSUPPORTED;   // 16-byte copies
  if (!a->workspace || misaligned(a->workspace, 256) || a->workspace_bytes < x4_workspace_bytes(a->rows, a->hidden_dim)) return LM_E_WORKSPACE;
  int sms = 0;
  rc = sm_count(&sms);
  if (rc != LM_OK) return rc;
  Rows4Dev R;
  unsigned char* ws = static_cast<unsigned char*>(a->workspace);
  const int padded = x4_padded(a->rows);
  R.x = static_cast<const uint16_t*>(a->hidden); R.x_stride = a->hidden_stride; R.rows = static_cast<int>(a->rows); R.hidden = static_cast<int>(a->hidden_dim);
  R.gamma = static_cast<const uint16_t*>(a->norm_weight); R.eps = a->eps; R.one_plus = a->one_plus; R.few = head4_few_rows(a->rows, a->hidden_dim) ? 1 : 0;
  R.xt = ws; ws += x4_xt_bytes(a->rows, a->hidden_dim);
  R.xb = reinterpret_cast<uint16_t*>(ws); ws += x4_xb_bytes(a->rows, a->hidden_dim);
  R.shift = reinterpret_cast<int*>(ws); R.bad = R.shift + padded;
  rc = launch_beside(nvfp4_rows_kernel, dim3(static_cast<unsigned>(R.few ? R.rows : padded)), kX4Threads, 0, 1, static_cast<cudaStream_t>(a->stream), R);
  if (rc != LM_OK) return rc;
  if (!R.few) return head_nvfp4_batch(a, R, sms);
  return a->rows <= kH4Rows ? head_nvfp4_few(lm_head_nvfp4_kernel<1, 4>, a, R, 1, sms) : head_nvfp4_few(lm_head_nvfp4_kernel<2, 3>, a, R, 2, sms);
}

// Whether writing `out` can change what is read of `in` (both [rows, vocab] in elements of `size` bytes): same place and strides is in place, sharing nothing is fine.
static int logits_overlap(const lm_logits_args* a, int64_t size, bool* same) {
  const uintptr_t in = reinterpret_cast<uintptr_t>(a->logits), out = reinterpret_cast<uintptr_t>(a->out);
  *same = in == out && (a->rows == 1 || a->row_stride == a->out_stride);
  if (*same) return LM_OK;
  const uintptr_t row = static_cast<uintptr_t>(a->vocab * size);
  const uintptr_t in_end = in + static_cast<uintptr_t>((a->rows - 1) * a->row_stride * size) + row, out_end = out + static_cast<uintptr_t>((a->rows - 1) * a->out_stride * size) + row;
  if (in_end <= out || out_end <= in) return LM_OK;
  if (a->row_stride != a->out_stride) return LM_E_INVALID;
  const uintptr_t stride = static_cast<uintptr_t>(a->row_stride * size), gap = (out > in ? out - in : in - out) % stride;    // columns of one wider matrix
  return gap >= row && stride - gap >= row ? LM_OK : LM_E_INVALID;
}

int lm_process_logits(const lm_logits_args* a) {
  if (!a || a->struct_size != sizeof(lm_logits_args)) return LM_E_INVALID;
  if (a->rows < 0 || a->vocab < 0 || (a->dtype != LM_DTYPE_BF16 && a->dtype != LM_DTYPE_F32)) return LM_E_INVALID;
  if (a->rows == 0 || a->vocab == 0) return LM_OK;
  if (!a->logits || !a->out || a->row_stride < a->vocab || a->out_stride < a->vocab) return LM_E_INVALID;
  if (a->history && (a->hist_len < 0 || a->hist_stride < 0)) return LM_E_INVALID;
  if (a->history && a->repetition == nullptr && !(a->repetition_s > 0.0f)) return LM_E_INVALID;
  if (a->bias_len < 0 || (a->bias_len > 0 && (!a->bias_ids || !a->bias_values || a->bias_ids_stride < 0 || a->bias_values_stride < 0))) return LM_E_INVALID;
  if (a->mask && (a->mask_stride < (a->vocab + 31) / 32 || a->mask_count < (a->mask_rows ? 0 : a->rows))) return LM_E_INVALID;
  if (a->vocab > LM_MAX_VOCAB || a->rows > 0x7FFFFFFF || (a->history && a->hist_len > kLogitsMaxHistory) || a->bias_len > kLogitsMaxBias || a->mask_count > 0x7FFFFFFF) return LM_E_UNSUPPORTED;
  const int64_t size = a->dtype == LM_DTYPE_F32 ? 4 : 2;
  if (misaligned(a->logits, static_cast<size_t>(size)) || misaligned(a->out, static_cast<size_t>(size))) return LM_E_INVALID;
  bool same = false;
  int rc = logits_overlap(a, size, &same);
  if (rc != LM_OK) return rc;
  const bool lists = (a->history && a->hist_len > 0) || a->bias_len > 0;
  if (same && !lists && !a->mask) return LM_OK;                             // nothing to do
  int sms = 0;
  rc = sm_count(&sms);
  if (rc != LM_OK) return rc;
  LogitsDev P;
  P.in = a->logits; P.in_stride = a->row_stride; P.out = a->out; P.out_stride = a->out_stride; P.in_place = same ? 1 : 0;
  P.rows = static_cast<int>(a->rows); P.vocab = static_cast<int>(a->vocab);
  P.history = a->hist_len > 0 ? a->history : nullptr; P.hist_len = static_cast<int>(a->hist_len); P.hist_stride = a->hist_stride; P.lengths = a->history_len; P.prompts = a->prompt_len;
  P.rho = a->repetition; P.rho_s = a->repetition_s; P.pi = a->presence; P.pi_s = a->presence_s; P.phi = a->frequency; P.phi_s = a->frequency_s;
  P.bias_ids = a->bias_ids; P.bias_ids_stride = a->bias_ids_stride; P.bias_values = a->bias_values; P.bias_values_stride = a->bias_values_stride; P.bias_len = static_cast<int>(a->bias_len);
  P.mask = a->mask; P.mask_stride = a->mask_stride; P.mask_rows = a->mask_rows; P.mask_count = static_cast<int>(a->mask_count);
  const bool f32 = a->dtype == LM_DTYPE_F32;
  cudaStream_t st = static_cast<cudaStream_t>(a->stream);
  const long long at_once = static_cast<long long>(kLogitsPerSM) * sms;
  P.table_log2 = 0;
  if (!lists) {
    // slices of as many logits as a block takes at once, shorter ones where these would leave SMs idle
    const long long per = f32 ? kMaskSlice<true> : kMaskSlice<false>, few = (static_cast<long long>(a->rows) * a->vocab + kMaskPerSM * sms - 1) / (kMaskPerSM * sms);
    P.slice = static_cast<int>(((few < per ? few : per) + 31) / 32 * 32);
    if (P.slice < kLogitsMinSlice) P.slice = kLogitsMinSlice;
    P.slices = static_cast<int>((a->vocab + P.slice - 1) / P.slice);
    const long long items = static_cast<long long>(P.rows) * P.slices;
    if (items > 0x7FFFFFFF) return LM_E_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>(items));
    return f32 ? launch_beside(logits_mask_kernel<true>, grid, kMaskThreads, 0, 1, st, P) : launch_beside(logits_mask_kernel<false>, grid, kMaskThreads, 0, 1, st, P);
  }
  // A block to a row, or to a slice of one. One block to an SM while the slices are short (the launch is then made ready beside its predecessor). Otherwise the number of slices for which the rounds
  // of kLogitsPerSM blocks to an SM are cheapest, a block's lists counted as the bytes that it could pass on meanwhile, and no slice so wide that what a round reads leaves L2 before the listed
  // tokens are read again. (History of 2048 and 300 biases, 151,936 wide: 128 rows 28.7 us in 3 slices, 45 in 1, 37 in 8; 256 rows 49, 55, 59; 4096 rows in 2 slices 516, in 1 547, in 4 551.)
  // Lists that are longer than the hash table takes: slices no wider than a word per token takes.
  const long long names = (P.history ? P.hist_len : 0) + P.bias_len, total = static_cast<long long>(a->rows) * a->vocab;
  long long slices = 1;
  if (total <= 16384LL * sms) slices = sms / a->rows;
  else {
    double best = 0.0;
    for (long long n = (a->vocab * size + kLogitsSliceBytes - 1) / kLogitsSliceBytes, last = n + 12; n <= last; n++) {
      const double rounds = static_cast<double>((n * a->rows + at_once - 1) / at_once), cost = rounds * static_cast<double>((a->vocab + n - 1) / n * size + 6144 + 8 * names);
      if (best == 0.0 || cost < best) { best = cost; slices = n; }
    }
  }
  if (slices < 1) slices = 1;
  if (slices > (a->vocab + kLogitsMinSlice - 1) / kLogitsMinSlice) slices = (a->vocab + kLogitsMinSlice - 1) / kLogitsMinSlice;
  const long long widest = names > kLogitsMaxNamed ? kLogitsMaxDirect : kLogitsMaxSlice;
  if (slices < (a->vocab + widest - 1) / widest) slices = (a->vocab + widest - 1) / widest;
  P.slice = static_cast<int>(((a->vocab + slices - 1) / slices + 31) / 32 * 32);
  P.slices = static_cast<int>((a->vocab + P.slice - 1) / P.slice);
  P.table_log2 = 8;
  while ((3LL << P.table_log2) < 4 * names) P.table_log2++;                 // three quarters full at most
  if (P.slice <= 2LL << P.table_log2) P.table_log2 = 0;                     // (no larger than the hash table: a word per token)
  const size_t smem = (P.table_log2 ? size_t{8} << P.table_log2 : static_cast<size_t>(P.slice) * 4) + static_cast<size_t>(P.slice) / 8 + 32;
  const bool bias = a->bias_len > 0;
  static void (*const kernels[8])(LogitsDev) = {logits_kernel<false, false, false>, logits_kernel<false, false, true>, logits_kernel<false, true, false>, logits_kernel<false, true, true>,
                                                logits_kernel<true, false, false>, logits_kernel<true, false, true>, logits_kernel<true, true, false>, logits_kernel<true, true, true>};
  const int which = (f32 ? 4 : 0) + (bias ? 2 : 0) + (P.mask ? 1 : 0);
  void (*const kernel)(LogitsDev) = kernels[which];
  rc = ensure_dynamic_smem(static_cast<KernelSlot>(kSlotLogits + which), reinterpret_cast<const void*>(kernel), smem);
  if (rc != LM_OK) return rc;
  const long long items = static_cast<long long>(P.rows) * P.slices;
  if (items > 0x7FFFFFFF) return LM_E_UNSUPPORTED;
  return launch_beside(kernel, dim3(static_cast<unsigned>(items)), bias ? kLogitsThreads<true> : kLogitsThreads<false>, smem, 1, st, P);
}

}  // extern "C"
