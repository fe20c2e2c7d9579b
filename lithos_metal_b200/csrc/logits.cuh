// The logits' processing in front of the sampler: penalties for repeated tokens, biases by token, and grammar masks, rounded once to the logits' type.
//
// Per row r, with c_all the occurrences of a token in history[r, :len] and c_out those from position prompt_len on:
//   z = float(logit); c_all > 0: z = z > 0 ? z / rho : z * rho; c_out > 0: z = (z - pi) - phi * c_out; z += the token's biases, in list order; masked: -inf.
// The penalties touch as many logits as the history has tokens, the biases as many as their list; a mask usually touches most. A block has a row, or a slice of one where there are few. It
// looks through the row's lists once: a bit in shared memory for every token of the history in its slice, and a table of these and the biased tokens with their counts: a word for every token of
// the slice, or where that is smaller a hash table (its size is given by the lists' lengths: it never fills up). Then it streams the slice, 16 bytes a load, four under way per thread: copied and masked (in place: only what changes is
// written, and read where a mask keeps some of eight), and logits whose bit is set are looked up and penalised right behind their chunk. Tokens with a bias are set behind that, by their
// (first) entry of the list. In place without a mask only the tokens that the lists name are touched.
// Bound by HBM where there are many rows: 4096 rows of 151,936 with histories of 2048 395 us, 6.4 TB/s = 0.98 of the copy rate; 1024 rows with biases and masks as well 129 us (98 for the bytes); 256 41 (24.5);
// 64 rows of 262,144 in place under masks 12.6 (a fill of as many bytes: 12.5). A few rows: launch, the lists and one trip to memory, 8 rows 6.6 us, 1 row 4.5. Blocks look through their lists before
// they stream, and few rows are few rounds of blocks: that is what the middle sizes lose. In place with a history of 2048 and without a mask 4096 rows take 330 us: lists and tables, and 2048 scattered lines a row.
// Where logits and result lie differently against 16 bytes they pass singly: 4096 rows of 50,257 from rows of 50,304 with a history 849 us into a tensor of 50,257 columns, 242 into one of 50,304; with a mask alone 621 and 129.
#pragma once
#include "common.cuh"

namespace lm {

// (Without biases more warps pay, 1024 rows with a history 121 us, with 384 threads 127; with them the compiler needs the registers: with 512 threads 147 us, spilling, with 384 127.)
template <bool kBias> constexpr int kLogitsThreads = kBias ? 384 : 512;
constexpr int kLogitsPerSM = 3;              // blocks
constexpr int kLogitsMinSlice = 1024;
constexpr int kLogitsSliceBytes = 160 * 1024;
constexpr int kLogitsMaxNamed = 12288;       // tokens in a hash table at most (16384 entries, 128 KB); longer lists: slices of
constexpr int kLogitsMaxDirect = 24576;      // at most so many tokens (96 KB)
constexpr int kLogitsMaxSlice = 524288;      // and never wider than this (64 KB of bits)

struct LogitsDev {
  const void* in; int64_t in_stride; void* out; int64_t out_stride; int in_place;
  int rows; int vocab;
  const int32_t* history; int hist_len; int64_t hist_stride; const int32_t* lengths; const int32_t* prompts;
  const float* rho; float rho_s; const float* pi; float pi_s; const float* phi; float phi_s;
  const int32_t* bias_ids; int64_t bias_ids_stride; const float* bias_values; int64_t bias_values_stride; int bias_len;
  const uint32_t* mask; int64_t mask_stride; const int32_t* mask_rows; int mask_count;
  int slice; int slices; int table_log2;     // the hash table has 2^table_log2 entries; 0: a word for every token of the slice
};

// a token's counts
constexpr uint32_t kOutMask = 0x1FFFFu;      // bits 0..16: occurrences behind the prompt
constexpr uint32_t kBiasOne = 1u << 17;      // bits 17..29: its biases (8191 at most)
constexpr uint32_t kBiasMask = 0x1FFFu << 17;
constexpr uint32_t kSeen = 1u << 30;         // it occurs
constexpr int kLogitsMaxHistory = 65536;
constexpr int kLogitsMaxBias = 8191;

template <bool F32> __device__ __forceinline__ float logit_at(const void* row, int64_t i) {
  return F32 ? static_cast<const float*>(row)[i] : __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(row)[i]) << 16);
}
template <bool F32> __device__ __forceinline__ void set_logit(void* row, int64_t i, float z) {
  if (F32) static_cast<float*>(row)[i] = z; else static_cast<uint16_t*>(row)[i] = __bfloat16_as_ushort(__float2bfloat16_rn(z));
}

// Eight logits; those whose bit of `keep` is clear become -inf.
__device__ __forceinline__ uint32_t two_signs(uint32_t bytes, uint32_t which) {   // two of four bytes' top bits, 16 times each (0x9988: of bytes 0 and 1)
  uint32_t r;
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(r) : "r"(bytes), "r"(which));
  return r;
}
__device__ __forceinline__ uint32_t two_kept(uint32_t w, uint32_t keep) { return (w & keep) | (0xFF80FF80u & ~keep); }
template <bool F32> struct Chunk;
template <> struct Chunk<false> {
  uint4 q;
  __device__ __forceinline__ void load(const void* p) { q = *static_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(void* p) const { *static_cast<uint4*>(p) = q; }
  __device__ __forceinline__ void apply(uint32_t keep) {
    const uint32_t lo = (keep & 15u) * 0x10204080u, hi = (keep >> 4) * 0x10204080u;    // a bit to the top of each byte
    q.x = two_kept(q.x, two_signs(lo, 0x9988u)); q.y = two_kept(q.y, two_signs(lo, 0xBBAAu)); q.z = two_kept(q.z, two_signs(hi, 0x9988u)); q.w = two_kept(q.w, two_signs(hi, 0xBBAAu));
  }
  __device__ __forceinline__ void store_once(void* p) const { __stcs(static_cast<uint4*>(p), q); }
};
template <> struct Chunk<true> {
  uint32_t v[8];
  __device__ __forceinline__ void load(const void* p) {
    const uint4 a = *static_cast<const uint4*>(p), b = *(static_cast<const uint4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  __device__ __forceinline__ void store(void* p) const { static_cast<uint4*>(p)[0] = make_uint4(v[0], v[1], v[2], v[3]); static_cast<uint4*>(p)[1] = make_uint4(v[4], v[5], v[6], v[7]); }
  __device__ __forceinline__ void store_once(void* p) const { __stcs(static_cast<uint4*>(p), make_uint4(v[0], v[1], v[2], v[3])); __stcs(static_cast<uint4*>(p) + 1, make_uint4(v[4], v[5], v[6], v[7])); }
  __device__ __forceinline__ void apply(uint32_t keep) {
#pragma unroll
    for (int e = 0; e < 8; e++) if (!((keep >> e) & 1u)) v[e] = 0xFF800000u;
  }
};

// A lane's kAhead chunks of eight logits, kStride chunks apart (a block's threads): their bits of a mask, 8 for each. Where these begin at words, a lane loads the word of four lanes' chunks and the
// lanes exchange them (mask_ahead, and mask_bits when they are wanted), elsewhere every lane loads its own bytes. (With bytes everywhere 256 masked rows of 151,936 took 35 us, and 18.6 in place
// where nothing had to be written.)
template <int kAhead, int kStride> __device__ __forceinline__ uint32_t mask_ahead(const uint8_t* mask, int first, int chunk, int chunks, int lane) {   // first: chunk 0's token; chunk: the lane's first
  const int shift = first & 7;
  uint32_t bits = 0u;
  if ((first & 31) == 0) {
    const int c = chunk - lane + (lane >> 3) * kStride + 4 * (lane & 7);
    if (lane < 8 * kAhead && c < chunks) bits = __ldg(reinterpret_cast<const uint32_t*>(mask + (first >> 3) + c));
  } else {
    const uint8_t* p = mask + (first >> 3) + chunk;
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      if (chunk + kStride * u < chunks) {
        uint32_t k = __ldg(p + kStride * u);
        if (shift) k = ((k | static_cast<uint32_t>(__ldg(p + kStride * u + 1)) << 8) >> shift) & 0xFFu;     // (v + 7 is in the row, and so is its byte)
        bits |= k << (8 * u);
      }
    }
  }
  return bits;
}
template <int kAhead> __device__ __forceinline__ uint32_t mask_bits(uint32_t ahead, int first, int lane) {    // (by the whole warp)
  if ((first & 31) != 0) return ahead;
  uint32_t bits = 0u;
  const uint32_t byte = static_cast<uint32_t>(lane & 3) * 0x11u + 0x40u;      // that byte of both words
#pragma unroll
  for (int u = 0; u < kAhead; u += 2) {
    const uint32_t a = __shfl_sync(kFull, ahead, 8 * u + (lane >> 2)), b = __shfl_sync(kFull, ahead, 8 * u + 8 + (lane >> 2));
    bits |= (__byte_perm(a, b, byte) & 0xFFFFu) << (8 * u);
  }
  return bits;
}

// The tokens' counts in shared memory: a hash table with linear probing, or (log2 = 0) a word per token of the slice.
constexpr uint32_t kNoToken = 0xFFFFFFFFu;
struct TokenTable {
  uint32_t* word; int log2; int slice;                                      // hash entries: token and counts, side by side
  __device__ __forceinline__ TokenTable(unsigned char* smem, int log2_, int slice_) : word(reinterpret_cast<uint32_t*>(smem)), log2(log2_), slice(slice_) {}
  __device__ __forceinline__ int entries() const { return log2 ? 1 << log2 : slice; }   // (a multiple of 32)
  __device__ __forceinline__ uint32_t* end() const { return word + (log2 ? 2 << log2 : slice); }
  __device__ __forceinline__ uint32_t home(uint32_t v) const { return (v * 2654435769u) >> (32 - log2); }     // (2^32 over the golden ratio: neighbours lie apart)
  template <int kThreads> __device__ __forceinline__ void clear() const {     // and the bits behind it
    const int hashed = log2 ? 2 << log2 : 0, all = (log2 ? 2 << log2 : slice) + slice / 32;
    for (int i = 4 * threadIdx.x; i < all; i += 4 * kThreads) { const uint32_t k = i < hashed ? kNoToken : 0u; *reinterpret_cast<uint4*>(word + i) = make_uint4(k, 0u, k, 0u); }
  }
  __device__ __forceinline__ uint32_t* insert(uint32_t v) const {            // the token's counts
    if (!log2) return word + v;
    for (uint32_t i = home(v);; i = (i + 1u) & ((1u << log2) - 1u)) {
      const uint32_t k = atomicCAS(&word[2 * i], kNoToken, v);
      if (k == kNoToken || k == v) return &word[2 * i + 1];
    }
  }
  __device__ __forceinline__ uint32_t counts(uint32_t v) const {             // of a token that is there
    if (!log2) return word[v];
    uint32_t i = home(v);
    uint2 e = *reinterpret_cast<const uint2*>(word + 2 * i);
    while (e.x != v) { i = (i + 1u) & ((1u << log2) - 1u); e = *reinterpret_cast<const uint2*>(word + 2 * i); }
    return e.y;
  }
};

// A block's slice of a row: what the parts of the kernel below each work out for themselves (kept over the streaming loop, the lists' values were spilled there: 1024 rows of 151,936 with a history
// of 2048 tokens 150 us, with a bias that is never reached in the code behind the loop 180).
template <bool F32, bool kMask> struct Slice {
  int row, lo, hi; const unsigned char* in; unsigned char* out; const uint8_t* mask; bool nothing, stream;
  __device__ __forceinline__ explicit Slice(const LogitsDev& P) {
    uint32_t item = blockIdx.x;
    asm volatile("" : "+r"(item));
    constexpr int kSize = F32 ? 4 : 2;
    row = static_cast<int>(item / static_cast<uint32_t>(P.slices)); lo = (static_cast<int>(item) - row * P.slices) * P.slice; hi = min(lo + P.slice, P.vocab);
    in = static_cast<const unsigned char*>(P.in) + row * P.in_stride * kSize; out = static_cast<unsigned char*>(P.out) + row * P.out_stride * kSize;
    const int which = kMask && P.mask ? (P.mask_rows ? P.mask_rows[row] : row) : -1;
    nothing = which >= P.mask_count && which >= 0;                          // the row's mask does not exist: everything is masked
    mask = which >= 0 && !nothing ? reinterpret_cast<const uint8_t*>(P.mask + which * P.mask_stride) : nullptr;     // the row's bits, or none
    stream = !P.in_place || mask || nothing;
  }
  __device__ __forceinline__ bool keeps(int v) const { return !nothing && (!mask || ((mask[v >> 3] >> (v & 7)) & 1u)); }
};

template <bool F32, bool kBias, bool kMask>
static __global__ void __launch_bounds__(kLogitsThreads<kBias>, kLogitsPerSM) logits_kernel(LogitsDev P) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ float s_knob[3];                                               // rho, pi, phi
  const TokenTable table(smem_raw, P.table_log2, P.slice);
  uint32_t* named = table.end();                                            // [slice / 32 + 1] a bit for every token of the history
  constexpr int kSize = F32 ? 4 : 2, kAhead = F32 ? 2 : 4, kThreads = kLogitsThreads<kBias>;
  const int tid = threadIdx.x;
  after_predecessor();
  auto penalised = [&](float z, uint32_t n) {
    if (n & (kSeen | kOutMask)) z = (z > 0.0f) ? __fdiv_rn(z, s_knob[0]) : __fmul_rn(z, s_knob[0]);
    if (n & kOutMask) z = __fsub_rn(__fsub_rn(z, s_knob[1]), __fmul_rn(s_knob[2], static_cast<float>(n & kOutMask)));
    return z;
  };
  // ---- the lists
  bool history;
  {
    const Slice<F32, kMask> S(P);
    const int n_hist = P.history && !S.nothing ? min(P.lengths ? max(P.lengths[S.row], 0) : P.hist_len, P.hist_len) : 0, n_bias = !kBias || S.nothing ? 0 : P.bias_len;
    history = n_hist > 0;
    if (tid == 0) { s_knob[0] = P.rho ? P.rho[S.row] : P.rho_s; s_knob[1] = P.pi ? P.pi[S.row] : P.pi_s; s_knob[2] = P.phi ? P.phi[S.row] : P.phi_s; }
    if (n_hist || n_bias) {
      const uint32_t width = static_cast<uint32_t>(S.hi - S.lo);
      const int32_t *hist = P.history + S.row * P.hist_stride, *ids = P.bias_ids + S.row * P.bias_ids_stride;
      table.clear<kThreads>();
      __syncthreads();
      const int prompt = P.prompts ? P.prompts[S.row] : 0;
      for (int base = tid; base < n_hist; base += 4 * kThreads) {
        uint32_t t[4];
#pragma unroll
        for (int e = 0; e < 4; e++) t[e] = base + e * kThreads < n_hist ? static_cast<uint32_t>(hist[base + e * kThreads]) - static_cast<uint32_t>(S.lo) : kNoToken;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t v = t[e];
          if (v < width) {
            uint32_t* n = table.insert(v);
            if (base + e * kThreads >= prompt) atomicAdd(n, 1u); else atomicOr(n, kSeen);
            atomicOr(&named[v >> 5], 1u << (v & 31));
          }
        }
      }
      for (int i = tid; i < n_bias; i += kThreads) {
        const uint32_t v = static_cast<uint32_t>(ids[i]) - static_cast<uint32_t>(S.lo);
        if (v < width) atomicAdd(table.insert(v), kBiasOne);
      }
      __syncthreads();
    }
  }
  // ---- the slice: [lo, head) singly, then chunks of 8 from 16-byte boundaries, then the rest singly
  {
    const Slice<F32, kMask> S(P);
    const unsigned char* const in = S.in;
    unsigned char* const out = S.out;
    const uint8_t* const mask = S.mask;
    const int lo = S.lo, hi = S.stream ? S.hi : S.lo;
    int head = lo, chunks = 0;
    if (((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(out) + static_cast<uintptr_t>(lo) * kSize;
      head = min(lo + static_cast<int>(((16u - (at & 15u)) & 15u) / kSize), hi);
      chunks = (hi - head) / 8;
    }
    const int tail = head + 8 * chunks, singles = (head - lo) + (hi - tail);
    for (int i = tid; i < singles; i += kThreads) {
      const int v = i < head - lo ? lo + i : tail + (i - (head - lo));
      if (!S.keeps(v)) { set_logit<F32>(out, v, -INFINITY); continue; }
      if (history && ((named[(v - lo) >> 5] >> ((v - lo) & 31)) & 1u)) {
        const uint32_t n = table.counts(static_cast<uint32_t>(v - lo));
        if (!kBias || !(n & kBiasMask)) { set_logit<F32>(out, v, penalised(logit_at<F32>(in, v), n)); continue; }
      }
      if (!P.in_place) {
        if (F32) reinterpret_cast<uint32_t*>(out)[v] = reinterpret_cast<const uint32_t*>(in)[v]; else reinterpret_cast<uint16_t*>(out)[v] = reinterpret_cast<const uint16_t*>(in)[v];
      }
    }
    const int shift = head & 7, lane = tid & 31;                            // (of a chunk's bits in their byte: lo is a multiple of 32)
    uint32_t next = mask ? mask_ahead<kAhead, kThreads>(mask, head, tid, chunks, lane) : 0u;
    for (int c0 = tid; c0 - lane < chunks; c0 += kThreads * kAhead) {   // (a warp together)
      const unsigned char* from = in + static_cast<int64_t>(head + 8 * c0) * kSize;
      unsigned char* to = out + static_cast<int64_t>(head + 8 * c0) * kSize;
      Chunk<F32> x[kAhead];
      const uint32_t keep = mask ? mask_bits<kAhead>(next, head, lane) : S.nothing ? 0u : 0xFFFFFFFFu;
      uint32_t touched = 0u;                                               // 8 bits for each chunk
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        const uint32_t k = (keep >> (8 * u)) & 0xFFu;
        if (c0 + u * kThreads < chunks && k != 0u && !(P.in_place && k == 0xFFu)) x[u].load(from + u * (kThreads * 8 * kSize));
      }
      if (mask) next = mask_ahead<kAhead, kThreads>(mask, head, c0 + kThreads * kAhead, chunks, lane);
      if (history) {
        const uint8_t* p = reinterpret_cast<const uint8_t*>(named) + ((head - lo) >> 3) + c0;
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
          if (c0 + u * kThreads < chunks) {
            uint32_t k = p[u * kThreads];
            if (shift) k = ((k | static_cast<uint32_t>(p[u * kThreads + 1]) << 8) >> shift) & 0xFFu;
            touched |= k << (8 * u);
          }
        }
        touched &= keep;
      }
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        const uint32_t k = (keep >> (8 * u)) & 0xFFu;
        if (c0 + u * kThreads < chunks && !(P.in_place && k == 0xFFu)) {
          if (k != 0xFFu) x[u].apply(k);
          x[u].store(to + u * (kThreads * 8 * kSize));
        }
      }
      for (; touched; touched &= touched - 1u) {                           // (behind the stores of their chunks, by the same thread)
        const int b = __ffs(static_cast<int>(touched)) - 1, u = b >> 3, v = (c0 + u * kThreads) * 8 + (b & 7);     // from head on
        const uint32_t n = table.counts(static_cast<uint32_t>(head - lo + v));
        if (kBias && (n & kBiasMask)) continue;                                       // (set below, from the logit itself)
        set_logit<F32>(out, head + v, penalised(logit_at<F32>(in, head + v), n));     // (read again, from the line just loaded)
      }
    }
  }
  // ---- tokens of the history where nothing was streamed, and those with a bias
  const Slice<F32, kMask> S(P);
  if ((history && !S.stream) || (kBias && !S.nothing)) {
    __syncthreads();
    const uint32_t width = static_cast<uint32_t>(S.hi - S.lo);
    if (!S.stream) {
      for (int i = tid; i < table.entries(); i += kThreads) {
        const uint32_t v = table.log2 ? table.word[2 * i] : static_cast<uint32_t>(i), n = table.word[table.log2 ? 2 * i + 1 : i];
        if ((n & (kSeen | kOutMask)) && !(n & kBiasMask)) set_logit<F32>(S.out, S.lo + static_cast<int>(v), penalised(logit_at<F32>(S.in, S.lo + static_cast<int>(v)), n));
      }
    }
    const int n_bias = !kBias || S.nothing ? 0 : P.bias_len;
    const int32_t* ids = P.bias_ids + S.row * P.bias_ids_stride;
    const float* values = P.bias_values + S.row * P.bias_values_stride;
    for (int base = tid & ~31; base < n_bias; base += kThreads) {      // (a warp together)
      const int i = base + (tid & 31), id = i < n_bias ? ids[i] : -1;
      const uint32_t v = static_cast<uint32_t>(id) - static_cast<uint32_t>(S.lo);
      const bool mine = i < n_bias && v < width && S.keeps(id);
      const uint32_t n = mine ? table.counts(v) : 0u;
      const bool alone = (n & kBiasMask) == kBiasOne;
      float z = mine ? penalised(logit_at<F32>(S.in, id), n) : 0.0f;
      if (mine && alone) set_logit<F32>(S.out, id, __fadd_rn(z, values[i]));
      // tokens listed more than once: the first entry adds all values in list order, the warp looks for them; any other entry's walk ends where it meets the first, and a warp's entries of one token
      // take one walk. (Equal entries then cost their additions, one behind the other; many tokens listed twice a walk over the list each.)
      for (uint32_t others = __ballot_sync(kFull, mine && !alone); others;) {
        const int lane = __ffs(static_cast<int>(others)) - 1, what = __shfl_sync(kFull, id, lane);
        float sum = __shfl_sync(kFull, z, lane);
        int first = -1;
        for (int e0 = 0; e0 < n_bias; e0 += 32) {
          const int e = e0 + (tid & 31);
          const bool same = e < n_bias && ids[e] == what;
          uint32_t m = __ballot_sync(kFull, same);
          if (first < 0 && m) first = e0 + __ffs(static_cast<int>(m)) - 1;
          if (first >= 0 && first != base + lane) break;
          const float value = same ? values[e] : 0.0f;
          for (; m; m &= m - 1u) sum = __fadd_rn(sum, __shfl_sync(kFull, value, __ffs(static_cast<int>(m)) - 1));
        }
        if ((tid & 31) == lane && first == i) set_logit<F32>(S.out, id, sum);
        others &= ~__ballot_sync(kFull, id == what);
      }
    }
  }
}

// Without lists: copied and masked (in place: masked), a block to a slice of kMaskSlice logits, four chunks of eight to a thread.
constexpr int kMaskThreads = 256, kMaskPerSM = 6;
template <bool F32> constexpr int kMaskAhead = F32 ? 2 : 4;
template <bool F32> constexpr int kMaskSlice = kMaskThreads * 8 * kMaskAhead<F32>;

template <bool F32>
static __global__ void __launch_bounds__(kMaskThreads, kMaskPerSM) logits_mask_kernel(LogitsDev P) {
  constexpr int kSize = F32 ? 4 : 2, kAhead = kMaskAhead<F32>;
  const int tid = threadIdx.x, lane = tid & 31;
  after_predecessor();
  const Slice<F32, true> S(P);
  int head = S.lo, chunks = 0;                                              // [lo, head) singly, then chunks of 8 from 16-byte boundaries, then the rest singly
  if (((reinterpret_cast<uintptr_t>(S.in) ^ reinterpret_cast<uintptr_t>(S.out)) & 15u) == 0) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(S.out) + static_cast<uintptr_t>(S.lo) * kSize;
    head = min(S.lo + static_cast<int>(((16u - (at & 15u)) & 15u) / kSize), S.hi);
    chunks = (S.hi - head) / 8;
  }
  const uint32_t keep = S.mask ? mask_bits<kAhead>(mask_ahead<kAhead, kMaskThreads>(S.mask, head, tid, chunks, lane), head, lane) : S.nothing ? 0u : 0xFFFFFFFFu;    // 8 bits for each chunk
  const int64_t at = static_cast<int64_t>(head + 8 * tid) * kSize;
  Chunk<F32> x[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; u++) {
    const uint32_t k = (keep >> (8 * u)) & 0xFFu;
    if (tid + u * kMaskThreads < chunks && k != 0u && !(P.in_place && k == 0xFFu)) x[u].load(S.in + at + u * (kMaskThreads * 8 * kSize));
  }
#pragma unroll
  for (int u = 0; u < kAhead; u++) {
    const uint32_t k = (keep >> (8 * u)) & 0xFFu;
    if (tid + u * kMaskThreads < chunks && !(P.in_place && k == 0xFFu)) {
      if (k != 0xFFu) x[u].apply(k);
      x[u].store_once(S.out + at + u * (kMaskThreads * 8 * kSize));
    }
  }
  const int tail = head + 8 * chunks, singles = (head - S.lo) + (S.hi - tail);
  for (int i = tid; i < singles; i += kMaskThreads) {
    const int v = i < head - S.lo ? S.lo + i : tail + (i - (head - S.lo));
    if (!S.keeps(v)) set_logit<F32>(S.out, v, -INFINITY);
    else if (!P.in_place) {
      if (F32) reinterpret_cast<uint32_t*>(S.out)[v] = reinterpret_cast<const uint32_t*>(S.in)[v]; else reinterpret_cast<uint16_t*>(S.out)[v] = reinterpret_cast<const uint16_t*>(S.in)[v];
    }
  }
}

}  // namespace lm
