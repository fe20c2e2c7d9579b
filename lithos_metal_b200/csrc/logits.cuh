// The logits' processing in front of the sampler: penalties for repeated tokens, biases by token, and grammar masks, rounded once to the logits' type.
//
// Per row r, with c_all the occurrences of a token in history[r, :len] and c_out those from position prompt_len on:
//   z = float(logit); c_all > 0: z = z > 0 ? z / rho : z * rho; c_out > 0: z = (z - pi) - phi * c_out; z += the token's biases, in list order; masked: -inf.
// The penalties touch as many logits as the history has tokens, the biases as many as their list; a mask usually touches most. So a row is cut into slices, a block
// each. Which of its slice's tokens the history holds, and how often, a block counts in shared memory addressed by the token (nothing can overflow, no order matters): a bit per token, and a word
// of counts that is cleared only where a bit is set. It streams its slice once, 16 bytes a load, several under way per thread since before the counting: copied, masked and penalised on the way
// (in place: only what changes is written, and read where a mask keeps some of eight). A token with a bias is set behind that by its (first) entry of the list. In place without a mask only the
// tokens the lists name are touched.
#pragma once
#include "common.cuh"

namespace lm {

constexpr int kLogitsThreads = 512;
constexpr int kLogitsMaxSlice = 24576;       // logits per slice at most: 96 KB of counts, two blocks to an SM
constexpr int kLogitsMinSlice = 1024;
struct LogitsDev {
  const void* in; int64_t in_stride; void* out; int64_t out_stride; int in_place;
  int rows; int vocab;
  const int32_t* history; int hist_len; int64_t hist_stride; const int32_t* lengths; const int32_t* prompts;
  const float* rho; float rho_s; const float* pi; float pi_s; const float* phi; float phi_s;
  const int32_t* bias_ids; int64_t bias_ids_stride; const float* bias_values; int64_t bias_values_stride; int bias_len;
  const uint32_t* mask; int64_t mask_stride; const int32_t* mask_rows; int mask_count;
  int slice; int slices;
};

// a token's word of counts
constexpr uint32_t kOutMask = 0x1FFFFu;      // bits 0..16: occurrences behind the prompt
constexpr uint32_t kBiasOne = 1u << 17;      // bits 17..29: its biases (8191 at most)
constexpr uint32_t kBiasMask = 0x1FFFu << 17;
constexpr uint32_t kSeen = 1u << 30;         // it occurs
constexpr uint32_t kClaimed = 1u << 31;
constexpr int kLogitsMaxHistory = 65536;
constexpr int kLogitsMaxBias = 8191;

template <bool F32> __device__ __forceinline__ float logit_at(const void* row, int64_t i) {
  return F32 ? static_cast<const float*>(row)[i] : __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(row)[i]) << 16);
}
template <bool F32> __device__ __forceinline__ void set_logit(void* row, int64_t i, float z) {
  if (F32) static_cast<float*>(row)[i] = z; else static_cast<uint16_t*>(row)[i] = __bfloat16_as_ushort(__float2bfloat16_rn(z));
}

// Eight logits; those whose bit of `keep` is clear become -inf.
__device__ __forceinline__ uint32_t two_kept(uint32_t w, uint32_t keep) {    // of two BF16: bytes of w or of two -inf
  return __byte_perm(w, 0xFF80FF80u, 0x7654u - (keep & 1u) * 0x44u - (keep & 2u) * 0x2200u);
}
template <bool F32> struct Chunk;
template <> struct Chunk<false> {
  uint4 q;
  __device__ __forceinline__ void load(const void* p) { q = __ldcs(static_cast<const uint4*>(p)); }
  __device__ __forceinline__ void store(void* p) const { *static_cast<uint4*>(p) = q; }
  __device__ __forceinline__ void apply(uint32_t keep) { q.x = two_kept(q.x, keep); q.y = two_kept(q.y, keep >> 2); q.z = two_kept(q.z, keep >> 4); q.w = two_kept(q.w, keep >> 6); }
  __device__ __forceinline__ float get(int e) const {
    const uint32_t w = e & 4 ? (e & 2 ? q.w : q.z) : (e & 2 ? q.y : q.x);
    return e & 1 ? bf16_hi(w) : bf16_lo(w);
  }
  __device__ __forceinline__ void set(int e, float z) {
    const uint32_t h = __bfloat16_as_ushort(__float2bfloat16_rn(z)), sel = e & 1 ? 0x5410u : 0x3254u;      // h in the upper or the lower half
    const int i = e >> 1;
    q.x = i == 0 ? __byte_perm(q.x, h, sel) : q.x; q.y = i == 1 ? __byte_perm(q.y, h, sel) : q.y; q.z = i == 2 ? __byte_perm(q.z, h, sel) : q.z; q.w = i == 3 ? __byte_perm(q.w, h, sel) : q.w;
  }
};
template <> struct Chunk<true> {
  uint32_t v[8];
  __device__ __forceinline__ void load(const void* p) {
    const uint4 a = __ldcs(static_cast<const uint4*>(p)), b = __ldcs(static_cast<const uint4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  __device__ __forceinline__ void store(void* p) const { static_cast<uint4*>(p)[0] = make_uint4(v[0], v[1], v[2], v[3]); static_cast<uint4*>(p)[1] = make_uint4(v[4], v[5], v[6], v[7]); }
  __device__ __forceinline__ void apply(uint32_t keep) {
#pragma unroll
    for (int e = 0; e < 8; e++) if (!((keep >> e) & 1u)) v[e] = 0xFF800000u;
  }
  __device__ __forceinline__ float get(int e) const {
    uint32_t r = v[0];
#pragma unroll
    for (int i = 1; i < 8; i++) r = i == e ? v[i] : r;
    return __uint_as_float(r);
  }
  __device__ __forceinline__ void set(int e, float z) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = i == e ? __float_as_uint(z) : v[i];
  }
};

template <bool F32>
static __global__ void __launch_bounds__(kLogitsThreads, 2) logits_kernel(LogitsDev P) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  uint32_t* counts = reinterpret_cast<uint32_t*>(smem_raw);                // [slice]
  uint32_t* named = counts + P.slice;                                       // [slice / 32 + 1] a bit for every token of the history
  constexpr int kSize = F32 ? 4 : 2, kAhead = F32 ? 4 : 6;
  const int tid = threadIdx.x;
  after_predecessor();
  const long long items = static_cast<long long>(P.rows) * P.slices;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const int row = static_cast<int>(item / P.slices), lo = static_cast<int>(item % P.slices) * P.slice, hi = min(lo + P.slice, P.vocab);
    const unsigned char* in = static_cast<const unsigned char*>(P.in) + row * P.in_stride * kSize;
    unsigned char* out = static_cast<unsigned char*>(P.out) + row * P.out_stride * kSize;
    const int which = P.mask ? (P.mask_rows ? P.mask_rows[row] : row) : -1;
    const int n_hist = P.history ? min(P.lengths ? max(P.lengths[row], 0) : P.hist_len, P.hist_len) : 0;
    const int n_bias = P.bias_len, prompt = P.prompts ? P.prompts[row] : 0;
    const float rho = P.rho ? P.rho[row] : P.rho_s, pi = P.pi ? P.pi[row] : P.pi_s, phi = P.phi ? P.phi[row] : P.phi_s;
    const bool nothing = which >= P.mask_count && which >= 0;               // the row's mask does not exist: everything is masked
    const uint8_t* mask = which >= 0 && !nothing ? reinterpret_cast<const uint8_t*>(P.mask + which * P.mask_stride) : nullptr;     // the row's bits, or none
    const bool stream = !P.in_place || mask || nothing;
    const uint32_t width = static_cast<uint32_t>(hi - lo);
    auto keeps = [&](int v) { return !nothing && (!mask || ((mask[v >> 3] >> (v & 7)) & 1u)); };
    // ---- the slice: [lo, head) singly, then chunks of 8 from 16-byte boundaries, then the rest singly
    int head = lo, chunks = 0;
    if (stream && ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(out) + static_cast<uintptr_t>(lo) * kSize;
      head = min(lo + static_cast<int>(((16u - (at & 15u)) & 15u) / kSize), hi);
      chunks = (hi - head) / 8;
    }
    const int shift = head & 7;                                              // of a chunk's bits in their byte (lo is a multiple of 32)
    // chunk c: its logits at in8 + c * 8 * kSize, its bits from mask8[c] on
    const unsigned char* in8 = in + static_cast<int64_t>(head) * kSize;
    unsigned char* out8 = out + static_cast<int64_t>(head) * kSize;
    const uint8_t* mask8 = mask ? mask + (head >> 3) : nullptr;
    auto bits_of = [&](const uint8_t* p, int c) -> uint32_t { return shift == 0 ? p[c] : ((p[c] | static_cast<uint32_t>(p[c + 1]) << 8) >> shift) & 0xFFu; };
    Chunk<F32> x[kAhead];
    uint32_t keep[kAhead];
    auto load_bits = [&](int c0) {
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        keep[u] = nothing ? 0u : 0xFFu;
        if (mask8 && c0 + u * kLogitsThreads < chunks) keep[u] = bits_of(mask8, c0 + u * kLogitsThreads);
      }
    };
    auto load = [&](int c0) {
      const unsigned char* p = in8 + static_cast<int64_t>(c0) * (8 * kSize);
#pragma unroll
      for (int u = 0; u < kAhead; u++)
        if (c0 + u * kLogitsThreads < chunks && keep[u] != 0u && !(P.in_place && keep[u] == 0xFFu)) x[u].load(p + u * (kLogitsThreads * 8 * kSize));
    };
    load_bits(tid);
    load(tid);
    // ---- counts, while the first chunks are on their way
    const int32_t* hist = P.history + row * P.hist_stride;
    const int32_t* ids = P.bias_ids + row * P.bias_ids_stride;
    const bool lists = !nothing && (n_hist || n_bias);
    // f(token in the slice, behind the prompt) for the history's tokens in the slice
    auto each_token = [&](auto f) {
      const bool fours = (reinterpret_cast<uintptr_t>(hist) & 15u) == 0;
      for (int i = 4 * tid; i < n_hist; i += 4 * kLogitsThreads) {
        int t[4];
        if (fours && i + 4 <= n_hist) { const int4 q = __ldg(reinterpret_cast<const int4*>(hist + i)); t[0] = q.x; t[1] = q.y; t[2] = q.z; t[3] = q.w; }
        else {
#pragma unroll
          for (int e = 0; e < 4; e++) t[e] = i + e < n_hist ? hist[i + e] : -1;
        }
#pragma unroll
        for (int e = 0; e < 4; e++) { const uint32_t v = static_cast<uint32_t>(t[e]) - static_cast<uint32_t>(lo); if (v < width) f(v, i + e >= prompt); }     // (-1, padding: never below a width)
      }
    };
    auto penalised = [&](float z, uint32_t n) {
      if (n & (kSeen | kOutMask)) z = (z > 0.0f) ? __fdiv_rn(z, rho) : __fmul_rn(z, rho);
      if (n & kOutMask) z = __fsub_rn(__fsub_rn(z, pi), __fmul_rn(phi, static_cast<float>(n & kOutMask)));
      return z;
    };
    if (lists) {
      for (int i = tid; i < P.slice / 32 + 1; i += kLogitsThreads) named[i] = 0u;
      if (n_hist) each_token([&](uint32_t v, bool) { counts[v] = 0u; });
      for (int i = tid; i < n_bias; i += kLogitsThreads) { const uint32_t v = static_cast<uint32_t>(ids[i]) - static_cast<uint32_t>(lo); if (v < width) counts[v] = 0u; }
      __syncthreads();
      if (n_hist) each_token([&](uint32_t v, bool behind) {
        if (behind) atomicAdd(&counts[v], 1u); else atomicOr(&counts[v], kSeen);
        atomicOr(&named[v >> 5], 1u << (v & 31));
      });
      for (int i = tid; i < n_bias; i += kLogitsThreads) { const uint32_t v = static_cast<uint32_t>(ids[i]) - static_cast<uint32_t>(lo); if (v < width) atomicAdd(&counts[v], kBiasOne); }
      __syncthreads();
    }
    const bool penalise_here = lists && n_hist;
    if (stream) {
      const int tail = head + 8 * chunks, singles = (head - lo) + (hi - tail);
      for (int i = tid; i < singles; i += kLogitsThreads) {
        const int v = i < head - lo ? lo + i : tail + (i - (head - lo));
        if (!keeps(v)) set_logit<F32>(out, v, -INFINITY);
        else if (penalise_here && ((named[(v - lo) >> 5] >> ((v - lo) & 31)) & 1u) && !(counts[v - lo] & kBiasMask)) set_logit<F32>(out, v, penalised(logit_at<F32>(in, v), counts[v - lo]));
        else if (!P.in_place) {
          if (F32) reinterpret_cast<uint32_t*>(out)[v] = reinterpret_cast<const uint32_t*>(in)[v]; else reinterpret_cast<uint16_t*>(out)[v] = reinterpret_cast<const uint16_t*>(in)[v];
        }
      }
      const uint8_t* named8 = reinterpret_cast<const uint8_t*>(named) + ((head - lo) >> 3);
      const uint32_t* counts8 = counts + (head - lo);
      for (int c0 = tid; c0 < chunks;) {
        unsigned char* p = out8 + static_cast<int64_t>(c0) * (8 * kSize);
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
          const int c = c0 + u * kLogitsThreads;
          if (c >= chunks) break;
          uint32_t touched = penalise_here ? bits_of(named8, c) & keep[u] : 0u;
          if (P.in_place && keep[u] == 0xFFu) {                             // (not loaded: what is named is set singly)
            for (; touched; touched &= touched - 1u) {
              const int v = 8 * c + __ffs(static_cast<int>(touched)) - 1;
              if (!(counts8[v] & kBiasMask)) set_logit<F32>(out8, v, penalised(logit_at<F32>(in8, v), counts8[v]));
            }
            continue;
          }
          for (; touched; touched &= touched - 1u) {
            const int e = __ffs(static_cast<int>(touched)) - 1;
            const uint32_t n = counts8[8 * c + e];
            if (!(n & kBiasMask)) x[u].set(e, penalised(x[u].get(e), n));    // (with a bias: set below, from the logit itself)
          }
          if (keep[u] != 0xFFu) x[u].apply(keep[u]);
          x[u].store(p + u * (kLogitsThreads * 8 * kSize));
        }
        c0 += kLogitsThreads * kAhead;
        if (c0 < chunks) { load_bits(c0); load(c0); }
      }
    }
    // ---- tokens of the history where nothing was streamed, and those with a bias
    if (lists && (!stream || n_bias)) {
      __syncthreads();
      if (!stream && n_hist) each_token([&](uint32_t v, bool) {
        const uint32_t n = atomicOr(&counts[v], kClaimed);                  // (the first thread to claim a token sets it)
        const int id = lo + static_cast<int>(v);
        if (!(n & (kClaimed | kBiasMask))) set_logit<F32>(out, id, penalised(logit_at<F32>(in, id), n));
      });
      const float* values = P.bias_values + row * P.bias_values_stride;
      for (int i = tid; i < n_bias; i += kLogitsThreads) {
        const int id = ids[i];
        const uint32_t v = static_cast<uint32_t>(id) - static_cast<uint32_t>(lo);
        if (v >= width || !keeps(id)) continue;
        const uint32_t n = counts[v];
        int others = static_cast<int>((n & kBiasMask) / kBiasOne) - 1;       // (a token listed more than once: the first entry adds all values in list order)
        bool first = true;
        for (int e = 0; others > 0 && first && e < i; e++) first = ids[e] != id;
        if (!first) continue;
        float z = __fadd_rn(penalised(logit_at<F32>(in, id), n), values[i]);
        for (int e = i + 1; others > 0 && e < n_bias; e++) if (ids[e] == id) { z = __fadd_rn(z, values[e]); others--; }
        set_logit<F32>(out, id, z);
      }
    }
    if (lists) __syncthreads();                                             // the tables are the next slice's
  }
}

}  // namespace lm
