// The logits' processing in front of the sampler: penalties for repeated tokens, biases by token, and grammar masks, rounded once to the logits' type.
//
// Per row r, with c_all the occurrences of a token in history[r, :len] and c_out those from position prompt_len on:
//   z = float(logit); c_all > 0: z = z > 0 ? z / rho : z * rho; c_out > 0: z = (z - pi) - phi * c_out; z += the token's biases, in list order; masked: -inf.
// The penalties touch as many logits as the history has tokens, the biases as many as their list; a mask usually touches most. So a row is cut into slices, a block
// each. A block streams its slice once (16 bytes a load; out of place: copy and mask; in place: only words of the mask that are not all ones or all zeros are read,
// without a mask nothing is) and then sets the few logits of its slice that a list names. Which those are, and how often, is counted in shared memory
// addressed by the token (nothing can overflow, no order matters): words are cleared only where a list names them. The first thread to claim a token sets it.
#pragma once
#include "common.cuh"

namespace lm {

constexpr int kLogitsThreads = 512;
constexpr int kLogitsMaxSlice = 12288;       // logits per slice at most: 48 KB of counts (96 with biases)
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

// Eight logits under the bits of `keep`.
template <bool F32> struct Chunk;
template <> struct Chunk<false> {
  uint4 q;
  __device__ __forceinline__ void load(const void* p) { q = __ldcs(static_cast<const uint4*>(p)); }
  __device__ __forceinline__ void store(void* p) const { *static_cast<uint4*>(p) = q; }
  static __device__ __forceinline__ uint32_t two(uint32_t w, uint32_t keep) {
    return (keep & 1u ? w & 0xFFFFu : 0xFF80u) | (keep & 2u ? w & 0xFFFF0000u : 0xFF800000u);
  }
  __device__ __forceinline__ void apply(uint32_t keep) {
    if (keep == 0xFFu) return;
    q.x = two(q.x, keep); q.y = two(q.y, keep >> 2); q.z = two(q.z, keep >> 4); q.w = two(q.w, keep >> 6);
  }
};
template <> struct Chunk<true> {
  uint4 a, b;
  __device__ __forceinline__ void load(const void* p) { a = __ldcs(static_cast<const uint4*>(p)); b = __ldcs(static_cast<const uint4*>(p) + 1); }
  __device__ __forceinline__ void store(void* p) const { static_cast<uint4*>(p)[0] = a; static_cast<uint4*>(p)[1] = b; }
  __device__ __forceinline__ void apply(uint32_t keep) {
    if (keep == 0xFFu) return;
    const uint32_t m = 0xFF800000u;
    if (!(keep & 1u)) a.x = m; if (!(keep & 2u)) a.y = m; if (!(keep & 4u)) a.z = m; if (!(keep & 8u)) a.w = m;
    if (!(keep & 16u)) b.x = m; if (!(keep & 32u)) b.y = m; if (!(keep & 64u)) b.z = m; if (!(keep & 128u)) b.w = m;
  }
};

template <bool F32>
static __global__ void __launch_bounds__(kLogitsThreads) logits_kernel(LogitsDev P) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  uint32_t* counts = reinterpret_cast<uint32_t*>(smem_raw);                // [slice]
  uint32_t* first = counts + P.slice;                                       // [slice], with biases: the token's first entry
  constexpr int kSize = F32 ? 4 : 2;
  const int tid = threadIdx.x;
  after_predecessor();
  const long long items = static_cast<long long>(P.rows) * P.slices;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const int row = static_cast<int>(item / P.slices), lo = static_cast<int>(item % P.slices) * P.slice, hi = min(lo + P.slice, P.vocab);
    const unsigned char* in = static_cast<const unsigned char*>(P.in) + row * P.in_stride * kSize;
    unsigned char* out = static_cast<unsigned char*>(P.out) + row * P.out_stride * kSize;
    const uint32_t* mask = nullptr;                                         // the row's words, or none
    bool nothing = false;                                                   // the row's mask does not exist: everything is masked
    if (P.mask) {
      const int m = P.mask_rows ? P.mask_rows[row] : row;
      if (m >= P.mask_count) nothing = true; else if (m >= 0) mask = P.mask + m * P.mask_stride;
    }
    const int n_hist = P.history ? min(P.lengths ? max(P.lengths[row], 0) : P.hist_len, P.hist_len) : 0;
    const int n_bias = P.bias_len;
    const int32_t* hist = P.history + row * P.hist_stride;
    const int32_t* ids = P.bias_ids + row * P.bias_ids_stride;
    const uint32_t width = static_cast<uint32_t>(hi - lo);
    auto keeps = [&](int v) { return !nothing && (!mask || ((mask[v >> 5] >> (v & 31)) & 1u)); };
    // ---- counts
    if (!nothing) {
      for (int i = tid; i < n_hist; i += kLogitsThreads) { const uint32_t v = static_cast<uint32_t>(hist[i]) - lo; if (v < width) { counts[v] = 0u; if (n_bias) first[v] = 0xFFFFFFFFu; } }
      for (int i = tid; i < n_bias; i += kLogitsThreads) { const uint32_t v = static_cast<uint32_t>(ids[i]) - lo; if (v < width) { counts[v] = 0u; first[v] = 0xFFFFFFFFu; } }
      __syncthreads();
      const int prompt = P.prompts ? P.prompts[row] : 0;
      for (int i = tid; i < n_hist; i += kLogitsThreads) {
        const uint32_t v = static_cast<uint32_t>(hist[i]) - lo;
        if (v < width) { atomicOr(&counts[v], kSeen); if (i >= prompt) atomicAdd(&counts[v], 1u); }
      }
      for (int i = tid; i < n_bias; i += kLogitsThreads) {
        const uint32_t v = static_cast<uint32_t>(ids[i]) - lo;
        if (v < width) { atomicAdd(&counts[v], kBiasOne); atomicMin(&first[v], static_cast<uint32_t>(i)); }
      }
    }
    // ---- the slice
    if (!P.in_place || mask || nothing) {
      const bool together = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0 && (reinterpret_cast<uintptr_t>(in) & (kSize - 1)) == 0;
      int head = lo, chunks = 0;                                            // [lo, head) singly, then chunks of 8 from 16-byte boundaries, then the rest singly
      if (together) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(out) + static_cast<uintptr_t>(lo) * kSize;
        head = min(lo + static_cast<int>(((16u - (at & 15u)) & 15u) / kSize), hi);
        chunks = (hi - head) / 8;
      }
      const int tail = head + 8 * chunks, singles = (head - lo) + (hi - tail);
      for (int i = tid; i < singles; i += kLogitsThreads) {
        const int v = i < head - lo ? lo + i : tail + (i - (head - lo));
        if (!keeps(v)) set_logit<F32>(out, v, -INFINITY);
        else if (!P.in_place) {
          if (F32) reinterpret_cast<uint32_t*>(out)[v] = reinterpret_cast<const uint32_t*>(in)[v]; else reinterpret_cast<uint16_t*>(out)[v] = reinterpret_cast<const uint16_t*>(in)[v];
        }
      }
      const int last = (P.vocab - 1) >> 5;
      auto bits8 = [&](int v) -> uint32_t {                                  // the mask's bits of v .. v + 7
        if (nothing) return 0u;
        if (!mask) return 0xFFu;
        const int w = v >> 5;
        return __funnelshift_r(__ldg(mask + w), __ldg(mask + min(w + 1, last)), v & 31) & 0xFFu;
      };
      constexpr int kAhead = F32 ? 2 : 4;
      for (int c0 = tid; c0 < chunks; c0 += kLogitsThreads * kAhead) {
        Chunk<F32> x[kAhead];
        uint32_t keep[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
          const int c = c0 + u * kLogitsThreads;
          keep[u] = c < chunks ? bits8(head + 8 * c) : 0u;
          if (c < chunks && keep[u] != 0u && !(P.in_place && keep[u] == 0xFFu)) x[u].load(in + static_cast<int64_t>(head + 8 * c) * kSize);
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
          const int c = c0 + u * kLogitsThreads;
          if (c >= chunks || (P.in_place && keep[u] == 0xFFu)) continue;
          x[u].apply(keep[u]);
          x[u].store(out + static_cast<int64_t>(head + 8 * c) * kSize);
        }
      }
    }
    __syncthreads();
    // ---- the logits that the lists name
    if (!nothing && (n_hist || n_bias)) {
      const float rho = P.rho ? P.rho[row] : P.rho_s, pi = P.pi ? P.pi[row] : P.pi_s, phi = P.phi ? P.phi[row] : P.phi_s;
      for (int i = tid; i < n_hist + n_bias; i += kLogitsThreads) {
        const uint32_t v = static_cast<uint32_t>(i < n_hist ? hist[i] : ids[i - n_hist]) - lo;
        if (v >= width) continue;
        const uint32_t n = atomicOr(&counts[v], kClaimed);
        if (n & kClaimed) continue;
        const int id = lo + static_cast<int>(v);
        if (!keeps(id)) continue;
        float z = logit_at<F32>(in, id);
        if (n & kSeen) z = (z > 0.0f) ? __fdiv_rn(z, rho) : __fmul_rn(z, rho);
        if (n & kOutMask) z = __fsub_rn(__fsub_rn(z, pi), __fmul_rn(phi, static_cast<float>(n & kOutMask)));
        if (n & kBiasMask) {
          const float* values = P.bias_values + row * P.bias_values_stride;
          int e = static_cast<int>(first[v]);
          z = __fadd_rn(z, values[e]);
          for (int left = static_cast<int>((n & kBiasMask) / kBiasOne) - 1; left > 0;)           // (a token listed more than once: its values in list order)
            if (++e < n_bias) { if (ids[e] == id) { z = __fadd_rn(z, values[e]); left--; } } else break;
        }
        set_logit<F32>(out, id, z);
      }
    }
    __syncthreads();                                                        // the tables are the next slice's
  }
}

}  // namespace lm
