// ragged.cuh — what the ragged-batch kernels share: where a sequence's tokens
// and keys lie, which keys a query sees, and the attention of one query row
// straight from the definition.
//
// A batch holds sequences of different lengths back to back: sequence b owns
// the token rows [cu[b], cu[b+1]). Its keys are its own rows (packed prompts)
// or kv_len[b] slots of a paged cache, the new tokens being the last ones.
// All lengths, offsets and page ids are device data, read only here, and each
// is checked before it addresses anything: a sequence whose numbers do not fit
// the call is skipped, a page id outside the cache reads as zeros, and both set
// the bad-shape bit of the device error word.
#pragma once

#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_bf16.h>

#include "kernels.h"
#include "sm100.cuh"

namespace rb {

struct Seq {
  int q0;  // first token row
  int n;   // new tokens (query rows); 0 when the sequence is skipped
  int kv;  // keys
};

__device__ __forceinline__ Seq load_seq(const RaggedBatch& r, int b) {
  Seq s;
  s.q0 = __ldg(r.cu + b);
  const int q1 = __ldg(r.cu + b + 1);
  s.n = q1 - s.q0;
  s.kv = r.kv_len ? __ldg(r.kv_len + b) : s.n;
  if (s.q0 < 0 || q1 < s.q0 || q1 > r.tokens || s.n > r.max_q || s.kv < 0 || s.kv > r.max_kv) {
    atomicOr(r.err, kErrBadShape);
    s.q0 = s.n = s.kv = 0;
  }
  return s;
}

// Sequence that owns token row t, or -1 for a row outside every sequence. One
// warp: each step reads 32 evenly spaced bounds at once, so 32768 sequences take
// three dependent loads. Where the bounds fall, against the contract, the result
// may be a sequence that does not hold the row: the caller compares.
__device__ __forceinline__ int find_seq(const int32_t* cu, int batch, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = batch;  // the answer is the number of b in [0, batch] with cu[b] <= t, less one
  if (t < __ldg(cu) || t >= __ldg(cu + batch)) return -1;
  while (hi - lo > 1) {    // cu[lo] <= t < cu[hi]
    const int step = (hi - lo + 31) / 32;
    const int at = lo + (lane + 1) * step;
    const bool le = at < hi && __ldg(cu + at) <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, le));
    hi = min(hi, lo + (c + 1) * step);
    lo += c * step;
  }
  return lo;
}

// Element offset of key row j's page slot, or -1 when its page id lies
// outside the cache (flagged).
__device__ __forceinline__ int64_t slot_offset(const KeyValues& kv, int b, int j, uint32_t* err) {
  const int page = __ldg(kv.table + b * kv.ld_table + (j >> kv.page_shift));
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(kv.num_pages)) {
    atomicOr(err, kErrBadShape);
    return -1;
  }
  return page * kv.page_stride + static_cast<int64_t>(j & ((1 << kv.page_shift) - 1)) * kv.ldk;
}

// The keys that position `pos` sees: [lo, hi], empty when lo > hi.
__device__ __forceinline__ void visible(int pos, int kv, int dlo, int dhi, int& lo, int& hi) {
  // |dlo|, |dhi| and pos are at most 2^30: no sum leaves 32 bits.
  lo = dlo <= -kRaggedNoBound ? 0 : max(0, pos + dlo);
  hi = dhi >= kRaggedNoBound ? kv - 1 : min(kv - 1, pos + dhi);
}

constexpr float kLog2e = 1.4426950408889634f;
// How far (in log2) a running maximum may rise above the exponent base before
// the base follows: weights stay below 2^8, within f16, and few steps rescale.
constexpr float kRescale = 8.0f;

template <bool BF16>
__device__ __forceinline__ float h2f(uint16_t x) {
  if (BF16) return __uint_as_float(static_cast<uint32_t>(x) << 16);
  return __half2float(__ushort_as_half(x));
}
template <bool BF16>
__device__ __forceinline__ uint16_t f2h(float x) {
  if (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  return __half_as_ushort(__float2half_rn(x));
}

// Two softmax weights (or outputs) as 16-bit values. A weight is rounded before
// P.V because the products take operands of V's type (TF32 would hold no more bits
// than f16, at half the rate and with V widened); its half step, 2^-11 in f16 and
// 2^-8 in bf16, enters the output as a mean over the keys. The weights' sum is
// taken before the rounding, in f32. Against 64 bits an output is off by up to 1.4
// times what a form in 32 bits with one rounding at the end is.
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// One query row by one warp, from the definition: scores, softmax statistics
// and sums in f32, one rounding at the end. Only the visible keys and values
// are read, so nothing that stands in a masked place can reach the row; a row
// that sees no key is zero. Lane l holds the columns l, l + 32, ...; the columns
// [c0, c1) are written.
template <int D, bool BF16, bool PAGED>
__device__ __noinline__ void row_attention(const AttnRagged& p, int b, const Seq& s, int i, int head, int c0 = 0,
                                           int c1 = D) {
  constexpr int NC = (D + 31) / 32;
  const int lane = threadIdx.x & 31;
  const int g = head / (p.n_head / p.n_kv_heads);
  int lo, hi;
  visible(s.kv - s.n + i, s.kv, p.dlo, p.dhi, lo, hi);
  const uint16_t* q = p.q + static_cast<int64_t>(s.q0 + i) * p.ldq + head * D;
  float qf[NC], acc[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    qf[c] = lane + 32 * c < D ? h2f<BF16>(q[lane + 32 * c]) : 0.0f;
    acc[c] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int j0 = lo; j0 <= hi; j0 += 4) {
    float x[4], v[4][NC];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = min(j0 + u, hi);
      int64_t ko, vo;
      bool there = true;
      if (PAGED) {
        ko = vo = slot_offset(p.kv, b, j, p.seqs.err);
        there = ko >= 0;
      } else {
        ko = static_cast<int64_t>(s.q0 + j) * p.kv.ldk;
        vo = static_cast<int64_t>(s.q0 + j) * p.kv.ldv;
      }
      x[u] = 0.0f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int col = lane + 32 * c;
        const bool in = there && col < D;
        x[u] = fmaf(qf[c], in ? h2f<BF16>(p.kv.k[ko + g * D + col]) : 0.0f, x[u]);
        v[u][c] = in ? h2f<BF16>(p.kv.v[vo + g * D + col]) : 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x[u] += __shfl_xor_sync(0xffffffffu, x[u], o);
      if (j0 + u > hi) break;
      float y = x[u] * p.scale;
      if (p.softcap != 0.0f) y = p.softcap * tanhf(y / p.softcap);
      // A NaN score passes through its weight; a row whose every score is
      // -inf ends as 0 / 0, as its softmax does.
      const float mn = fmaxf(m, y);
      const float a = m == mn ? 1.0f : expf(m - mn);
      const float w = y == -INFINITY ? 0.0f : expf(y - mn);
      l = l * a + w;
#pragma unroll
      for (int c = 0; c < NC; ++c) acc[c] = fmaf(w, v[u][c], acc[c] * a);
      m = mn;
    }
  }
  uint16_t* out = p.out + static_cast<int64_t>(s.q0 + i) * p.ldo + head * D;
  const float inv = lo > hi ? 0.0f : 1.0f / l;
#pragma unroll
  for (int c = 0; c < NC; ++c)
    if (lane + 32 * c >= c0 && lane + 32 * c < c1) out[lane + 32 * c] = f2h<BF16>(lo > hi ? 0.0f : acc[c] * inv);
}

}  // namespace rb
