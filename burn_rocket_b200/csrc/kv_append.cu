// kv_append.cu — new tokens' keys and values into a paged cache, the q/k
// RMSNorm and the position rotation applied on the way.
//
// Token i of sequence b stands at position kv_len[b] - n_b + i. Its q heads
// are normed, rotated and written to q_out, its k heads likewise into the
// cache slot of the position, its v heads copied there:
//   norm(x) = x / sqrt(mean(x^2) + eps) * w           (f32, optional)
//   rot(a, b) = (a cos - b sin, b cos + a sin)         (the two halves of a head)
// with one rounding to the 16-bit type at the end.
//
// One read of q, k, v and one write each: HBM bound, and for a few tokens the
// chain of dependent loads (sequence bounds -> its lengths -> page id and
// angles) is all there is. A warp takes 2 or 3 passes of 512 / D heads of one
// token, whichever wastes fewer lanes (more on a tie); lane groups of D/16 lanes
// hold a head, each lane eight elements of either half (16-byte accesses), and
// the whole share's loads are issued before the chain is walked. Six blocks an SM
// hide the chain: 4 passes at 108 registers took 59 us for 23238 tokens of 32/4 x
// 64 bf16 heads without a norm (238 MB), 3 at 80 registers 47 us (5.1 TB/s), 2 50;
// 16/8 x 128 f16 heads with norms 57, 60 and 56 us (263 MB, 4.7 TB/s); one decode
// token of 32 sequences 4.2, 4.3 and 3.6.
#include "ragged.cuh"

namespace rb {

namespace append {

__device__ __forceinline__ void unpack8(const uint4& u, bool bf16, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (bf16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8], bool bf16) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (bf16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

template <int D, bool BF16, int PASSES>
__global__ void __launch_bounds__(128, 6) kv_append_kernel(const KvAppend p, int shares) {
  constexpr int LH = D / 16;       // lanes a head
  constexpr int HP = 32 / LH;      // heads a pass
  const int lane = threadIdx.x & 31;
  const int64_t task = blockIdx.x * 4ll + (threadIdx.x >> 5);
  const int t = static_cast<int>(task / shares), share = static_cast<int>(task % shares);
  if (t >= p.seqs.tokens) return;
  const int units = p.n_head + 2 * p.n_kv_heads;  // q heads, k heads, v heads
  const int col = 8 * (lane % LH);
  uint4 lo[PASSES], hi[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int u = (share * PASSES + i) * HP + lane / LH;
    lo[i] = hi[i] = make_uint4(0u, 0u, 0u, 0u);
    if (u >= units) continue;
    const uint16_t* src = u < p.n_head ? p.q + t * p.ldq + u * D
                          : u < p.n_head + p.n_kv_heads ? p.k + t * p.ldk + (u - p.n_head) * D
                                                        : p.v + t * p.ldv + (u - p.n_head - p.n_kv_heads) * D;
    lo[i] = *reinterpret_cast<const uint4*>(src + col);
    hi[i] = *reinterpret_cast<const uint4*>(src + D / 2 + col);
  }
  const int b = find_seq(p.seqs.cu, p.seqs.batch, t);
  if (b < 0) return;  // a row behind the last sequence
  const Seq s = load_seq(p.seqs, b);
  // A skipped sequence, or bounds that fall: then the search can end at a
  // sequence on either side of the row.
  if (t < s.q0 || t - s.q0 >= s.n) {
    atomicOr(p.seqs.err, kErrBadShape);
    return;
  }
  if (s.kv < s.n || s.kv > p.max_pos) {  // a position outside the angle table: none of the sequence's tokens
    atomicOr(p.seqs.err, kErrBadShape);
    return;
  }
  const int pos = s.kv - s.n + t - s.q0;
  const int64_t slot = slot_offset(p.cache, b, pos, p.seqs.err);
  if (slot < 0) return;
  float c8[8], s8[8];
  load8(p.cos_t + static_cast<int64_t>(pos) * (D / 2) + col, c8);
  load8(p.sin_t + static_cast<int64_t>(pos) * (D / 2) + col, s8);
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int u = (share * PASSES + i) * HP + lane / LH;
    const bool is_q = u < p.n_head, is_k = !is_q && u < p.n_head + p.n_kv_heads;
    float a[8], c[8];
    unpack8(lo[i], BF16, a);
    unpack8(hi[i], BF16, c);
    const float* w = is_q ? p.q_norm : is_k ? p.k_norm : nullptr;
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(a[e], a[e], fmaf(c[e], c[e], ss));
#pragma unroll
    for (int o = LH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (w) {
      const float inv = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
      float wa[8], wc[8];
      load8(w + col, wa);
      load8(w + D / 2 + col, wc);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        a[e] *= inv * wa[e];
        c[e] *= inv * wc[e];
      }
    }
    if (u >= units) continue;
    uint4 oa = lo[i], oc = hi[i];
    if (is_q || is_k) {
      float ra[8], rc[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ra[e] = a[e] * c8[e] - c[e] * s8[e];
        rc[e] = c[e] * c8[e] + a[e] * s8[e];
      }
      oa = pack8(ra, BF16);
      oc = pack8(rc, BF16);
    }
    uint16_t* dst = is_q ? p.q_out + t * p.ldo + u * D
                    : is_k ? p.k_cache + slot + (u - p.n_head) * D
                           : p.v_cache + slot + (u - p.n_head - p.n_kv_heads) * D;
    *reinterpret_cast<uint4*>(dst + col) = oa;
    *reinterpret_cast<uint4*>(dst + D / 2 + col) = oc;
  }
}

template <int D, int PASSES>
static int launch(const KvAppend& a, int passes, cudaStream_t st) {
  const int shares = (passes + PASSES - 1) / PASSES;
  const int64_t blocks = (static_cast<int64_t>(a.seqs.tokens) * shares + 3) / 4;
  if (blocks > 0x7fffffff) return report_error(RB_E_SHAPE, "kv_append: too many tokens");
  if (a.bf16) kv_append_kernel<D, true, PASSES><<<static_cast<unsigned>(blocks), 128, 0, st>>>(a, shares);
  else kv_append_kernel<D, false, PASSES><<<static_cast<unsigned>(blocks), 128, 0, st>>>(a, shares);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? RB_OK : report_error(RB_E_DEVICE, cudaGetErrorString(e));
}

template <int D>
static int launch(const KvAppend& a, cudaStream_t st) {
  constexpr int HP = 512 / D;  // heads a pass
  const int passes = (a.n_head + 2 * a.n_kv_heads + HP - 1) / HP;
  return (passes + 2) / 3 * 3 <= (passes + 1) / 2 * 2 ? launch<D, 3>(a, passes, st) : launch<D, 2>(a, passes, st);
}

}  // namespace append

int launch_kv_append(const KvAppend& a, cudaStream_t st) {
  return a.head_dim == 128 ? append::launch<128>(a, st) : append::launch<64>(a, st);
}

}  // namespace rb
