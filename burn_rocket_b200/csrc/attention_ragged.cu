// attention_ragged.cu — attention over a ragged batch: packed whole prompts,
// or new tokens over a paged key/value cache.
//
//   out_i = sum_j softmax_j(cap(scale q_i . k_j)) v_j
//
// over the keys j that the mask lets query i see (one interval per query); a
// query that sees none is zero.
#include "ragged.cuh"

namespace rb {

namespace ragged {

// One warp per (token, head).
template <int D, bool BF16, bool PAGED>
__global__ void __launch_bounds__(256) rows_kernel(const __grid_constant__ AttnRagged p) {
  const int64_t task = blockIdx.x * static_cast<int64_t>(blockDim.x >> 5) + (threadIdx.x >> 5);
  const int t = static_cast<int>(task / p.n_head), head = static_cast<int>(task % p.n_head);
  if (t >= p.seqs.tokens) return;
  const int b = find_seq(p.seqs.cu, p.seqs.batch, t);
  if (b < 0) return;
  const Seq s = load_seq(p.seqs, b);
  if (t - s.q0 < s.n) row_attention<D, BF16, PAGED>(p, b, s, t - s.q0, head);
}

template <int D>
static int launch_rows(const AttnRagged& a, cudaStream_t st) {
  const int64_t blocks = (static_cast<int64_t>(a.seqs.tokens) * a.n_head + 7) / 8;
  if (blocks > 0x7fffffff) return RB_E_SHAPE;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (a.kv.table) {
    if (a.bf16) rows_kernel<D, true, true><<<grid, 256, 0, st>>>(a);
    else rows_kernel<D, false, true><<<grid, 256, 0, st>>>(a);
  } else {
    if (a.bf16) rows_kernel<D, true, false><<<grid, 256, 0, st>>>(a);
    else rows_kernel<D, false, false><<<grid, 256, 0, st>>>(a);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? RB_OK : report_error(RB_E_DEVICE, cudaGetErrorString(e));
}

}  // namespace ragged

int launch_attention_ragged(const AttnRagged& a, cudaStream_t st) {
  if (a.kv.table && static_cast<int64_t>(a.seqs.max_q) * (a.n_head / a.n_kv_heads) <= 16)
    return launch_attention_decode(a, st);
  if (a.head_dim == 128) return ragged::launch_rows<128>(a, st);
  if (a.head_dim == 64) return ragged::launch_rows<64>(a, st);
  if (a.head_dim == 72) return ragged::launch_rows<72>(a, st);
  return RB_E_UNSUPPORTED;
}

}  // namespace rb
