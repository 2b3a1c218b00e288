// attention_ragged.cu — which kernel a ragged-batch attention call runs, its
// tensor maps and how its work is divided.
#include "attention_tile.cuh"

namespace rb {

static int launch_attention_tile(const AttnRagged& a, cudaStream_t st) {
  using namespace tile;
  TileParams p{};
  p.a = a;
  p.group = a.n_head / a.n_kv_heads;
  p.tq = BM / p.group;
  const int d = a.head_dim, span = 2 * p.tq;
  const uint64_t tokens = a.seqs.tokens, row = 2ull * d;
  CUtensorMap tm[6];
  auto maps = [&](int at, uint32_t cols, int swizzle) -> int {
    int rc;
    {
      const uint64_t dims[3] = {uint64_t(d), uint64_t(a.n_head), tokens}, strides[2] = {row, 2ull * a.ldq};
      const uint32_t box[3] = {cols, uint32_t(p.group), uint32_t(p.tq)};
      if ((rc = make_tmap_16bit(&tm[at], a.q, 3, dims, strides, box, swizzle)) != RB_OK) return rc;
    }
    for (int i = 0; i < 2; ++i) {
      const void* base = i ? a.kv.v : a.kv.k;
      const uint64_t ld = 2ull * (i ? a.kv.ldv : a.kv.ldk);
      if (a.kv.table) {
        const uint32_t page = 1u << a.kv.page_shift;
        const uint64_t dims[4] = {uint64_t(d), uint64_t(a.n_kv_heads), page, uint64_t(a.kv.num_pages)};
        const uint64_t strides[3] = {row, ld, 2ull * a.kv.page_stride};
        const uint32_t box[4] = {cols, 1, page, 1};
        rc = make_tmap_16bit(&tm[at + 1 + i], base, 4, dims, strides, box, swizzle);
      } else {
        const uint64_t dims[3] = {uint64_t(d), uint64_t(a.n_kv_heads), tokens}, strides[2] = {row, ld};
        const uint32_t box[3] = {cols, 1, uint32_t(BN)};
        rc = make_tmap_16bit(&tm[at + 1 + i], base, 3, dims, strides, box, swizzle);
      }
      if (rc != RB_OK) return rc;
    }
    return RB_OK;
  };
  int rc = maps(0, 64, 128);
  if (rc != RB_OK) return rc;
  if (d == 72) {
    if ((rc = maps(3, 16, 32)) != RB_OK) return rc;
  } else {
    for (int i = 0; i < 3; ++i) tm[3 + i] = tm[i];
  }
  // At most this many units: every sequence ends in one part-filled span.
  const int64_t units = (static_cast<int64_t>(a.seqs.tokens) / span + std::min(a.seqs.batch, a.seqs.tokens)) * a.n_kv_heads;
  if (units > 0x7fffffff) return report_error(RB_E_SHAPE, "ragged attention: batch too large");
  // The keys of the longest unit: a window's, or the expected length.
  const int keys = a.dlo <= -kRaggedNoBound ? a.hint_kv : std::min(a.hint_kv, span - 1 - a.dlo + std::max(a.dhi, 0));
  const Work w{units, (keys + BN - 1) / BN};
  if (d == 128) return launch_d128(tm, p, w, st);
  return d == 64 ? launch_d64(tm, p, w, st) : launch_d80(tm, p, w, st);
}

int launch_attention_ragged(const AttnRagged& a, cudaStream_t st) {
  if (a.kv.table && static_cast<int64_t>(a.seqs.max_q) * (a.n_head / a.n_kv_heads) <= 16)
    return launch_attention_decode(a, st);
  return launch_attention_tile(a, st);
}

}  // namespace rb
