// attention_decode.cu — attention of a few new tokens per sequence over a paged
// key/value cache: decode steps and short runs of drafted tokens.
//
// The query rows of one KV head, tokens x group heads of at most 16 rows, share
// every key and value, so the work is one read of the sequence's cache: HBM
// bound, with the tensor cores far from busy (a 16-row tile does 16 multiply-adds
// per 16-bit element read, an SM receives ~11 elements a clock). The kernel is
// built around bytes in flight:
//   * A warp walks 16-key blocks (a block lies in one page) on its own: K and V
//     go to its ring of shared-memory stages by cp.async, 16 bytes a lane,
//     zero-filled where a key is out of every row's sight, so nothing that lies in
//     unused slots is ever read.
//   * S = Q K^T and O += P V by m16n8k16 with f32 accumulation, P rounded to the
//     16-bit type (pack2 says why); the online softmax keeps running row maxima
//     and sums in f32, the exponent base moving only when a maximum exceeds it by
//     2^8.
//   * The blocks of a (sequence, KV head) go round-robin to the warps of a
//     cluster of 1 to 16 CTAs, whose partial (O, m, l) are merged through
//     distributed shared memory: no global workspace, no second kernel, nothing
//     for two calls to share.
//   Measured: 64 sequences of 4096 keys, 16/8 heads x 128 (1.07 GB): 193 us, 5.6
//   TB/s, DRAM 68% of its peak, issue slots 32%; each wave of CTAs pays ~5 us of
//   set-up loads and merge.
//   * A row whose result is not finite is computed again from the definition
//     (row_attention): a masked value that is not finite enters the tile product
//     as 0 * NaN.
#include <algorithm>
#include <atomic>

#include "ragged.cuh"

namespace rb {

namespace decode {

constexpr int kWarps = 4;
constexpr int kRows = 16;

template <int D>
struct Geo {
  static constexpr int CH = D / 8;               // 16-byte chunks a key row
  static constexpr int TILE = kRows * D * 2;     // one 16-key K or V block
  static constexpr int STAGES = 6144 / (kRows * D);  // 3 at D = 128, 6 at D = 64
  static constexpr int RING = STAGES * 2 * TILE; // a warp's ring: 24 KB
  static constexpr int BYTES = kWarps * RING;    // 96 KB: two CTAs an SM
  // After the main loop the rings hold the partial results.
  static constexpr int PART = kRows * D * 4;     // one f32 partial O
  static_assert((kWarps + 1) * PART + 4096 <= BYTES, "partials fit the rings");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The sequence with r longer ones before it (of equal ones the lower index
// first), among at most 128: bisection on the key count, four sequences a lane.
__device__ __forceinline__ int ranked_sequence(const RaggedBatch& q, int r) {
  const int lane = threadIdx.x & 31;
  int kv[4], hi = 0;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int b = 32 * g + lane;
    kv[g] = b < q.batch ? max(0, min(__ldg(q.kv_len + b), q.max_kv)) : -1;
    hi = max(hi, kv[g]);
  }
  auto above = [&](int x) {  // sequences with more than x keys
    return __reduce_add_sync(0xffffffffu, (kv[0] > x) + (kv[1] > x) + (kv[2] > x) + (kv[3] > x));
  };
  int lo = -1;  // above(lo) > r >= above(hi)
  hi = __reduce_max_sync(0xffffffffu, hi);
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (above(mid) > r) lo = mid;
    else hi = mid;
  }
  int idx = r - above(hi), b = 0;  // among those with exactly hi keys
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const unsigned m = __ballot_sync(0xffffffffu, kv[g] == hi);
    const int c = __popc(m);
    if (idx >= 0 && idx < c) b = 32 * g + __fns(m, 0, idx + 1);
    idx -= c;
  }
  return b;
}

// Grid: (sequence * KV heads + KV head) * cluster size + rank; neighbouring
// clusters read neighbouring heads of the same slots. Where the grid is more than
// the GPU holds at a time, `longest_first` sends the long sequences ahead.
template <int D, bool BF16>
__global__ void __launch_bounds__(kWarps * 32, 2) decode_kernel(const __grid_constant__ AttnRagged p, bool longest_first) {
  using G = Geo<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t ranks = cluster_size(), rank = cluster_ctarank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int unit = blockIdx.x / ranks;
  const int head_kv = unit % p.n_kv_heads;
  int b = unit / p.n_kv_heads;
  if (longest_first) b = ranked_sequence(p.seqs, b);
  const int group = p.n_head / p.n_kv_heads;
  const Seq s = load_seq(p.seqs, b);
  const int rows = s.n * group;  // at most kRows: load_seq skips more tokens than the launch has room for
  if (rows <= 0) return;  // the whole cluster
  const int first_pos = s.kv - s.n;  // position of the sequence's first new token
  // Keys that any row sees, and those that every row sees.
  int lo, hi, lo_all, hi_all;
  visible(first_pos, s.kv, p.dlo, p.dhi, lo, hi_all);
  visible(first_pos + s.n - 1, s.kv, p.dlo, p.dhi, lo_all, hi);
  const int block0 = lo / kRows, blocks = hi < lo ? 0 : hi / kRows - block0 + 1;

  // Q fragments: rows g and g + 8, columns 16 k + 2 t (+ 8).
  const int g = lane >> 2, t = lane & 3;
  uint32_t qf[D / 16][4];
  int row_lo[2], row_hi[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = g + 8 * h, i = r / group;
    const bool there = g + 8 * h < rows;
    const uint16_t* q = p.q + (there ? static_cast<int64_t>(s.q0 + i) * p.ldq + (head_kv * group + r % group) * D : 0);
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      qf[k][h] = there ? __ldg(reinterpret_cast<const uint32_t*>(q + 16 * k + 2 * t)) : 0u;
      qf[k][2 + h] = there ? __ldg(reinterpret_cast<const uint32_t*>(q + 16 * k + 8 + 2 * t)) : 0u;
    }
    visible(first_pos + i, s.kv, p.dlo, p.dhi, row_lo[h], row_hi[h]);
    if (!there) row_lo[h] = 0, row_hi[h] = -1;
  }

  // This warp's blocks: first, first + stride, ...
  const int first = rank * kWarps + warp, stride = ranks * kWarps;
  const int mine = blocks > first ? (blocks - first + stride - 1) / stride : 0;
  const uint32_t ring = smem_u32(smem) + warp * G::RING;
  const int32_t* table = p.kv.table + b * p.kv.ld_table;
  // Page ids of the warp's next 32 blocks, one a lane, and of the 32 after.
  auto page_ids = [&](int it0) {
    const int it = it0 + lane;
    return it < mine ? __ldg(table + ((block0 + first + it * stride) * kRows >> p.kv.page_shift)) : -1;
  };
  int ids = page_ids(0), ids_next = page_ids(32);
  auto issue = [&](int it) {
    if (it < mine) {
      if (it > 0 && (it & 31) == 0) {
        ids = ids_next;
        ids_next = page_ids(it + 32);
      }
      const int page = __shfl_sync(0xffffffffu, ids, it & 31);
      bool good = static_cast<unsigned>(page) < static_cast<unsigned>(p.kv.num_pages);
      if (!good && lane == 0) atomicOr(p.seqs.err, kErrBadShape);
      const int j0 = (block0 + first + it * stride) * kRows;
      const int64_t at = good ? page * p.kv.page_stride +
                                    static_cast<int64_t>(j0 & ((1 << p.kv.page_shift) - 1)) * p.kv.ldk + head_kv * D
                              : 0;
      const uint32_t st = ring + (it % G::STAGES) * 2 * G::TILE;
#pragma unroll
      for (int i = 0; i < kRows * G::CH / 32; ++i) {
        const int row = i * (32 / G::CH) + lane / G::CH, c = lane % G::CH;
        const bool read = good && j0 + row >= lo && j0 + row <= hi;
        const int64_t src = at + (read ? row * p.kv.ldk + c * 8 : 0);
        const uint32_t dst = st + row * (D * 2) + ((c ^ (row & 7)) << 4);
        cp_async16(dst, p.kv.k + src, read);
        cp_async16(dst + G::TILE, p.kv.v + src, read);
      }
    }
    cp_async_commit();
  };

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  const float c = p.scale * kLog2e;
#pragma unroll
  for (int it = 0; it < G::STAGES - 1; ++it) issue(it);
  for (int it = 0; it < mine; ++it) {
    cp_async_wait<G::STAGES - 2>();
    __syncwarp();
    issue(it + G::STAGES - 1);  // into the stage that the previous block left
    const uint32_t st = ring + (it % G::STAGES) * 2 * G::TILE;
    float x[2][4] = {};
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      uint32_t kf[4];
      const int row = (lane & 7) + ((lane >> 4) << 3), ch = 2 * k + ((lane >> 3) & 1);
      ldsm4(kf, st + row * (D * 2) + ((ch ^ (row & 7)) << 4));
      mma16816<BF16>(x[0], qf[k], kf[0], kf[1]);
      mma16816<BF16>(x[1], qf[k], kf[2], kf[3]);
    }
    const int j0 = (block0 + first + it * stride) * kRows;
    const bool inner = j0 >= lo_all && j0 + kRows - 1 <= hi_all;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float y = x[n][e] * c;
        if (p.softcap != 0.0f) y = p.softcap * kLog2e * tanhf(x[n][e] * p.scale / p.softcap);
        const int j = j0 + 8 * n + 2 * t + (e & 1);
        x[n][e] = inner || (j >= row_lo[e >> 1] && j <= row_hi[e >> 1]) ? y : -INFINITY;
      }
    // Exponent base: the first visible maximum, moved when a new one is 2^8 above.
    float base[2];
    bool move = false;
    float alpha[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = fmaxf(fmaxf(x[0][2 * h], x[0][2 * h + 1]), fmaxf(x[1][2 * h], x[1][2 * h + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      alpha[h] = 1.0f;
      if (mx > m[h] + kRescale || (m[h] == -INFINITY && mx > m[h])) {
        alpha[h] = ex2(m[h] - mx);
        m[h] = mx;
        move = true;
      }
      base[h] = m[h] == -INFINITY ? 0.0f : m[h];  // nothing visible yet: weights are 0
    }
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] *= alpha[e >> 1];
      l[0] *= alpha[0];
      l[1] *= alpha[1];
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[n][e] = ex2(x[n][e] - base[e >> 1]);
        l[e >> 1] += x[n][e];
      }
    const uint32_t pf[4] = {pack2<BF16>(x[0][0], x[0][1]), pack2<BF16>(x[0][2], x[0][3]),
                            pack2<BF16>(x[1][0], x[1][1]), pack2<BF16>(x[1][2], x[1][3])};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      uint32_t vf[4];
      const int row = lane & 15, ch = 2 * i + (lane >> 4);
      ldsm4_t(vf, st + G::TILE + row * (D * 2) + ((ch ^ (row & 7)) << 4));
      mma16816<BF16>(o[2 * i], pf, vf[0], vf[1]);
      mma16816<BF16>(o[2 * i + 1], pf, vf[2], vf[3]);
    }
    __syncwarp();  // the block is read: its stage may be filled again
  }
  cp_async_wait<0>();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
  }

  // The warps' partials, then the CTA's, then the cluster's.
  __syncthreads();  // the rings are free
  float* parts = reinterpret_cast<float*>(smem);            // [kWarps + 1][kRows][D]
  float* stat = parts + (kWarps + 1) * kRows * D;           // m, l: [kWarps + 1][2][kRows]
  float* all = stat + (kWarps + 1) * 2 * kRows;             // m, l of every rank: [ranks][2][kRows]
  int* redo = reinterpret_cast<int*>(all + 16 * 2 * kRows); // rows to compute again
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (g + 8 * h >= rows) continue;
    float* dst = parts + (warp * kRows + g + 8 * h) * D + 2 * t;
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
      *reinterpret_cast<float2*>(dst + 8 * i) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
    if (t == 0) {
      stat[warp * 2 * kRows + g + 8 * h] = m[h];
      stat[warp * 2 * kRows + kRows + g + 8 * h] = l[h];
    }
  }
  if (threadIdx.x == 0) *redo = 0;
  __syncthreads();
  for (int e = threadIdx.x; e < rows * D; e += kWarps * 32) {
    const int r = e / D;
    float M = -INFINITY, acc = 0.0f, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, stat[w * 2 * kRows + r]);
    const float base = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float a = ex2(stat[w * 2 * kRows + r] - base);
      acc = fmaf(a, parts[w * kRows * D + e], acc);
      sum = fmaf(a, stat[w * 2 * kRows + kRows + r], sum);
    }
    parts[kWarps * kRows * D + e] = acc;
    if (e % D == 0) {
      stat[kWarps * 2 * kRows + r] = M;
      stat[kWarps * 2 * kRows + kRows + r] = sum;
    }
  }
  if (ranks > 1) cluster_sync_all();
  else __syncthreads();
  for (int e = threadIdx.x; e < static_cast<int>(ranks) * 2 * kRows; e += kWarps * 32)
    if (e % kRows < rows)
      all[e] = ld_cluster(mapa_shared(stat + kWarps * 2 * kRows + e % (2 * kRows), e / (2 * kRows)));
  __syncthreads();
  // Each rank finishes its share of the columns, in groups of four.
  const int c0 = static_cast<int>(rank * (D / 4) / ranks) * 4, c1 = static_cast<int>((rank + 1) * (D / 4) / ranks) * 4;
  const int cols = c1 - c0;
  for (int e = threadIdx.x; e < rows * cols; e += kWarps * 32) {
    const int r = e / cols, col = c0 + e % cols;
    float M = -INFINITY, acc = 0.0f, sum = 0.0f;
    for (uint32_t w = 0; w < ranks; ++w) M = fmaxf(M, all[w * 2 * kRows + r]);
    const float base = M == -INFINITY ? 0.0f : M;
    for (uint32_t w = 0; w < ranks; ++w) {
      const float a = ex2(all[w * 2 * kRows + r] - base);
      acc = fmaf(a, ld_cluster(mapa_shared(parts + (kWarps * kRows + r) * D + col, w)), acc);
      sum = fmaf(a, all[w * 2 * kRows + kRows + r], sum);
    }
    const int i = r / group, head = head_kv * group + r % group;
    int rl, rh;
    visible(first_pos + i, s.kv, p.dlo, p.dhi, rl, rh);
    const float y = rl > rh ? 0.0f : acc / sum;
    if (!(fabsf(y) <= 3.0e38f)) atomicOr(redo, 1 << r);
    else p.out[static_cast<int64_t>(s.q0 + i) * p.ldo + head * D + col] = f2h<BF16>(y);
  }
  if (ranks > 1) cluster_sync_all();  // no rank leaves while its partials are read
  else __syncthreads();
  const int again = *redo;
  for (int r = warp; r < rows; r += kWarps)
    if (again >> r & 1)
      row_attention<D, BF16, true>(p, b, s, r / group, head_kv * group + r % group, c0, c1);
}

// Cluster size for one call. Measured on this kernel (flushed L2): a CTA alone
// streams a 128-wide key (512 bytes) in 14 ns, the GPU 6.3 TB/s, and each wave of
// clusters costs 5 us more. 8 x 4096 keys x 8 heads: sizes 1, 2, 4, 8 took 63,
// 41, 37, 43 us; 64 x 4096: 184, 197, 209, 238; 3 x 33000 sizes 8, 10, 12, 16:
// 84, 80, 92, 96 (sizes above 10 leave fewer than 24 clusters resident); 64
// sequences of 33 to 8100 keys x 4 heads 1, 2, 3, 4, 8: 147, 109, 119, 125, 158.
// The constants below are fitted to these; between them the chosen sizes were
// timed, not the others: 8, 16, 32 and 48 sequences of 300 to 8000 keys x 8 heads
// take 2.2, 1.3, 1.1 and 1.1 times the bytes at the copy rate, 128 and 256 of 33
// to 4000 x 4 heads 1.1.
static int pick_ranks(const int* active, int64_t units, int batch, double keys, int d) {
  const double key_ns = 14.0 * d / 128;
  const double all_ns = 0.6 * units * keys * d * 4 / 6300.0 * active[1];  // (lengths vary: most lie below the longest)
  int best = 1;
  double least = 1e30;
  for (int r = 1; r <= 16; ++r) {
    if (active[r] <= 0 || (r > 1 && keys < r * kWarps * kRows)) continue;
    const double waves = static_cast<double>((units + active[r] - 1) / active[r]), run = keys / r * key_ns;
    const double all = all_ns / (active[r] * r);  // sizes that leave SMs empty stream less
    // A few sequences are alike: each wave lasts as long. Many even out, but
    // for the last long ones.
    const double cost = batch <= 4 ? std::max(all, waves * run) + 5000.0 * waves
                                   : std::max(all, run) + 0.35 * run + 5000.0 * waves;
    if (cost < least) least = cost, best = r;
  }
  return best;
}

template <int D, bool BF16>
static int launch(const AttnRagged& a, cudaStream_t st) {
  auto kernel = decode_kernel<D, BF16>;
  static std::atomic<int> resident[64][17];  // clusters of each size that a device holds; [0]: known
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return report_error(RB_E_DEVICE, "attention_paged: device ordinal");
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = Geo<D>::BYTES;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (!resident[dev][0].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo<D>::BYTES) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return report_error(RB_E_DEVICE, "attention_paged: kernel attributes");
    for (int r = 1; r <= 16; ++r) {
      int n = 0;
      at[0].val.clusterDim.x = r;
      cfg.gridDim = dim3(r);
      if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) n = 0;
      resident[dev][r] = n;
    }
    cudaGetLastError();
    resident[dev][0].store(1, std::memory_order_release);
  }
  int active[17];
  for (int r = 1; r <= 16; ++r) active[r] = resident[dev][r].load(std::memory_order_relaxed);
  const int64_t units = static_cast<int64_t>(a.seqs.batch) * a.n_kv_heads;
  const int keys = a.dlo <= -kRaggedNoBound ? a.hint_kv : std::min(a.hint_kv, a.seqs.max_q - a.dlo);
  const int ranks = pick_ranks(active, units, a.seqs.batch, std::max(keys, 1), D);
  if (units * ranks > 0x7fffffff) return report_error(RB_E_SHAPE, "attention_paged: batch too large");
  const bool longest_first = units > active[ranks] && a.seqs.batch > 1 && a.seqs.batch <= 128;
  cfg.gridDim = dim3(static_cast<unsigned>(units * ranks));
  cfg.stream = st;
  at[0].val.clusterDim.x = ranks;
  cfg.numAttrs = ranks > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, longest_first);
  return e == cudaSuccess ? RB_OK : report_error(RB_E_DEVICE, cudaGetErrorString(e));
}

}  // namespace decode

int launch_attention_decode(const AttnRagged& a, cudaStream_t st) {
  using namespace decode;
  if (static_cast<int64_t>(a.seqs.max_q) * (a.n_head / a.n_kv_heads) > kRows)
    return report_error(RB_E_SHAPE, "attention_paged: too many rows for the few-row kernel");
  if (a.head_dim == 128) return a.bf16 ? launch<128, true>(a, st) : launch<128, false>(a, st);
  return a.bf16 ? launch<64, true>(a, st) : launch<64, false>(a, st);
}

}  // namespace rb
