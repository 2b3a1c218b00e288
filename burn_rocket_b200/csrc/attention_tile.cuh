// attention_tile.cuh — the tensor-core kernel of ragged-batch attention: packed
// whole prompts, and chunks of new tokens over a paged cache.
//
// Work unit: one KV head of one sequence and two consecutive query "slots".
// A slot is 128 UMMA rows: floor(128 / group) tokens times the query heads that
// share the KV head, so a key tile is loaded once for every head that reads it
// and a short run of tokens still fills rows. Warp 0 finds units and feeds TMA (Q
// per unit, K and V rings of 128-key tiles; from a paged cache one box a page),
// warp 1 issues UMMAs, warps 4-7 and 8-11 are the softmax of slot 0 and 1, one row
// a thread. Per slot TMEM holds S (128 x 128 f32, P written over it as 16-bit
// values: pack2 says why) and O (f32); the two slots alternate on the tensor pipe,
// S(j+1) following P·V(j).
//
// Masks are one interval of keys per row: tiles outside a slot's are skipped,
// tiles inside every row's take no predicate. What is masked must not reach a
// row even when it is NaN: scores are selected, not multiplied; value rows past
// a sequence's last key (the next sequence, a page's unused slots) are zeroed in
// shared memory before P·V reads them; a value masked for some rows of the tile
// only (0 * NaN in the product) leaves a non-finite result, and such a row is
// computed again from the definition (row_attention).
//
// Schedules:
//   * persistent: a CTA an SM walks units ranked by cost, heaviest first and back
//     and forth over the CTAs, the next unit's Q and first tiles loading while
//     this one finishes;
//   * split: where there are fewer units than SMs, a cluster of CTAs takes equal
//     runs of one unit's key tiles and merges (O, m, l) through distributed
//     shared memory: no workspace in global memory.
//
// Bound: a slot's chain per 128 keys, about 3400 clocks (TMEM load 180, maximum
// 200, exponentials and P stores 1430 of which the MUFU needs 1024, store wait
// 170, P·V and the next S 1400), beside 2048 of UMMA for both slots: tensor pipe
// 48% active. 8 x 2048 tokens causal, 32/4 heads x 128: 287 us, 957 TFLOP/s; 64 x
// 512 causal, 16/8 heads: 132 us (the dense kernel 205); 16 x 2394 bidirectional,
// 16 heads x 72: 652 us (dense 822); a unit of one or two key tiles pays as much
// again to start and end. A softcap adds a tanhf and two divisions a score to the
// chain, which then bounds everything: 8 x 2048 causal, 16/8 heads x 128: 1406 us
// against 149 without.
#pragma once

#include <algorithm>
#include <atomic>

#include "ragged.cuh"

namespace rb {

namespace tile {

constexpr int BM = 128;  // rows of a slot
constexpr int BN = 128;  // keys of a tile
// Three warpgroups: warps 0-3 (TMA, UMMA, two idle), 4-7 and 8-11 (softmax of
// slot 0 and 1). The block starts with kLaunchRegs a thread; the first warpgroup
// hands registers to the other two, whose 128 scores a row do not fit 168 (with
// 150 to 250 bytes of spills 64 x 512 causal took 204 us, without 148; 88 / 208
// already spills in the first warpgroup). The hand-over itself waits without a
// limit, so three things are held: the shares come from the launch's registers
// (asserted below), the kernel was compiled for just that many a thread (checked
// by the host before the first launch; the assertion alone says nothing of it), and
// all four warps of the first warpgroup execute the `dec`, the idle ones too.
constexpr int kThreads = 12 * 32;
constexpr int kSoftWarp0 = 4;
constexpr int kSoftThreads = 8 * 32;
constexpr int kLaunchRegs = 168, kRoleRegs = 104, kSoftRegs = 200;
static_assert(kRoleRegs + 2 * kSoftRegs <= 3 * kLaunchRegs, "the shares come from the launch's registers");

struct TileParams {
  AttnRagged a;
  int group;   // query heads a KV head
  int tq;      // tokens a slot: floor(BM / group)
};

// As the dense kernel stages heads: D/64 128-byte-swizzled atoms and, for the
// 72-wide heads (D = 80), a 32-byte-swizzled tail of 16 columns.
template <int D>
struct Smem {
  static constexpr int ATOMS = D / 64;
  static constexpr int TAIL = D % 64;
  static_assert(TAIL == 0 || TAIL == 16, "head width");
  static constexpr int Q_ATOM = BM * 128;
  static constexpr int KV_ATOM = BN * 128;
  static constexpr int Q_TAIL_OFF = ATOMS * Q_ATOM;
  static constexpr int KV_TAIL_OFF = ATOMS * KV_ATOM;
  static constexpr int Q_TILE = ATOMS * Q_ATOM + BM * TAIL * 2;
  static constexpr int KV_TILE = ATOMS * KV_ATOM + BN * TAIL * 2;
  static_assert(Q_TILE % 1024 == 0 && KV_TILE % 1024 == 0, "1024-byte tiles");
  static constexpr int FREE = 232448 - 1024 - 1024 - 2 * Q_TILE;
  static constexpr int NKV = FREE / KV_TILE;
  static constexpr int VS = NKV / 2 > 4 ? 4 : NKV / 2;
  static constexpr int KS = NKV - VS > 4 ? 4 : NKV - VS;
  static constexpr int K_OFF = 2 * Q_TILE;
  static constexpr int V_OFF = K_OFF + KS * KV_TILE;
  static constexpr int BAR_OFF = V_OFF + VS * KV_TILE;
  static constexpr int BYTES = BAR_OFF + 1024 + 1024;
  static_assert(BYTES <= 232448, "shared memory");
  // Split: the idle rings hold [slot][D / 4][BM] float4 of O, then m and l.
  static constexpr int PART = BM * D * 4;
  static_assert(2 * PART + 4 * BM * 4 + 16 * 2 * 2 * BM * 4 <= BAR_OFF, "partials fit");
};

struct Item {
  int b, q0, n, kv;  // sequence (b < 0: no more work)
  int i0;            // first token of slot 0, in the sequence
  int g;             // KV head
  int ja, jb;        // this CTA's key tiles
  int lo[2], hi[2];  // a slot's key tiles (empty when lo > hi)
};

// NaN if any operand is: a NaN score has to show in its row.
__device__ __forceinline__ float max2n(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3n(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// The softmax warps among themselves.
__device__ __forceinline__ void soft_sync() {
  asm volatile("barrier.cta.sync 1, %0;" ::"n"(kSoftThreads) : "memory");
}

// Among each four lanes: lane i's chunk e and lane e's chunk i change places.
__device__ __forceinline__ void transpose4(uint4 (&w)[4], int lane) {
  auto swap = [](uint4& a, uint4& b, bool upper, int mask) {  // the lower lane's b with the upper lane's a
    uint4 s = upper ? a : b;
    s.x = __shfl_xor_sync(0xffffffffu, s.x, mask);
    s.y = __shfl_xor_sync(0xffffffffu, s.y, mask);
    s.z = __shfl_xor_sync(0xffffffffu, s.z, mask);
    s.w = __shfl_xor_sync(0xffffffffu, s.w, mask);
    if (upper) a = s;
    else b = s;
  };
  swap(w[0], w[1], lane & 1, 1);
  swap(w[2], w[3], lane & 1, 1);
  swap(w[0], w[2], lane & 2, 2);
  swap(w[1], w[3], lane & 2, 2);
}

// Where a unit lies (one warp). A sequence has L = ceil(n / span) spans of
// span = 2 tq tokens; span t of sequence b costs F + t + 1 (in spans of keys,
// F = floor(first position / span)) when causal and L otherwise. Up to 128
// sequences are held in registers, four a lane, and units are ranked by cost,
// highest first: the units of cost >= T are counted in closed form, and the T
// of rank r is found by bisection. Larger batches take their units in order.
struct Finder {
  int L[4], F[4], q0[4], n[4], kv[4];
  int total, top;   // ranked: units, and the highest cost
  int seq, before;  // in order: a sequence and the units before it
  bool causal, ranked;

  __device__ __forceinline__ Seq fetch(const TileParams& p, int b) const {
    return b < p.a.seqs.batch ? load_seq(p.a.seqs, b) : Seq{0, 0, 0};
  }
  __device__ __forceinline__ void init(const TileParams& p) {
    const int lane = threadIdx.x & 31, span = 2 * p.tq;
    causal = p.a.dhi == 0;
    ranked = p.a.seqs.batch <= 128;
    seq = before = total = top = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const Seq s = ranked ? fetch(p, 32 * g + lane) : Seq{0, 0, 0};
      q0[g] = s.q0;
      n[g] = s.n;
      kv[g] = s.kv;
      L[g] = (s.n + span - 1) / span;
      F[g] = causal ? max(0, s.kv - s.n) / span : 0;
      total += L[g];
      top = max(top, L[g] ? L[g] + F[g] : 0);
    }
    total = __reduce_add_sync(0xffffffffu, total);
    top = __reduce_max_sync(0xffffffffu, top);
  }
  __device__ __forceinline__ int at_least(int g, int T) const {  // units of cost >= T of the lane's sequence g
    return causal ? max(0, L[g] - max(0, T - 1 - F[g])) : (L[g] >= T ? L[g] : 0);
  }
  __device__ __forceinline__ int count(int T) const {
    return __reduce_add_sync(0xffffffffu, at_least(0, T) + at_least(1, T) + at_least(2, T) + at_least(3, T));
  }
  __device__ __forceinline__ bool find(const TileParams& p, int r, int& b, int& t, Seq& s) {
    const int lane = threadIdx.x & 31, span = 2 * p.tq;
    if (!ranked) {
      if (r < before) seq = before = 0;
      while (seq < p.a.seqs.batch) {
        const Seq x = fetch(p, seq + lane);
        const int own = (x.n + span - 1) / span;
        int sum = own;  // inclusive prefix
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += y;
        }
        const int all = __shfl_sync(0xffffffffu, sum, 31);
        if (r < before + all) {
          const int at = __ffs(__ballot_sync(0xffffffffu, r < before + sum)) - 1;
          b = seq + at;
          t = r - before - __shfl_sync(0xffffffffu, sum - own, at);
          s = Seq{__shfl_sync(0xffffffffu, x.q0, at), __shfl_sync(0xffffffffu, x.n, at),
                  __shfl_sync(0xffffffffu, x.kv, at)};
          return true;
        }
        before += all;
        seq += 32;
      }
      return false;
    }
    if (r >= total) return false;
    int lo = 1, hi = top + 1, above = 0;  // count(lo) > r >= count(hi) = above
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2, c = count(mid);
      if (c > r) lo = mid;
      else hi = mid, above = c;
    }
    int idx = r - above;  // among the units of cost lo
    if (!causal) {
      t = idx % lo;
      idx /= lo;
    }
    bool found = false;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const unsigned m = __ballot_sync(0xffffffffu, at_least(g, lo) > at_least(g, lo + 1));
      const int c = __popc(m), at = !found && idx < c ? __fns(m, 0, idx + 1) : 0;
      const int f = __shfl_sync(0xffffffffu, F[g], at), a = __shfl_sync(0xffffffffu, q0[g], at);
      const int d = __shfl_sync(0xffffffffu, n[g], at), e = __shfl_sync(0xffffffffu, kv[g], at);
      if (!found && idx < c) {
        found = true;
        b = 32 * g + at;
        if (causal) t = lo - 1 - f;
        s = Seq{a, d, e};
      }
      idx -= c;
    }
    return found;
  }
};

// One warp: the item of unit u, this CTA being `rank` of `ranks`.
__device__ __forceinline__ Item make_item(const TileParams& p, Finder& f, int u, int rank, int ranks) {
  Item it;
  Seq s;
  int level;
  it.b = -1;
  if (u < 0 || !f.find(p, u / p.a.n_kv_heads, it.b, level, s)) {
    it.b = -1;
    return it;
  }
  it.q0 = s.q0;
  it.n = s.n;
  it.kv = s.kv;
  it.g = u % p.a.n_kv_heads;
  it.i0 = level * 2 * p.tq;
  int j0 = 1 << 30, j1 = -1;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int ia = it.i0 + k * p.tq, ib = min(it.n, ia + p.tq) - 1;
    it.lo[k] = 1;
    it.hi[k] = 0;
    if (ia > ib) continue;
    int lo, hi, x;
    visible(s.kv - s.n + ia, s.kv, p.a.dlo, p.a.dhi, lo, x);
    visible(s.kv - s.n + ib, s.kv, p.a.dlo, p.a.dhi, x, hi);
    if (lo > hi) continue;
    it.lo[k] = lo / BN;
    it.hi[k] = hi / BN;
    j0 = min(j0, it.lo[k]);
    j1 = max(j1, it.hi[k]);
  }
  const long long len = max(0, j1 - j0 + 1);
  it.ja = len ? j0 + static_cast<int>(len * rank / ranks) : 0;
  it.jb = len ? j0 + static_cast<int>(len * (rank + 1) / ranks) - 1 : -1;
  return it;
}

template <int D, bool BF16, bool SOFTCAP, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
            const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmQt,
            const __grid_constant__ CUtensorMap tmKt, const __grid_constant__ CUtensorMap tmVt,
            const __grid_constant__ TileParams p) {
  using L = Smem<D>;
  constexpr int KS = L::KS, VS = L::VS;
  constexpr int DH = D == 80 ? 72 : D;  // real head width
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* q_full = bars;
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_empty + 1;      // [KS]
  uint64_t* k_empty = k_full + KS;     // [KS]
  uint64_t* v_full = k_empty + KS;     // [VS]
  uint64_t* v_empty = v_full + VS;     // [VS]
  uint64_t* s_full = v_empty + VS;     // [slot] S of the slot's next tile is in TMEM
  uint64_t* p_full = s_full + 2;       // [slot] P is in TMEM
  uint64_t* o_done = p_full + 2;       // [slot] a P·V retired
  uint64_t* o_free = o_done + 2;       // [slot] the unit's O was read out
  uint64_t* i_full = o_free + 2;       // [2] an item is there
  uint64_t* i_empty = i_full + 2;      // [2] every role has read it
  uint64_t* p_half = i_empty + 2;      // [slot] the first half of P is in TMEM
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(p_half + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* redo = tmem_slot + 2;      // [8] rows to compute again (one a bit when split, else a flag)
  Item* items = reinterpret_cast<Item*>(redo + 8);  // [2]
  static_assert((2 + 2 * KS + 2 * VS + 14) * 8 + 48 + 2 * sizeof(Item) <= 1024, "barrier area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t* err = p.a.seqs.err;
  const int ranks = SPLIT ? cluster_size() : 1, rank = SPLIT ? cluster_ctarank() : 0;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < KS; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < VS; ++i) mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&p_half[i], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&o_free[i], 4);
      mbar_init(&i_full[i], 1);
      mbar_init(&i_empty[i], 9);
    }
    *abort_flag = 0;
    for (int i = 0; i < 8; ++i) redo[i] = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // The k-th unit of this CTA: back and forth over the CTAs, so that each gets
  // early (heavy) and late (light) units alike; one a cluster when split.
  auto unit_of = [&](int k) -> int {
    if (SPLIT) return k == 0 ? static_cast<int>(blockIdx.x) / ranks : -1;
    return k * gridDim.x + ((k & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
  };
  Finder finder;
  Item first_item;
  if (warp == 0) {  // the first unit is found while the block sets up
    finder.init(p);
    first_item = make_item(p, finder, unit_of(0), rank, ranks);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // Reads item k (lane 0 of a warp or a single thread waits; `arrive` once a role).
  auto get_item = [&](int k, Item& it) -> bool {
    if (!mbar_wait(&i_full[k & 1], (k >> 1) & 1, err, abort_flag)) return false;
    it = items[k & 1];
    return true;
  };

  if (warp < kSoftWarp0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRoleRegs));
  }
  if (warp == 0) {
    // ------------------------------------------------------------ units and TMA
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    const KeyValues& kv = p.a.kv;
    const int qrows = p.tq * p.group;
    const int page = kv.table ? 1 << kv.page_shift : 0;
    const int per_tile = kv.table ? BN >> kv.page_shift : 0;  // pages a tile
    int kv_base = 0, loaded = 0;
    for (int k = 0;; ++k) {
      const Item it = k == 0 ? first_item : make_item(p, finder, unit_of(k), rank, ranks);
      if (k >= 2 && !warp_wait(&i_empty[k & 1], ((k >> 1) - 1) & 1, err, abort_flag)) break;
      if (lane == 0) {
        items[k & 1] = it;
        mbar_arrive(&i_full[k & 1]);
      }
      __syncwarp();
      if (it.b < 0) break;
      if (it.ja > it.jb) continue;  // no keys: zeros
      if (loaded > 0 && !warp_wait(q_empty, (loaded - 1) & 1, err, abort_flag)) break;
      ++loaded;
      if (lane == 0) {
        const int slots = it.i0 + p.tq < it.n ? 2 : 1;
        mbar_arrive_expect_tx(q_full, slots * qrows * (L::ATOMS * 128 + L::TAIL * 2));
        for (int s = 0; s < slots; ++s) {
          uint8_t* dst = smem + s * L::Q_TILE;
          const int row = it.q0 + it.i0 + s * p.tq;
          for (int a = 0; a < L::ATOMS; ++a)
            tma_load_3d(dst + a * L::Q_ATOM, &tmQ, q_full, a * 64, it.g * p.group, row);
          if (L::TAIL) tma_load_3d(dst + L::Q_TAIL_OFF, &tmQt, q_full, L::ATOMS * 64, it.g * p.group, row);
        }
      }
      // Page ids of the next 32 pages, one a lane, and of the 32 after.
      const int page0 = kv.table ? it.ja * per_tile : 0;
      const int pages = kv.table ? (it.kv + page - 1) >> kv.page_shift : 0;
      const int32_t* table = kv.table + it.b * kv.ld_table;
      int first_key, none;  // that any row of the unit sees
      visible(it.kv - it.n + it.i0, it.kv, p.a.dlo, p.a.dhi, first_key, none);
      auto fetch = [&](int at) {
        const int idx = page0 + at + lane;
        if (!kv.table || idx >= pages || idx >= (it.jb + 1) * per_tile) return 0;
        if (idx < first_key >> kv.page_shift) return kv.num_pages;  // behind the window: it may be gone
        const int id = __ldg(table + idx);
        if (static_cast<unsigned>(id) < static_cast<unsigned>(kv.num_pages)) return id;
        atomicOr(err, kErrBadShape);
        return kv.num_pages;  // past the map: reads as zeros
      };
      int ids[2] = {fetch(0), fetch(32)}, ids_at = 0;  // ids_at: page offset of ids[0]
      // K runs one tile ahead of V, so both page batches are held until V has
      // passed: a tile's pages lie in one batch (per_tile divides 32).
      auto page_id = [&](int off) {  // off: page offset from page0, warp-uniform base + lane
        const int at = off - ids_at;
        const int x = __shfl_sync(0xffffffffu, ids[0], at & 31), y = __shfl_sync(0xffffffffu, ids[1], at & 31);
        return at < 32 ? x : y;
      };
      auto load = [&](bool is_k, int j) -> bool {
        const int pos = kv_base + j - it.ja, nst = is_k ? KS : VS, st = pos % nst;
        uint64_t* full = is_k ? &k_full[st] : &v_full[st];
        if (!warp_wait(is_k ? &k_empty[st] : &v_empty[st], ((pos / nst) & 1) ^ 1, err, abort_flag)) return false;
        uint8_t* dst = smem + (is_k ? L::K_OFF : L::V_OFF) + st * L::KV_TILE;
        const CUtensorMap* map = is_k ? &tmK : &tmV;
        if (!kv.table) {
          if (lane == 0) {
            mbar_arrive_expect_tx(full, L::KV_TILE);
            for (int a = 0; a < L::ATOMS; ++a)
              tma_load_3d(dst + a * L::KV_ATOM, map, full, a * 64, it.g, it.q0 + j * BN);
            if (L::TAIL)
              tma_load_3d(dst + L::KV_TAIL_OFF, is_k ? &tmKt : &tmVt, full, L::ATOMS * 64, it.g, it.q0 + j * BN);
          }
        } else {
          const int n = min(per_tile, pages - j * per_tile);  // pages that hold keys
          if (lane == 0) mbar_arrive_expect_tx(full, n * page * 128 * L::ATOMS);
          const int id = page_id((j - it.ja) * per_tile + min(lane, per_tile - 1));
          __syncwarp();
          if (lane < n)
            for (int a = 0; a < L::ATOMS; ++a)
              tma_load_4d(dst + a * L::KV_ATOM + lane * page * 128, map, full, a * 64, it.g, 0, id);
          __syncwarp();
        }
        return true;
      };
      bool ok = load(true, it.ja);
      for (int j = it.ja; ok && j <= it.jb; ++j) {
        if (j < it.jb) ok = load(true, j + 1);
        if (ok) ok = load(false, j);
        if (kv.table && (j + 1 - it.ja) * per_tile >= ids_at + 32) {
          ids_at += 32;
          ids[0] = ids[1];
          ids[1] = fetch(ids_at + 32);
        }
      }
      if (!ok) break;
      kv_base += it.jb - it.ja + 1;
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ UMMA issuer
    if (elect_one_sync()) {
      constexpr uint32_t idesc_s = idesc_f16(BM, BN, BF16, false, false);
      constexpr uint32_t idesc_o = idesc_f16(BM, L::ATOMS * 64, BF16, false, true);
      constexpr uint32_t idesc_ot = idesc_f16(BM, L::TAIL ? L::TAIL : 16, BF16, false, true);
      const uint32_t q_addr = smem_u32(smem);
      const uint32_t k_addr = smem_u32(smem + L::K_OFF), v_addr = smem_u32(smem + L::V_OFF);
      const uint64_t q_desc = desc_kmajor_sw128(q_addr), k_desc = desc_kmajor_sw128(k_addr);
      const uint64_t v_desc = desc_mnmajor_sw128(v_addr, L::KV_ATOM, 1024);
      const uint64_t qt_desc = desc_kmajor_sw32(q_addr), kt_desc = desc_kmajor_sw32(k_addr);
      const uint64_t vt_desc = desc_mnmajor_sw32(v_addr);
      int n_pv[2] = {0, 0}, n_out[2] = {0, 0};
      int kv_base = 0, loaded = 0;
      Item it;
      for (int k = 0;; ++k) {
        if (!get_item(k, it)) break;
        mbar_arrive(&i_empty[k & 1]);
        if (it.b < 0) break;
        if (it.ja > it.jb) continue;
        int rlo[2], rhi[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          rlo[s] = max(it.ja, it.lo[s]);
          rhi[s] = min(it.jb, it.hi[s]);
        }
        bool first_pv[2] = {true, true};
        bool ok = mbar_wait(q_full, loaded & 1, err, abort_flag);
        ++loaded;
        auto pos_of = [&](int j) { return kv_base + j - it.ja; };
        // UMMAs of one thread run in order: S(j) may overwrite the P(j-1) that
        // the P·V before it reads.
        auto issue_s = [&](int j, int s) {
          const uint32_t st = pos_of(j) % KS, d_tmem = tmem_base + s * 256;
#pragma unroll
          for (int ks = 0; ks < L::ATOMS * 4; ++ks)
            umma_f16_ss(d_tmem, desc_add(q_desc, s * L::Q_TILE + (ks >> 2) * L::Q_ATOM + (ks & 3) * 32),
                        desc_add(k_desc, st * L::KV_TILE + (ks >> 2) * L::KV_ATOM + (ks & 3) * 32), idesc_s, ks > 0);
          if (L::TAIL)
            umma_f16_ss(d_tmem, desc_add(qt_desc, s * L::Q_TILE + L::Q_TAIL_OFF),
                        desc_add(kt_desc, st * L::KV_TILE + L::KV_TAIL_OFF), idesc_s, 1u);
          umma_commit(&s_full[s]);
        };
        int k_ready = it.ja - 1;
        auto wait_k = [&](int j) -> bool {
          if (j <= k_ready) return true;
          if (!mbar_wait(&k_full[pos_of(j) % KS], (pos_of(j) / KS) & 1, err, abort_flag)) return false;
          tc_fence_after();
          k_ready = j;
          return true;
        };
        for (int j = it.ja; ok && j <= it.jb; ++j) {
          for (int s = 0; ok && s < 2; ++s)
            if (rlo[s] <= rhi[s] && rlo[s] == j && (ok = wait_k(j))) issue_s(j, s);
          if (!ok || !(ok = wait_k(j))) break;
          umma_commit(&k_empty[pos_of(j) % KS]);
          if (j == it.jb) umma_commit(q_empty);
          const uint32_t vs = pos_of(j) % VS;
          bool v_ready = false;
          for (int s = 0; ok && s < 2; ++s) {
            if (!(rlo[s] <= j && j <= rhi[s])) continue;
            if (!(ok = mbar_wait(&p_half[s], n_pv[s] & 1, err, abort_flag))) break;
            tc_fence_after();
            if (first_pv[s] && n_out[s] > 0) {  // the last unit's O must be out
              if (!(ok = mbar_wait(&o_free[s], (n_out[s] - 1) & 1, err, abort_flag))) break;
              tc_fence_after();
            }
            if (!v_ready) {
              if (!(ok = mbar_wait(&v_full[vs], (pos_of(j) / VS) & 1, err, abort_flag))) break;
              tc_fence_after();
              v_ready = true;
            }
            const uint32_t o_tmem = tmem_base + s * 256 + 128, p_tmem = tmem_base + s * 256;
            auto pv = [&](int ks) {
              const uint32_t acc = (!first_pv[s] || ks > 0) ? 1u : 0u;
              umma_f16_ts(o_tmem, p_tmem + ks * 8, desc_add(v_desc, vs * L::KV_TILE + ks * 2048), idesc_o, acc);
              if (L::TAIL)
                umma_f16_ts(o_tmem + L::ATOMS * 64, p_tmem + ks * 8,
                            desc_add(vt_desc, vs * L::KV_TILE + L::KV_TAIL_OFF + ks * 512), idesc_ot, acc);
            };
#pragma unroll
            for (int ks = 0; ks < BN / 32; ++ks) pv(ks);
            if (!(ok = mbar_wait(&p_full[s], n_pv[s] & 1, err, abort_flag))) break;
            tc_fence_after();
#pragma unroll
            for (int ks = BN / 32; ks < BN / 16; ++ks) pv(ks);
            umma_commit(&o_done[s]);
            ++n_pv[s];
            first_pv[s] = false;
            if (j + 1 <= rhi[s] && (ok = wait_k(j + 1))) issue_s(j + 1, s);
          }
          if (!ok) break;
          if (!v_ready && !(ok = mbar_wait(&v_full[vs], (pos_of(j) / VS) & 1, err, abort_flag))) break;
          umma_commit(&v_empty[vs]);
        }
        if (!ok) break;
        for (int s = 0; s < 2; ++s)
          if (rlo[s] <= rhi[s]) ++n_out[s];
        kv_base += it.jb - it.ja + 1;
      }
    }
  }
  if (warp < kSoftWarp0) {
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) drain_after_abort();
    if (SPLIT) __syncthreads();  // the partials are out of TMEM
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem_base, 512);
    }
    if (SPLIT) {
      cluster_sync_all();
      cluster_sync_all();
    }
  } else {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    float part_m = -INFINITY, part_l = 0.0f;  // split: this thread's row of the CTA's run
    bool part_o = false;
    const int s = (warp - kSoftWarp0) >> 2;
    const int row = (warp & 3) * 32 + lane;  // TMEM lane
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_col = s * 256, o_col = s * 256 + 128;
    const int tok = row / p.group, sub = row - tok * p.group;
    int it_n = 0, kv_base = 0;
    Item next;
    auto take_item = [&](int k) -> bool {
      if (!__all_sync(0xffffffffu, get_item(k, next))) return false;
      __syncwarp();
      if (lane == 0) mbar_arrive(&i_empty[k & 1]);
      return true;
    };
    bool going = take_item(0);
    for (int k = 0; going && next.b >= 0; ++k) {
      const Item it = next;
      const int slo = s ? it.lo[1] : it.lo[0], shi = s ? it.hi[1] : it.hi[0];
      const int lo = max(it.ja, slo), hi = min(it.jb, shi);
      const int ia = it.i0 + s * p.tq;                // the slot's first token
      const int i = ia + tok, first_pos = it.kv - it.n;
      const bool valid = tok < p.tq && i < it.n;
      int row_lo, row_hi, all_lo, all_hi, x0;
      visible(first_pos + i, it.kv, p.a.dlo, p.a.dhi, row_lo, row_hi);
      visible(first_pos + ia, it.kv, p.a.dlo, p.a.dhi, x0, all_hi);
      visible(first_pos + min(it.n, ia + p.tq) - 1, it.kv, p.a.dlo, p.a.dhi, all_lo, x0);
      float m_used = -INFINITY, l = 0.0f;
      bool ok = true;
      for (int j = lo; j <= hi; ++j, ++it_n) {
        if (!__all_sync(0xffffffffu, mbar_wait(&s_full[s], it_n & 1, err, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        float x[BN];
        {
          uint32_t r0[32], r1[32], r2[32], r3[32];
          tmem_ld32(lane_base + s_col, r0);
          tmem_ld32(lane_base + s_col + 32, r1);
          tmem_ld32(lane_base + s_col + 64, r2);
          tmem_ld32(lane_base + s_col + 96, r3);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            x[e] = __uint_as_float(r0[e]);
            x[32 + e] = __uint_as_float(r1[e]);
            x[64 + e] = __uint_as_float(r2[e]);
            x[96 + e] = __uint_as_float(r3[e]);
          }
        }
        if (SOFTCAP) {
#pragma unroll
          for (int e = 0; e < BN; ++e) x[e] = p.a.softcap * tanhf(__fmul_rn(x[e], p.a.scale) / p.a.softcap) / p.a.scale;
        }
        const int ka = j * BN;
        const bool inner = ka >= all_lo && ka + BN - 1 <= all_hi;
        const int vlo = max(row_lo - ka, 0), vhi = min(row_hi - ka, BN - 1);
        if (!inner) {  // one mask word per 32 columns
#pragma unroll
          for (int c0 = 0; c0 < BN; c0 += 32) {
            const int a = min(max(vlo - c0, 0), 32), z = min(max(vhi + 1 - c0, 0), 32);  // columns [a, z)
            const uint32_t up = z == 32 ? 0xffffffffu : (1u << z) - 1u, down = a == 32 ? 0xffffffffu : (1u << a) - 1u;
            const uint32_t mask = up & ~down;
#pragma unroll
            for (int e = 0; e < 32; ++e) x[c0 + e] = (mask >> e & 1u) ? x[c0 + e] : -INFINITY;
          }
        }
        float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
        for (int e = 0; e < BN; e += 8) {
          m0 = max3n(m0, x[e], x[e + 1]);
          m1 = max3n(m1, x[e + 2], x[e + 3]);
          m2 = max3n(m2, x[e + 4], x[e + 5]);
          m3 = max3n(m3, x[e + 6], x[e + 7]);
        }
        const float mraw = max2n(max2n(m0, m1), max2n(m2, m3));
        const float c = p.a.scale * kLog2e, mt = mraw * c;
        float alpha = 1.0f;
        bool need = false;
        if (j == lo) {
          m_used = mt;
        } else if (valid && !(mt <= m_used + kRescale)) {  // (a row without a query may hold anything, NaN too)
          alpha = ex2(m_used - mt);
          m_used = mt;
          need = true;
        }
        const float nm = m_used == -INFINITY ? 0.0f : -m_used;  // nothing visible yet: weights are 0
        // The first 64 keys' weights go to P·V while the others are computed,
        // unless O or V has to be touched first.
        const bool late = __any_sync(0xffffffffu, need) || it.kv - ka < BN;
        uint64_t rs[2] = {0ull, 0ull};
#pragma unroll
        for (int c0 = 0; c0 < BN; c0 += 32) {
          uint32_t pk[16];
          const uint64_t c2 = f2_pack(c, c), nm2 = f2_pack(nm, nm);
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float y0, y1;
            f2_unpack(f2_fma(f2_pack(x[c0 + e], x[c0 + e + 1]), c2, nm2), y0, y1);
            const float p0 = ex2(y0), p1 = ex2(y1);
            rs[(e / 2) & 1] = f2_add(rs[(e / 2) & 1], f2_pack(p0, p1));
            pk[e / 2] = pack2<BF16>(p0, p1);
          }
          if (c0 == 64 && !late) {  // (here, where the first half's stores are long done)
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_half[s]);
          }
          tmem_st16(lane_base + s_col + c0 / 2, pk);
        }
        float a0, a1, a2, a3;
        f2_unpack(rs[0], a0, a1);
        f2_unpack(rs[1], a2, a3);
        l = l * alpha + ((a0 + a1) + (a2 + a3));
        // S(j)'s commit retired P·V(j-1): O is idle until p_full.
        if (__any_sync(0xffffffffu, need)) {
          uint32_t r[32];
#pragma unroll
          for (int c0 = 0; c0 < D; c0 += 32) {
            tmem_ld32(lane_base + o_col + c0, r);
            tmem_wait_ld();
            uint32_t u0[16], u1[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              u0[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
              u1[e] = __float_as_uint(__uint_as_float(r[16 + e]) * alpha);
            }
            tmem_st16(lane_base + o_col + c0, u0);
            tmem_st16(lane_base + o_col + c0 + 16, u1);
          }
        }
        // Value rows past the last key: their weights are 0, and 0 * NaN is not.
        if (it.kv - ka < BN) {
          const int pos = kv_base + j - it.ja, vs = pos % VS;
          if (!__all_sync(0xffffffffu, mbar_wait(&v_full[vs], (pos / VS) & 1, err, abort_flag))) {
            ok = false;
            break;
          }
          if (row >= it.kv - ka) {
            uint8_t* v = smem + L::V_OFF + vs * L::KV_TILE;
            const uint4 z = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int a = 0; a < L::ATOMS; ++a)
#pragma unroll
              for (int e = 0; e < 8; ++e) reinterpret_cast<uint4*>(v + a * L::KV_ATOM + row * 128)[e ^ (row & 7)] = z;
            if (L::TAIL) {
              reinterpret_cast<uint4*>(v + L::KV_TAIL_OFF + row * 32)[0] = z;
              reinterpret_cast<uint4*>(v + L::KV_TAIL_OFF + row * 32)[1] = z;
            }
          }
          fence_proxy_async_smem();
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (late) mbar_arrive(&p_half[s]);
          mbar_arrive(&p_full[s]);
        }
      }
      if (!ok) break;
      kv_base += max(0, it.jb - it.ja + 1);
      const bool has = lo <= hi;
      if (!SPLIT) going = take_item(k + 1);  // while the last P·V runs
      if (has) {
        if (!__all_sync(0xffffffffu, mbar_wait(&o_done[s], (it_n - 1) & 1, err, abort_flag))) break;
        tc_fence_after();
      }
      if (SPLIT) {  // one unit a cluster: merged below
        part_m = has ? m_used : -INFINITY;
        part_l = has ? l : 0.0f;
        part_o = has;
        break;
      }
      const int head = it.g * p.group + sub;
      uint16_t* out = p.a.out + static_cast<int64_t>(it.q0 + i) * p.a.ldo + head * DH;
      if (!has) {  // no row of the slot sees a key
        if (valid)
#pragma unroll
          for (int e = 0; e < DH / 8; ++e) reinterpret_cast<uint4*>(out)[e] = make_uint4(0u, 0u, 0u, 0u);
        continue;
      }
      const bool empty = row_lo > row_hi;
      const unsigned valid_rows = __ballot_sync(0xffffffffu, valid);
      const float inv = 1.0f / l;
      uint16_t* to[4];  // the rows of this lane's four
#pragma unroll
      for (int e = 0; e < 4; ++e)
        to[e] = reinterpret_cast<uint16_t*>(
            __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(out), (lane & ~3) + e));
      const uint64_t inv2 = f2_pack(inv, inv), zero2 = f2_pack(0.0f, 0.0f);
      uint64_t check[4] = {zero2, zero2, zero2, zero2};  // stays 0 while every value is finite
      // Not unrolled: this code runs once a unit, and each of its instructions is
      // fetched anew.
#pragma unroll 1
      for (int at = 0; at < DH; at += 32) {
        uint32_t r[32];
        tmem_ld32(lane_base + o_col + at, r);
        tmem_wait_ld();
        uint4 w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t u[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint64_t y =
                f2_mul(f2_pack(__uint_as_float(r[8 * e + 2 * q]), __uint_as_float(r[8 * e + 2 * q + 1])), inv2);
            if (DH % 32 == 0 || at + 8 * e < DH) check[q] = f2_fma(y, zero2, check[q]);
            float y0, y1;
            f2_unpack(y, y0, y1);
            u[q] = empty ? 0u : pack2<BF16>(y0, y1);
          }
          w[e] = make_uint4(u[0], u[1], u[2], u[3]);
        }
        if (DH % 32 == 0 || at + 32 <= DH) {
          // Four lanes turn their four chunks about, so that one store covers
          // 64 contiguous bytes of eight rows instead of 16 of thirty-two.
          transpose4(w, lane);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (valid_rows >> ((lane & ~3) + e) & 1) *reinterpret_cast<uint4*>(to[e] + at + 8 * (lane & 3)) = w[e];
        } else if (valid) {
          *reinterpret_cast<uint4*>(out + at) = w[0];  // the last 8 columns of a 72-wide head
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_free[s]);  // the next unit's first P·V may overwrite O
      float c0, c1;
      f2_unpack(f2_add(f2_add(check[0], check[1]), f2_add(check[2], check[3])), c0, c1);
      __syncwarp();  // before the mark: other lanes stored parts of the row
      if (valid && !empty && !(c0 + c1 == 0.0f)) {  // marked by a NaN of either type
        *reinterpret_cast<uint32_t*>(out) = 0x7fff7fffu;
        redo[0] = 1;
      }
    }

    tc_fence_before();
    __syncthreads();
    if (*abort_flag) drain_after_abort();
    if (SPLIT) {  // the rings are idle: they take the partials
      tc_fence_after();
      float4* part = reinterpret_cast<float4*>(smem + s * L::PART);
      float* stat = reinterpret_cast<float*>(smem + 2 * L::PART) + s * 2 * BM;
      if (__any_sync(0xffffffffu, part_o)) {
        const uint32_t o = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + s * 256 + 128;
  #pragma unroll
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t r[32];
          tmem_ld32(o + c0, r);
          tmem_wait_ld();
  #pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c0 + 4 * e < D)
              part[(c0 / 4 + e) * BM + row] = make_float4(__uint_as_float(r[4 * e]), __uint_as_float(r[4 * e + 1]),
                                                          __uint_as_float(r[4 * e + 2]), __uint_as_float(r[4 * e + 3]));
        }
      }
      stat[row] = part_m;
      stat[BM + row] = part_l;
      tc_fence_before();
    }
    if (SPLIT) __syncthreads();
    if (!SPLIT && redo[0] && !*abort_flag) {  // (redo is read after the barrier above)
      // The marked rows of this CTA's units, again from the definition.
      Finder finder;
      finder.init(p);
      for (int k = 0;; ++k) {
        const Item it = make_item(p, finder, unit_of(k), 0, 1);
        if (it.b < 0) break;
        for (int rr = warp - kSoftWarp0; rr < 2 * p.tq * p.group; rr += kSoftThreads / 32) {
          const int i = it.i0 + rr / p.group, head = it.g * p.group + rr % p.group;
          if (i >= it.n) break;
          const uint16_t mark = p.a.out[static_cast<int64_t>(it.q0 + i) * p.a.ldo + head * DH];
          if ((mark & 0x7fffu) != 0x7fffu) continue;
          const Seq seq{it.q0, it.n, it.kv};
          if (p.a.kv.table) row_attention<DH, BF16, true>(p.a, it.b, seq, i, head);
          else row_attention<DH, BF16, false>(p.a, it.b, seq, i, head);
        }
      }
    }
    if (SPLIT) {
      cluster_sync_all();  // every partial is written
      const Item it = items[0];
      if (it.b >= 0 && !*abort_flag) {
        const float* stat = reinterpret_cast<const float*>(smem + 2 * L::PART);       // [slot][m, l][BM]
        float* all = reinterpret_cast<float*>(smem + 2 * L::PART) + 4 * BM;           // [rank][slot][m, l][rows]
        // Rank k finishes the rows [k, k + 1) * 2 BM / ranks.
        const int r0 = rank * 2 * BM / ranks, share = (rank + 1) * 2 * BM / ranks - r0;
        for (int e = threadIdx.x - kSoftWarp0 * 32; e < ranks * 2 * share; e += kSoftThreads) {
          const int w = e / (2 * share), f = e / share % 2, rr = r0 + e % share;
          all[e] = ld_cluster(mapa_shared(stat + (rr / BM) * 2 * BM + f * BM + rr % BM, w));
        }
        soft_sync();
        for (int e = threadIdx.x - kSoftWarp0 * 32; e < share * (DH / 8); e += kSoftThreads) {
          const int rr = r0 + e % share, oct = e / share;
          const int sl = rr / BM, row = rr % BM, tok = row / p.group, i = it.i0 + sl * p.tq + tok;
          if (tok >= p.tq || i >= it.n) continue;
          int row_lo, row_hi;
          visible(it.kv - it.n + i, it.kv, p.a.dlo, p.a.dhi, row_lo, row_hi);
          const float* st = all + rr - r0;
          float M = -INFINITY, sum = 0.0f;
          for (int w = 0; w < ranks; ++w) M = max2n(M, st[w * 2 * share]);
          float acc[8] = {};
          for (int w = 0; w < ranks; ++w) {
            const float lw = st[(w * 2 + 1) * share];
            if (lw == 0.0f) continue;  // no visible key in this run (a NaN sum is taken)
            const float a = ex2(st[w * 2 * share] - M);
            sum = fmaf(a, lw, sum);
            const uint32_t src = mapa_shared(smem + sl * L::PART + (2 * oct * BM + row) * 16, w);
            const float4 u = ld_cluster4(src), v = ld_cluster4(src + BM * 16);
            acc[0] = fmaf(a, u.x, acc[0]); acc[1] = fmaf(a, u.y, acc[1]);
            acc[2] = fmaf(a, u.z, acc[2]); acc[3] = fmaf(a, u.w, acc[3]);
            acc[4] = fmaf(a, v.x, acc[4]); acc[5] = fmaf(a, v.y, acc[5]);
            acc[6] = fmaf(a, v.z, acc[6]); acc[7] = fmaf(a, v.w, acc[7]);
          }
          const bool empty = row_lo > row_hi;
          const float inv = 1.0f / sum;
          float check = 0.0f;
          uint32_t w4[4];
  #pragma unroll
          for (int q = 0; q < 4; ++q) {
            check = fmaf(acc[2 * q] * inv, 0.0f, fmaf(acc[2 * q + 1] * inv, 0.0f, check));
            w4[q] = empty ? 0u : pack2<BF16>(acc[2 * q] * inv, acc[2 * q + 1] * inv);
          }
          if (!empty && !(check == 0.0f)) {
            atomicOr(&redo[rr >> 5], 1u << (rr & 31));
          } else {
            uint16_t* out = p.a.out + static_cast<int64_t>(it.q0 + i) * p.a.ldo +
                            (it.g * p.group + row - tok * p.group) * DH + oct * 8;
            *reinterpret_cast<uint4*>(out) = make_uint4(w4[0], w4[1], w4[2], w4[3]);
          }
        }
        soft_sync();
        for (int rr = r0 + warp - kSoftWarp0; rr < r0 + share; rr += kSoftThreads / 32)
          if (redo[rr >> 5] >> (rr & 31) & 1) {
            const int row = rr % BM, tok = row / p.group;
            const Seq seq{it.q0, it.n, it.kv};
            const int i = it.i0 + (rr / BM) * p.tq + tok, head = it.g * p.group + row - tok * p.group;
            if (p.a.kv.table) row_attention<DH, BF16, true>(p.a, it.b, seq, i, head);
            else row_attention<DH, BF16, false>(p.a, it.b, seq, i, head);
          }
      }
      cluster_sync_all();  // no CTA leaves while its partials are read
    }
  }
}

// How many units a call has at most, and how many key tiles the longest.
struct Work {
  int64_t units;
  int tiles;
};

template <int D, bool BF16, bool SOFTCAP, bool SPLIT>
int launch_kernel(const CUtensorMap* tm, const TileParams& p, unsigned grid, int ranks, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Smem<D>::BYTES;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ranks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = SPLIT ? 1 : 0;
  const cudaError_t e =
      cudaLaunchKernelEx(&cfg, tile_kernel<D, BF16, SOFTCAP, SPLIT>, tm[0], tm[1], tm[2], tm[3], tm[4], tm[5], p);
  return e == cudaSuccess ? RB_OK : report_error(RB_E_DEVICE, cudaGetErrorString(e));
}

// Per device and kernel pair: attributes set, the register split checked, and
// the clusters of each size that the device holds.
template <int D, bool BF16, bool SOFTCAP>
int launch_tile(const CUtensorMap* tm, const TileParams& p, const Work& w, cudaStream_t st) {
  static std::atomic<int> resident[64][9];  // [0]: known
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return report_error(RB_E_DEVICE, "ragged attention: device ordinal");
  if (!resident[dev][0].load(std::memory_order_acquire)) {
    auto whole = tile_kernel<D, BF16, SOFTCAP, false>;
    auto split = tile_kernel<D, BF16, SOFTCAP, true>;
    cudaFuncAttributes fw, fs;
    if (cudaFuncSetAttribute(whole, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::BYTES) != cudaSuccess ||
        cudaFuncSetAttribute(split, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::BYTES) != cudaSuccess ||
        cudaFuncGetAttributes(&fw, whole) != cudaSuccess || cudaFuncGetAttributes(&fs, split) != cudaSuccess)
      return report_error(RB_E_DEVICE, "ragged attention: kernel attributes");
    // A warpgroup that asks for more than the launch holds would wait forever.
    if (fw.numRegs != kLaunchRegs || fs.numRegs != kLaunchRegs)
      return report_error(RB_E_DEVICE, "ragged attention: register split");
    for (int r = 1; r <= 8; ++r) {
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(r);
      cfg.blockDim = dim3(kThreads);
      cfg.dynamicSmemBytes = Smem<D>::BYTES;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = r;
      at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, split, &cfg) != cudaSuccess) n = 0;
      resident[dev][r] = n;
    }
    cudaGetLastError();
    resident[dev][0].store(1, std::memory_order_release);
  }
  // A cluster a unit only while every unit finds one at once, and two key tiles
  // a CTA at least: a second wave costs more than the split gains (2 x 8000 keys,
  // 16 new tokens, 8 KV heads: 65 us with 16 clusters of 8, of which 14 are
  // resident).
  int ranks = 1;
  for (int r = 2; r <= 8; ++r)
    if (w.units <= resident[dev][r].load(std::memory_order_relaxed) && w.tiles >= 2 * r) ranks = r;
  if (ranks > 1)
    return launch_kernel<D, BF16, SOFTCAP, true>(tm, p, static_cast<unsigned>(w.units * ranks), ranks, st);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(w.units, p.a.num_sms));
  return launch_kernel<D, BF16, SOFTCAP, false>(tm, p, grid, 1, st);
}

template <int D>
int launch_types(const CUtensorMap* tm, const TileParams& p, const Work& w, cudaStream_t st) {
  if (p.a.softcap != 0.0f)
    return p.a.bf16 ? launch_tile<D, true, true>(tm, p, w, st) : launch_tile<D, false, true>(tm, p, w, st);
  return p.a.bf16 ? launch_tile<D, true, false>(tm, p, w, st) : launch_tile<D, false, false>(tm, p, w, st);
}

// Instantiated one head width a file, so that they compile side by side.
int launch_d64(const CUtensorMap* tm, const TileParams& p, const Work& w, cudaStream_t st);
int launch_d80(const CUtensorMap* tm, const TileParams& p, const Work& w, cudaStream_t st);
int launch_d128(const CUtensorMap* tm, const TileParams& p, const Work& w, cudaStream_t st);

}  // namespace tile

}  // namespace rb
