// Eviction from a paged cache by accumulated attention weight.
//
// One cluster of CTAs per (sequence, key head). Every slot gets a 32-bit key whose unsigned
// order is the order of keeping: EV_MUST for the positions that must stay, else the
// weight's bits made monotone (NaN lowest). A slot below the budget whose page is absent can
// take no row: it keeps its place (EV_HELD, above all others), and in such a sequence the
// slots behind the budget that need not stay come last (0), so that a row that must stay
// never moves to where it would be lost. Which slots go:
//   - up to EV_FEW of them (a decode step drops one): the smallest key, of equals the highest
//     slot, is looked for that many times;
//   - more: the budget-th largest key is found eleven bits a pass by a histogram in shared
//     memory (at most 3 passes over keys that stay in registers, fewer once a bin's border
//     hits the budget exactly). Keys above it stay, of those equal to it the lowest slots.
//     (Counting against three thresholds a pass needs no atomics but up to 16 passes, each
//     with a barrier of the cluster: 22 us for 32768 slots on eight CTAs.)
// Either way the result does not depend on any order of execution. Then the i-th slot below
// the budget that is not kept (a hole) takes the i-th kept slot behind the budget (a mover).
// Holes and movers are disjoint ranges of slots, so all rows move at once and in place.
// Reading the weights and positions and moving the rows is the work that cannot be left out;
// a long sequence gets several CTAs (they share the counts through distributed shared
// memory), because one SM moves rows at a small part of the memory's rate.
// 4 x up to 32768 slots to 8192, 8 heads, bf16: 44.5 us, 20 of them the moves at the memory's rate,
// the others the latency of the passes and the numbering. 64 x 513 slots to 512, 12 heads: 5.6 us.
#pragma once
#include "paged_common.cuh"

namespace cb {

constexpr int EV_MAX_CTAS = 8;
constexpr int EV_MAX_THREADS = 1024;
constexpr int EV_MAX_PER_THREAD = 32;
// longest sequence: its keys stay in the registers of one cluster
constexpr int EV_MAX_LEN = EV_MAX_CTAS * EV_MAX_THREADS * EV_MAX_PER_THREAD;

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t cluster_addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
  return v;
}

__device__ __forceinline__ uint32_t evict_key(float w) {
  if (w != w) return 1u;
  const uint32_t bits = __float_as_uint(w + 0.0f);  // -0 counts as 0
  return bits >> 31 ? ~bits : bits | 0x80000000u;
}

constexpr uint32_t EV_MUST = 0xfffffffeu;  // (of a weight: at most 0xff800000, infinity)
constexpr uint32_t EV_HELD = 0xffffffffu;

constexpr int EV_FEW = 8;
constexpr int EV_BINS = 2048;

template <int THREADS, int PER>
struct EvictShared {
  static constexpr int WARPS = THREADS / 32;
  uint32_t count[3][3];    // sums of three counts over the block, three buffers in turn
  uint32_t least[2][2];    // this CTA's smallest key and its highest slot, two buffers
  uint32_t warp_key[WARPS], warp_slot[WARPS];
  int few[EV_FEW];         // the slots that go, when they are few
  uint32_t hist[2][EV_BINS];         // two passes' histograms in turn
  uint32_t coarse[2][EV_BINS / 32];  // and their sums over 32 bins
  uint32_t total[EV_BINS / 32], fine[32];  // sums over the cluster
  uint32_t scan[PER * WARPS];
  uint32_t scan2[PER * WARPS];
  uint32_t warp_sum[32], warp_sum2[32];
};

// Exclusive scan of n values in shared memory (n <= 1024, in place) over the block.
template <int THREADS>
__device__ __forceinline__ void block_scan(uint32_t* v, int n, uint32_t* warp_sum) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  __syncthreads();
  uint32_t run = 0;
  for (int base = 0; base < n; base += THREADS) {
    const int i = base + t;
    const uint32_t x = i < n ? v[i] : 0;
    uint32_t incl = x;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += up;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    // every warp scans the warps' sums
    const uint32_t own = lane < THREADS / 32 ? warp_sum[lane] : 0;
    uint32_t sums = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, sums, off);
      if (lane >= off) sums += up;
    }
    const uint32_t before = run + __shfl_sync(0xffffffffu, sums - own, warp);
    run += __shfl_sync(0xffffffffu, sums, 31);
    if (i < n) v[i] = before + incl - x;
    __syncthreads();
  }
}

struct EvictArgs {
  const float* weights;
  float* weights_out;
  const int* positions;
  int* positions_out;
  const int* next_position;
  int budget, sinks, recent;
  int* len_out;
  int* list;  // [batch * kv_heads][2][list_stride]: holes, movers
  int list_stride;
};

// Grid: (sequence * kv_heads + key head) * ctas + rank, clusters of `ctas`. A CTA holds
// THREADS * PER slots in order: slot = base + e * THREADS + thread.
template <int THREADS, int PER>
__global__ void __launch_bounds__(THREADS)
    paged_evict_kernel(const PagedKV kv, const EvictArgs a, int ctas) {
  __shared__ EvictShared<THREADS, PER> sm;
  constexpr int WARPS = THREADS / 32;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int rank = blockIdx.x % ctas;
  const int item = blockIdx.x / ctas;
  const int head = item % kv.kv_heads, b = item / kv.kv_heads;
  const int n = min(max(__ldg(kv.len + b), 0), kv.max_len);
  const int new_len = min(n, a.budget);
  if (rank == 0 && head == 0 && t == 0) a.len_out[b] = new_len;

  const bool copy_w = a.weights_out != a.weights, copy_p = a.positions_out != a.positions;
  const int base = rank * THREADS * PER;

  // ---- the keys. Written to another array, weights and positions of every slot below the
  // new length are copied at once (a hole's are overwritten when its mover comes).
  uint32_t key[PER];
  bool held = false;  // a slot below the new length is absent
  {
    const int recent_from = __ldg(a.next_position + b) - a.recent;
    constexpr int BATCH = PER < 8 ? PER : 8;  // loads in flight
#pragma unroll
    for (int e0 = 0; e0 < PER; e0 += BATCH) {
      int at[BATCH], p[BATCH];
      float w[BATCH];
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        const int s = base + (e0 + e) * THREADS + t;
        const int id = s < n ? kv.page_id(b, s) : -1;
        at[e] = id >= 0 ? kv.page_row(id, head, s) : -1;
      }
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        p[e] = at[e] >= 0 ? a.positions[at[e]] : 0;
        w[e] = at[e] >= 0 ? a.weights[at[e]] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        const int s = base + (e0 + e) * THREADS + t;
        const bool must = p[e] < a.sinks || (a.recent > 0 && p[e] >= recent_from);
        // 0: no slot, or an absent one behind the new length (never kept: as many others are there)
        key[e0 + e] = at[e] < 0 ? (s < new_len ? EV_HELD : 0u) : must ? EV_MUST : evict_key(w[e]);
        held |= at[e] < 0 && s < new_len;
        if (at[e] >= 0 && s < new_len) {
          if (copy_w) a.weights_out[at[e]] = w[e];
          if (copy_p) a.positions_out[at[e]] = p[e];
        }
      }
    }
  }
  if (n <= a.budget) return;  // everything stays (the whole cluster ends here)
  if (ctas > 1)  // the other CTAs' slots too
    for (int s = t << kv.page_shift; s < new_len; s += THREADS << kv.page_shift)
      held |= kv.page_id(b, s) < 0;
  if (__syncthreads_or(held)) {
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (base + e * THREADS + t >= new_len && key[e] != EV_MUST) key[e] = 0u;
  }

  auto cluster_barrier = [&] {
    __syncwarp();
    if (ctas > 1) cluster_sync(); else __syncthreads();
  };
  // One row, by a warp: lanes 0-15 K, 16-31 V, lane 0 also the weight and the position.
  auto pool = [&](int at) {
    return static_cast<uint4*>(lane < 16 ? kv.k : kv.v) + (size_t)at * (PG_HD / 8) + (lane & 15);
  };

  // ---- few slots go: look for each
  if (n - a.budget <= EV_FEW) {
    const int go = n - a.budget;
    uint32_t gone = 0;
    for (int round = 0; round < go; ++round) {
      uint32_t k = 0xffffffffu, top = 0;  // the smallest key, and its highest slot + 1
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int s = base + e * THREADS + t;
        if (s < n && !(gone >> e & 1u) && key[e] <= k) {
          k = key[e];
          top = (uint32_t)s + 1;
        }
      }
      uint32_t least = __reduce_min_sync(0xffffffffu, k);
      uint32_t slot = __reduce_max_sync(0xffffffffu, k == least ? top : 0u);
      if (lane == 0) {
        sm.warp_key[warp] = least;
        sm.warp_slot[warp] = slot;
      }
      __syncthreads();
      k = lane < WARPS ? sm.warp_key[lane] : 0xffffffffu;
      top = lane < WARPS ? sm.warp_slot[lane] : 0u;
      least = __reduce_min_sync(0xffffffffu, k);
      slot = __reduce_max_sync(0xffffffffu, k == least ? top : 0u);
      if (ctas > 1) {
        uint32_t* mine = sm.least[round & 1];
        if (t == 0) {
          mine[0] = least;
          mine[1] = slot;
        }
        __syncwarp();
        cluster_sync();
        // (a buffer is written again two rounds later, behind another cluster barrier)
        k = lane < ctas ? ld_cluster_u32(mapa_shared(smem_u32(mine), lane)) : 0xffffffffu;
        top = lane < ctas ? ld_cluster_u32(mapa_shared(smem_u32(mine + 1), lane)) : 0u;
        least = __reduce_min_sync(0xffffffffu, k);
        slot = __reduce_max_sync(0xffffffffu, k == least ? top : 0u);
      } else {
        __syncthreads();
      }
      const int out = (int)slot - 1, local = out - base;
      if (local >= 0 && local < THREADS * PER && local % THREADS == t) gone |= 1u << (local / THREADS);
      if (t == 0) sm.few[round] = out;
    }
    // no CTA leaves while another may still read its least; and the copies of phase one are done
    cluster_barrier();
    if (rank != 0) return;
    for (int i = warp; i < go; i += WARPS) {
      const int src = new_len + i;
      int nth = 0, dst = -1;
      bool stays = true;
      for (int j = 0; j < go; ++j) {
        const int f = sm.few[j];
        stays &= f != src;
      }
      if (!stays) continue;
      for (int c = 0; c < i; ++c) {  // kept slots behind the budget that come before this one
        bool kept = true;
        for (int j = 0; j < go; ++j) kept &= sm.few[j] != new_len + c;
        nth += kept;
      }
      for (int j = 0; j < go; ++j) {  // the hole of that number
        int lower = 0;
        for (int g = 0; g < go; ++g) lower += sm.few[g] < sm.few[j];
        if (sm.few[j] < new_len && lower == nth) dst = sm.few[j];
      }
      const int src_id = kv.page_id(b, src), dst_id = dst >= 0 ? kv.page_id(b, dst) : -1;
      if (src_id < 0 || dst_id < 0) continue;  // (neither is: absent slots stay out of both)
      const int from = kv.page_row(src_id, head, src), at = kv.page_row(dst_id, head, dst);
      *pool(at) = *pool(from);
      if (lane == 0) a.weights_out[at] = a.weights[from];
      if (lane == 1) a.positions_out[at] = a.positions[from];
    }
    return;
  }

  // Sums of three counts of this block over the cluster; `before`: over lower ranks only.
  // Three buffers in turn: the one cleared here was last read two barriers ago.
  int turn = 0;
  auto cluster_counts = [&](uint32_t (&c)[3], uint32_t (&before)[3]) {
    const int clear = turn == 2 ? 0 : turn + 1;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const uint32_t w = __reduce_add_sync(0xffffffffu, c[j]);
      if (lane == 0 && w) atomicAdd(&sm.count[turn][j], w);
    }
    if (t < 3) sm.count[clear][t] = 0;
    cluster_barrier();
    if (ctas > 1) {
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        const uint32_t got =
            lane < ctas ? ld_cluster_u32(mapa_shared(smem_u32(&sm.count[turn][j]), lane)) : 0u;
        c[j] = __reduce_add_sync(0xffffffffu, got);
        before[j] = __reduce_add_sync(0xffffffffu, lane < rank ? got : 0u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        c[j] = *const_cast<volatile uint32_t*>(&sm.count[turn][j]);
        before[j] = 0;
      }
    }
    turn = clear;
  };
  if (t < 3) sm.count[0][t] = 0;
  __syncthreads();

  // ---- the budget-th largest key T: the histogram of the keys within [T, T + 2^(shift + 11))
  // (all of them at first), the bin that holds it, and on within that bin. Of the other CTAs'
  // histograms only the sums over 32 bins and then the 32 bins in question are read (all of
  // them would be 64 KB a CTA and pass over the SMs' network).
  uint32_t T = 0;
  uint32_t want = (uint32_t)a.budget;  // that many of the range's largest keys stay
  bool exact = false;                  // all keys >= T stay
  // Two entries per lane, from the top down: the one with which their sum reaches `want`.
  auto reach = [&](uint32_t hi, uint32_t lo, uint32_t& above, uint32_t& inside) -> int {
    uint32_t incl = hi + lo;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += up;
    }
    const int src = __ffs(__ballot_sync(0xffffffffu, incl >= want)) - 1;
    const uint32_t before = incl - hi - lo;
    const bool second = before + hi < want;
    above = __shfl_sync(0xffffffffu, second ? before + hi : before, src);
    inside = __shfl_sync(0xffffffffu, second ? lo : hi, src);
    return 2 * src + (int)__shfl_sync(0xffffffffu, (uint32_t)second, src);
  };
  // Sums over the cluster of `count` words at the same place in every CTA, to `out`.
  auto gather = [&](const uint32_t* words, int count, uint32_t* out) {
    for (int i = t; i < count * 8; i += THREADS) {
      const int r = i & 7;
      uint32_t v = 0;
      if (ctas == 1)
        v = r == 0 ? words[i >> 3] : 0u;
      else if (r < ctas)
        v = ld_cluster_u32(mapa_shared(smem_u32(words + (i >> 3)), r));
#pragma unroll
      for (int off = 1; off < 8; off <<= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
      if (r == 0) out[i >> 3] = v;
    }
    __syncthreads();
  };
  int pass = 0;
  for (int shift = 21;; shift = shift == 21 ? 10 : 0, ++pass) {
    uint32_t* hist = sm.hist[pass & 1];
    uint32_t* coarse = sm.coarse[pass & 1];
    // (a buffer was last read two passes ago, two barriers of the cluster back)
    for (int i = t; i < EV_BINS; i += THREADS) hist[i] = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const uint32_t bin = (key[e] - T) >> shift;
      // (the last pass's range is 2^10: its bins are the lower half)
      if (base + e * THREADS + t < n && key[e] >= T && bin < (shift == 0 ? 1024u : EV_BINS))
        atomicAdd(&hist[bin], 1u);
    }
    __syncthreads();
    for (int i = warp; i < EV_BINS / 32; i += WARPS) {
      const uint32_t sum = __reduce_add_sync(0xffffffffu, hist[i * 32 + lane]);
      if (lane == 0) coarse[i] = sum;
    }
    cluster_barrier();
    uint32_t above, inside;
    gather(coarse, EV_BINS / 32, sm.total);
    const int big = EV_BINS / 32 - 1 - reach(sm.total[EV_BINS / 32 - 1 - 2 * lane],
                                             sm.total[EV_BINS / 32 - 2 - 2 * lane], above, inside);
    want -= above;
    gather(hist + big * 32, 32, sm.fine);
    const int bin = big * 32 + 31 - reach(lane < 16 ? sm.fine[31 - 2 * lane] : 0u,
                                          lane < 16 ? sm.fine[30 - 2 * lane] : 0u, above, inside);
    want -= above;
    T += (uint32_t)bin << shift;
    exact = inside == want;
    if (exact || shift == 0) break;
  }

  uint32_t keep = 0;  // bit e: this thread's element e stays
  if (exact) {
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (base + e * THREADS + t < n && key[e] >= T) keep |= 1u << e;
  } else {
    // of the keys equal to T only some stay, the lowest slots: number them
    uint32_t above[3] = {0, 0, 0}, above_before[3];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const bool equal = base + e * THREADS + t < n && key[e] == T;
      above[0] += key[e] > T;
      above[1] += equal;
      const unsigned eq = __ballot_sync(0xffffffffu, equal);
      if (lane == 0) sm.scan[e * WARPS + warp] = __popc(eq);
    }
    cluster_counts(above, above_before);
    const uint32_t equals_kept = (uint32_t)a.budget - above[0];
    block_scan<THREADS>(sm.scan, PER * WARPS, sm.warp_sum);
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const bool equal = base + e * THREADS + t < n && key[e] == T;
      const unsigned eq = __ballot_sync(0xffffffffu, equal);
      const uint32_t place =
          above_before[1] + sm.scan[e * WARPS + warp] + __popc(eq & ((1u << lane) - 1));
      if (key[e] > T || (equal && place < equals_kept)) keep |= 1u << e;
    }
    __syncthreads();
  }

  // ---- number the holes and the movers in slot order
  uint32_t own[3] = {0, 0, 0}, first[3];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int s = base + e * THREADS + t;
    const bool kept = keep >> e & 1u;
    const unsigned hole = __ballot_sync(0xffffffffu, s < new_len && !kept);
    const unsigned mover = __ballot_sync(0xffffffffu, s >= new_len && kept);
    own[0] += s < new_len && !kept;
    own[1] += s >= new_len && kept;
    if (lane == 0) {
      sm.scan[e * WARPS + warp] = __popc(hole);
      sm.scan2[e * WARPS + warp] = __popc(mover);
    }
  }
  cluster_counts(own, first);
  const int moves = (int)own[0];  // as many holes as movers
  block_scan<THREADS>(sm.scan, PER * WARPS, sm.warp_sum);
  block_scan<THREADS>(sm.scan2, PER * WARPS, sm.warp_sum2);
  int* holes = a.list + (size_t)item * 2 * a.list_stride;
  int* movers = holes + a.list_stride;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int s = base + e * THREADS + t;
    const bool kept = keep >> e & 1u;
    const unsigned hole = __ballot_sync(0xffffffffu, s < new_len && !kept);
    const unsigned mover = __ballot_sync(0xffffffffu, s >= new_len && kept);
    const unsigned below = (1u << lane) - 1;
    if (s < new_len && !kept)
      holes[first[0] + sm.scan[e * WARPS + warp] + __popc(hole & below)] = s;
    if (s >= new_len && kept)
      movers[first[1] + sm.scan2[e * WARPS + warp] + __popc(mover & below)] = s;
  }
  cluster_barrier();  // the lists are whole; no CTA reads another's counts behind this

  // ---- move: a warp takes 16 rows at a time, whose places its lanes look up together
  const int stride = ctas * WARPS * 16;
  for (int i0 = (rank * WARPS + warp) * 16; i0 < moves; i0 += stride) {
    int from = -1, at = -1;
    if (lane < 16 && i0 + lane < moves) {
      const int src = __ldcg(movers + i0 + lane), dst = __ldcg(holes + i0 + lane);
      const int src_id = kv.page_id(b, src), dst_id = kv.page_id(b, dst);
      if (src_id >= 0 && dst_id >= 0) {  // (both are: absent slots are in neither list)
        from = kv.page_row(src_id, head, src);
        at = kv.page_row(dst_id, head, dst);
      }
    }
    float w = 0.f;
    int p = 0;
    if (from >= 0) {
      w = a.weights[from];
      p = a.positions[from];
    }
#pragma unroll
    for (int half = 0; half < 16; half += 8) {
      uint4 x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = __shfl_sync(0xffffffffu, from, half + j);
        if (row >= 0) x[j] = *pool(row);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = __shfl_sync(0xffffffffu, at, half + j);
        if (row >= 0) *pool(row) = x[j];
      }
    }
    if (from >= 0) {
      a.weights_out[at] = w;
      a.positions_out[at] = p;
    }
  }
}

}  // namespace cb
