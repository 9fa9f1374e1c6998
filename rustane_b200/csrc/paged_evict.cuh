// Eviction from a paged cache by accumulated attention weight.
//
// One cluster of CTAs per (sequence, key head). Every slot gets a 32-bit key whose unsigned
// order is the order of keeping: all ones for the positions that must stay, else the
// weight's bits made monotone (NaN lowest). The budget-th largest key is found two bits a
// pass by counting (16 passes over keys that stay in registers: no atomics, so no pile-up on
// the few exponents that weights have, and the result does not depend on any order). Keys
// above it stay, of those equal to it the lowest slots. Then the i-th slot below the budget
// that is not kept (a hole) takes the i-th kept slot behind the budget (a mover); the
// numbering is a scan over ballots. Holes and movers are disjoint ranges of slots, so all
// rows move at once and in place. Reading the weights and positions and moving the rows is
// the work that cannot be left out: the kernel is bound by the latency of the passes for
// short sequences and by the moved rows for long ones, which is why a long sequence gets
// several CTAs (they share the counts through distributed shared memory).
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

// Per-block counts of up to three predicates per element, in one word each.
template <int THREADS, int PER>
struct EvictShared {
  static constexpr int WARPS = THREADS / 32;
  uint32_t part[3][WARPS];
  uint32_t cluster[2][3];  // this CTA's counts, read by the others; two buffers in turn
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
    uint32_t before = run;
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += warp_sum[w];
      run += warp_sum[w];
    }
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

  auto meta = [&](int slot, int id) { return (size_t)kv.page_row(id, head, slot); };
  const bool out_of_place_w = a.weights_out != a.weights;
  const bool out_of_place_p = a.positions_out != a.positions;
  const int base = rank * THREADS * PER;

  if (n <= a.budget) {  // everything stays (the whole cluster takes this branch)
    for (int s = base + t; s < min(n, base + THREADS * PER); s += THREADS) {
      const int id = kv.page_id(b, s);
      if (id < 0) continue;
      const size_t at = meta(s, id);
      if (out_of_place_w) a.weights_out[at] = a.weights[at];
      if (out_of_place_p) a.positions_out[at] = a.positions[at];
    }
    return;
  }

  // ---- the keys
  uint32_t key[PER];
  {
    const int recent_from = __ldg(a.next_position + b) - a.recent;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int s = base + e * THREADS + t;
      key[e] = 0;  // no slot, or one that is absent: kept last
      if (s < n) {
        const int id = kv.page_id(b, s);
        if (id >= 0) {
          const size_t at = meta(s, id);
          const int p = a.positions[at];
          const bool must = p < a.sinks || (a.recent > 0 && p >= recent_from);
          key[e] = must ? 0xffffffffu : evict_key(a.weights[at]);
        }
      }
    }
  }

  // Sums of this block's three counts over the cluster; `before` those of lower ranks only.
  int turn = 0;
  auto cluster_counts = [&](uint32_t (&c)[3], uint32_t (&before)[3]) {
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      c[j] = __reduce_add_sync(0xffffffffu, c[j]);
      if (lane == 0) sm.part[j][warp] = c[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      c[j] = __reduce_add_sync(0xffffffffu, lane < WARPS ? sm.part[j][lane] : 0u);
      before[j] = 0;
    }
    if (ctas > 1) {
      if (t < 3) sm.cluster[turn][t] = t == 0 ? c[0] : t == 1 ? c[1] : c[2];
      __syncwarp();
      cluster_sync();
      // A buffer is written again two calls later, behind another cluster barrier.
      uint32_t got = 0;
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        got = lane < ctas ? ld_cluster_u32(mapa_shared(smem_u32(&sm.cluster[turn][j]), lane)) : 0u;
        c[j] = __reduce_add_sync(0xffffffffu, got);
        before[j] = __reduce_add_sync(0xffffffffu, lane < rank ? got : 0u);
      }
      turn ^= 1;
    } else {
      __syncthreads();
    }
  };

  // ---- the budget-th largest key: the largest T with at least `budget` keys >= T
  uint32_t T = 0, dummy[3];
  for (int shift = 30; shift >= 0; shift -= 2) {
    uint32_t c[3] = {0, 0, 0};
    const uint32_t t1 = T | (1u << shift), t2 = T | (2u << shift), t3 = T | (3u << shift);
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      c[0] += key[e] >= t1;
      c[1] += key[e] >= t2;
      c[2] += key[e] >= t3;
    }
    cluster_counts(c, dummy);
    const uint32_t want = (uint32_t)a.budget;
    T = c[2] >= want ? t3 : c[1] >= want ? t2 : c[0] >= want ? t1 : T;
  }

  // ---- how many keys equal to T stay, and where this thread's equals lie among all
  uint32_t above[3] = {0, 0, 0}, above_before[3];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const bool slot = base + e * THREADS + t < n;
    above[0] += key[e] > T;
    above[1] += slot && key[e] == T;
  }
  cluster_counts(above, above_before);
  const uint32_t equals_kept = (uint32_t)a.budget - above[0];

  uint32_t keep = 0;  // bit e: this thread's element e stays
  if (above[1] == equals_kept) {
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (base + e * THREADS + t < n && key[e] >= T) keep |= 1u << e;
  } else {
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const unsigned eq = __ballot_sync(0xffffffffu, base + e * THREADS + t < n && key[e] == T);
      if (lane == 0) sm.scan[e * WARPS + warp] = __popc(eq);
    }
    block_scan<THREADS>(sm.scan, PER * WARPS, sm.warp_sum);
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const bool slot = base + e * THREADS + t < n;
      const unsigned eq = __ballot_sync(0xffffffffu, slot && key[e] == T);
      const uint32_t place =
          above_before[1] + sm.scan[e * WARPS + warp] + __popc(eq & ((1u << lane) - 1));
      if (slot && (key[e] > T || (key[e] == T && place < equals_kept))) keep |= 1u << e;
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
    if (lane == 0) {
      sm.scan[e * WARPS + warp] = __popc(hole);
      sm.scan2[e * WARPS + warp] = __popc(mover);
      own[0] += __popc(hole);
      own[1] += __popc(mover);
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
    if (s < new_len && kept && (out_of_place_w || out_of_place_p)) {
      const int id = kv.page_id(b, s);
      if (id >= 0) {
        const size_t at = meta(s, id);
        if (out_of_place_w) a.weights_out[at] = a.weights[at];
        if (out_of_place_p) a.positions_out[at] = a.positions[at];
      }
    }
  }
  __syncwarp();
  if (ctas > 1) cluster_sync(); else __syncthreads();  // the lists are whole

  // ---- move: a warp takes four rows at a time, lanes 0-15 K and 16-31 V
  constexpr int ROWS = 4;
  const int stride = ctas * WARPS * ROWS;
  for (int i0 = (rank * WARPS + warp) * ROWS; i0 < moves; i0 += stride) {
    uint4 x[ROWS];
    int64_t to[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      to[j] = -1;
      if (i0 + j >= moves) continue;
      const int src = __ldcg(movers + i0 + j), dst = __ldcg(holes + i0 + j);
      const int src_id = kv.page_id(b, src), dst_id = kv.page_id(b, dst);
      if (src_id < 0 || dst_id < 0) continue;  // a slot that is absent
      const size_t from = meta(src, src_id), at = meta(dst, dst_id);
      const uint4* pool = static_cast<const uint4*>(lane < 16 ? kv.k : kv.v);
      x[j] = pool[from * (PG_HD / 8) + (lane & 15)];
      to[j] = (int64_t)at;
      if (lane == 0) a.weights_out[at] = a.weights[from];
      if (lane == 1) a.positions_out[at] = a.positions[from];
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
      if (to[j] >= 0)
        static_cast<uint4*>(lane < 16 ? kv.k : kv.v)[to[j] * (PG_HD / 8) + (lane & 15)] = x[j];
  }
  // no CTA leaves while another may still read its counts: the last reads of them lie
  // before the barrier above
}

}  // namespace cb
