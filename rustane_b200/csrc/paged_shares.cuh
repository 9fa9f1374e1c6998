// Equal shares of a step's attention work.
//
// The query rows of each key head in each sequence are cut into tiles of ROWS, a tile's keys
// into steps of KEYS. Sequences differ in length, so the steps of all tiles (sequence, key
// head, tile in this order: neighbours share K and V in L2), and UNITS more per tile for its
// own cost, are laid end to end, and every worker takes an equal share of these units. A
// worker that has all steps of a tile writes its output; of a tile that is cut, each worker
// writes its part (at most two: its first and its last tile), and a second kernel joins them.
// Units are counted in 32 bits (the host refuses steps that could have 2^31 of them).
#pragma once
#include "paged_common.cuh"

namespace cb {

constexpr int SHARE_CHUNK = 1024;  // sequences whose units are added up at a time

// What is to be joined: one record per worker, the tile that begins in its share and goes on
// behind it. Part 2 w is worker w's first segment, 2 w + 1 its last one.
struct ShareJoin {
  int count;  // parts, 0 = no such tile
  int first;  // part of this worker; the others are 2 (w + 1), 2 (w + 2), ...
  int row0, head, f0, rows;
};
struct ShareParts {
  float* o;    // the parts' outputs, normalised within the part
  float* lse;  // and base-2 log-sum-exps
  ShareJoin* join;
};
__device__ __forceinline__ int share_part(const ShareJoin& jn, int worker, int p) {
  return p == 0 ? jn.first : 2 * (worker + p);
}

struct ShareTable {  // in shared memory
  uint32_t seq_units[SHARE_CHUNK];
  uint32_t base, longer;  // the first `longer` workers have base + 1 units, the others base
  uint32_t workers;       // with a share

  __device__ __forceinline__ uint32_t begin_of(uint32_t worker) const {
    return base * worker + min(worker, longer);
  }
  __device__ __forceinline__ uint32_t worker_of(uint32_t unit) const {
    const uint32_t border = (base + 1) * longer;
    const uint32_t worker = unit < border ? unit / (base + 1) : longer + (unit - border) / base;
    return min(worker, workers - 1);
  }
};

// LEAST: units of a share at least; above UNITS, so that every share has a step.
template <int ROWS, int KEYS, int UNITS, int LEAST>
struct PagedShares {
  static_assert(LEAST > UNITS, "a share without a step");

  // Steps of a tile: up to the last slot that its last row sees. A tile that sees nothing has
  // one step too (in which everything is masked): it writes its zeros.
  static __device__ __forceinline__ int tile_steps(const PagedSeq& seq, int group, int tile) {
    const int last = min((tile + 1) * ROWS, seq.n * group) - 1;
    return max(1, (seq.limit(last / group) + KEYS - 1) / KEYS);
  }
  static __device__ __forceinline__ int tiles(const PagedSeq& seq, int group) {
    return (seq.n * group + ROWS - 1) / ROWS;
  }

  // A worker's walk over its share: segments of tiles.
  struct Walk {
    PagedSeq seq;
    int b, head, tile;
    int u0;             // the segment's first unit within the tile
    int j0, j1, steps;  // the segment: steps j0 .. j1 - 1 of the tile's `steps`
    uint32_t at, end;   // the segment's first unit among all, and the share's end

    __device__ __forceinline__ int u1() const {
      return min(steps + UNITS, u0 + (int)(end - at));
    }
    __device__ __forceinline__ void segment(int group) {
      steps = tile_steps(seq, group, tile);
      j0 = max(0, u0 - UNITS);
      j1 = max(0, u1() - UNITS);
    }
    // The next segment; false when the share is done.
    __device__ __forceinline__ bool next(const PagedKV& kv, int group) {
      do {
        at += (uint32_t)(u1() - u0);
        if (at >= end) return false;
        u0 = 0;
        if (++tile >= tiles(seq, group)) {
          tile = 0;
          if (++head >= kv.kv_heads) {
            head = 0;
            do {
              if (++b >= kv.batch) return false;
              seq = paged_seq(kv, b);
            } while (seq.n == 0);
          }
        }
        segment(group);
      } while (j1 == j0);  // a share may end before a tile's first step
      return true;
    }
    __device__ __forceinline__ bool whole() const { return j0 == 0 && j1 == steps; }
    __device__ __forceinline__ int rows(int group) const {
      return min(ROWS, seq.n * group - tile * ROWS);
    }
    // The join record of a segment that begins its tile and does not end it.
    __device__ __forceinline__ ShareJoin join(const ShareTable& table, int worker, int part,
                                              int group) const {
      ShareJoin jn;
      jn.count = (int)table.worker_of(at - u0 + UNITS + steps - 1) - worker + 1;
      jn.first = part;
      jn.row0 = seq.row0;
      jn.head = head;
      jn.f0 = tile * ROWS;
      jn.rows = rows(group);
      return jn;
    }
  };

  // The whole block: adds up the units of all sequences and puts every warp's walk at the
  // beginning of its share (workers 0 .. most - 1; warps may be of one worker or of several).
  // False in the warps whose worker has none.
  static __device__ __forceinline__ bool begin(const PagedKV& kv, int group, ShareTable& table,
                                               int most, int worker, Walk& walk) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int warps = blockDim.x >> 5;
    // A warp per sequence where sequences are few and have many tiles, else a thread (their
    // loads are one after another).
    const bool by_warp = kv.max_new * group > 8 * ROWS && kv.batch <= 8 * warps;
    auto add_up = [&](int base, int count) {
      if (by_warp) {
        for (int i = warp; i < count; i += warps) {
          const PagedSeq s = paged_seq(kv, base + i);
          const int n_tiles = tiles(s, group);
          uint32_t n = 0;
          for (int t = lane; t < n_tiles; t += 32) n += tile_steps(s, group, t) + UNITS;
          n = __reduce_add_sync(0xffffffffu, n);
          if (lane == 0) table.seq_units[i] = n;
        }
      } else {
        for (int i = threadIdx.x; i < count; i += blockDim.x) {
          const PagedSeq s = paged_seq(kv, base + i);
          const int n_tiles = tiles(s, group);
          uint32_t n = 0;
          for (int t = 0; t < n_tiles; ++t) n += tile_steps(s, group, t) + UNITS;
          table.seq_units[i] = n;
        }
      }
      __syncthreads();
    };
    auto inclusive = [&](uint32_t n) {
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, n, off);
        if (lane >= off) n += up;
      }
      return n;
    };
    uint32_t total = 0;  // of one key head
    for (int base = 0; base < kv.batch; base += SHARE_CHUNK) {
      const int count = min(SHARE_CHUNK, kv.batch - base);
      __syncthreads();
      add_up(base, count);
      uint32_t n = 0;
      for (int i = lane; i < count; i += 32) n += table.seq_units[i];
      total += __reduce_add_sync(0xffffffffu, n);
    }
    const uint32_t all = total * kv.kv_heads;
    const uint32_t workers = max(1u, min((uint32_t)most, all / LEAST));
    if (threadIdx.x == 0) {
      table.base = all / workers;
      table.longer = all - all / workers * workers;
      table.workers = workers;
    }
    __syncthreads();
    const uint32_t lo = (uint32_t)worker < workers ? table.begin_of(worker) : all;
    const uint32_t hi = (uint32_t)worker < workers ? table.begin_of(worker + 1) : all;
    // heads of one sequence lie side by side: unit lo lies in the sequence that holds unit
    // lo / kv_heads of one head
    const uint32_t want = lo / kv.kv_heads;
    uint32_t before = 0;  // units of one head of the sequences in front
    bool found = lo >= hi, placed = false;
    for (int base = 0; base < kv.batch; base += SHARE_CHUNK) {
      const int count = min(SHARE_CHUNK, kv.batch - base);
      if (kv.batch > SHARE_CHUNK) {
        __syncthreads();
        add_up(base, count);
      }
      for (int i0 = 0; i0 < count && !found; i0 += 32) {
        const uint32_t n = i0 + lane < count ? table.seq_units[i0 + lane] : 0;
        const uint32_t incl = inclusive(n);
        const unsigned past = __ballot_sync(0xffffffffu, before + incl > want);
        if (!past) {
          before += __shfl_sync(0xffffffffu, incl, 31);
          continue;
        }
        found = true;
        const int src = __ffs(past) - 1, b = base + i0 + src;
        const uint32_t one = __shfl_sync(0xffffffffu, n, src);
        uint32_t r = lo - (before + __shfl_sync(0xffffffffu, incl - n, src)) * kv.kv_heads;
        const uint32_t head = r / one;
        if (head >= (uint32_t)kv.kv_heads) break;  // (row starts that do not ascend)
        r -= head * one;
        const PagedSeq s = paged_seq(kv, b);
        const int n_tiles = tiles(s, group);
        uint32_t run = 0;
        for (int t0 = 0; t0 < n_tiles; t0 += 32) {
          const uint32_t m = t0 + lane < n_tiles ? tile_steps(s, group, t0 + lane) + UNITS : 0;
          const uint32_t sum = inclusive(m);
          const unsigned in = __ballot_sync(0xffffffffu, run + sum > r);
          if (in) {
            bool some = true;
            if (lane == __ffs(in) - 1) {
              walk.seq = s;
              walk.b = b;
              walk.head = (int)head;
              walk.tile = t0 + lane;
              walk.u0 = (int)(r - run - (sum - m));
              walk.at = lo;
              walk.end = hi;
              walk.segment(group);
              if (walk.j1 == walk.j0) some = walk.next(kv, group);
            }
            placed = __all_sync(0xffffffffu, some);
            break;
          }
          run += __shfl_sync(0xffffffffu, sum, 31);
        }
      }
    }
    __syncthreads();
    return placed;
  }
};

}  // namespace cb
