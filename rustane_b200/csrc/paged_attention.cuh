// Attention of new tokens over a paged cache, for few query rows per key head (a decode
// step), and the attention weight that every slot got from a step.
//
// The query rows of one key head in one sequence, n tokens x `group` heads (row f = token
// f / group, head f % group), are cut into tiles of 16: the m16n8k16 matrix instruction's
// rows. Per tile
//   s_rk = scale log2(e) q_r . k_k,  m = max_k s, l = sum_k 2^(s - m),
//   o_r = sum_k 2^(s_rk - m) v_k / l
// with the running maximum and sum (32 bits) of an online softmax. K and V are read once per
// 16 rows, so for a decode step the kernel is bound by the reads of the cache. The sum is a
// compensated one: a lane adds a term per block, and where one slot far outweighs the others each
// of 30000 plain additions would round the same way (the log-sum-exp was off by 6e-4).
//
// A warp is a worker of its own (paged_shares.cuh): it takes an equal share of all tiles'
// blocks of 16 keys through a ring that TMA fills, running ahead over the borders of tiles, and
// meets no other warp until the join. (A CTA per tile and part of the keys, whose four warps
// joined in shared memory, left the SMs idle at every CTA's start and end and in the last
// wave: 76 us for the first case below, where this form then took 65.)
//
// Measured: 4 x up to 32768 slots, 32 / 8 heads, bf16, 331 MB: 66.9 us, 4.9 TB/s; 64 x up to 512
// slots, 12 / 12 heads, f16, 111 MB: 25.8 us, 4.3 TB/s. The walk to a worker's first block comes
// before the reads, the slowest SM's tail and the join (alone and cold: 12 and 7 us) behind them.
//
// A weight of 0 does not keep an infinity or NaN out of a product. V of slots behind the
// sequence's end, which may hold anything, reads as 0; and of the slots that only later ones of
// the step's tokens see, infinities and NaN read as 0 and are added afterwards to the rows that
// do see them.
#pragma once
#include "paged_shares.cuh"

namespace cb {

constexpr int PR_ROWS = 16;    // query rows of a tile
constexpr int PR_WARPS = 8;    // one CTA per SM
constexpr int PR_STAGES = 3;   // blocks in flight per warp
constexpr int PR_BLOCK = 16;   // keys of a block
constexpr int PR_STAGE_BYTES = 2 * PR_BLOCK * PG_HD * 2;  // K and V
constexpr int PR_RING = PR_WARPS * PR_STAGES * PR_STAGE_BYTES;
// A tile counts two blocks for its Q and its output (one to four measured within 4 %).
using PrShares = PagedShares<PR_ROWS, PR_BLOCK, 2, 6>;

struct PrShared {  // behind the ring
  uint64_t full[PR_WARPS][PR_STAGES];
  int absent[PR_WARPS][PR_STAGES];  // the block's page is outside the pool
  int failed;
  PrShares::Walk use[PR_WARPS], ahead[PR_WARPS];  // of what is computed, and loaded
  ShareTable table;
};
constexpr int PR_SMEM = PR_RING + (int)sizeof(PrShared) + 1024;
static_assert(PR_SMEM <= 232448, "shared memory");

// Sum over the four lanes of a quad (the columns of an accumulator row).
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}

// Parts: o [2 workers][16 rows][128], lse [2 workers][16]; worker = warp * gridDim + CTA.
template <typename T, bool LOADS>
__global__ void __launch_bounds__(PR_WARPS * 32, 1)
    paged_rows_kernel(const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const PagedKV kv,
                      const T* __restrict__ q, int64_t q_stride, int heads, float scale_log2,
                      T* __restrict__ out, int64_t out_stride, float* __restrict__ lse,
                      const ShareParts parts) {
  using H = Half16<T>;
  extern __shared__ uint8_t pr_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(pr_smem_raw) + 1023) & ~uintptr_t(1023));
  PrShared& sh = *reinterpret_cast<PrShared*>(smem + PR_RING);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = heads / kv.kv_heads;
  const int worker = warp * gridDim.x + blockIdx.x;
  uint8_t* ring = smem + warp * PR_STAGES * PR_STAGE_BYTES;
  uint64_t* full = sh.full[warp];
  PrShares::Walk& w = sh.use[warp];
  PrShares::Walk& ahead = sh.ahead[warp];
  if (lane == 0) {
    for (int i = 0; i < PR_STAGES; ++i) mbar_init(&full[i], 1);
    sh.failed = 0;
    fence_mbar_init();
  }
  pdl_launch_dependents();  // (the join; it waits for this kernel's end)
  const bool some_work = PrShares::begin(kv, group, sh.table, gridDim.x * PR_WARPS, worker, w);
  if (lane == 0) parts.join[worker].count = 0;  // (set below where a tile goes on)
  if (!some_work) return;

  // Lane 0 loads: block next_j of `ahead`, whose page's id was asked for one block before.
  bool more = false;
  int next_j = 0, next_id = -1;
  uint32_t loaded = 0;  // blocks
  auto issue = [&](int id) {
    const int stage = loaded % PR_STAGES;
    // rows behind the matrix read as zero (a page outside the pool)
    const int row = id >= 0 ? kv.page_row(id, ahead.head, next_j * PR_BLOCK) : kv.cache_rows();
    uint8_t* dst = ring + stage * PR_STAGE_BYTES;
    sh.absent[warp][stage] = id < 0;
    if constexpr (LOADS) {
      mbar_arrive_expect_tx(&full[stage], PR_STAGE_BYTES);
      tma_load_2d(dst, &tmK, &full[stage], 0, row);
      tma_load_2d(dst + 2048, &tmK, &full[stage], 64, row);
      tma_load_2d(dst + 4096, &tmV, &full[stage], 0, row);
      tma_load_2d(dst + 6144, &tmV, &full[stage], 64, row);
      ++loaded;
    }
    if (++next_j == ahead.j1) {
      more = ahead.next(kv, group);
      next_j = ahead.j0;
    }
  };
  auto id_of = [&](const PrShares::Walk& x, int j) {
    return j * PR_BLOCK < x.seq.end ? kv.page_id(x.b, j * PR_BLOCK) : -1;
  };
  {
    // the ring's first blocks: a lane each asks for their ids (of the first segment) at once
    const int n = w.j1 - w.j0;
    const int id = lane < min(n, PR_STAGES) ? id_of(w, w.j0 + lane) : -1;
    if (lane == 0) {
      ahead = w;
      more = true;
      next_j = ahead.j0;
    }
#pragma unroll
    for (int i = 0; i < PR_STAGES; ++i) {
      const int id_i = __shfl_sync(0xffffffffu, id, i);
      if (lane == 0 && more) issue(i < n ? id_i : id_of(ahead, next_j));
    }
    if (more) next_id = id_of(ahead, next_j);
  }
  __syncwarp();

  const int r0 = lane >> 2, c2 = (lane & 3) * 2;
  uint32_t g = 0;  // blocks used
  bool first_segment = true, ok = true, go_on;
  do {
    const PagedSeq seq = w.seq;
    const int head = w.head, f0 = w.tile * PR_ROWS, rows = w.rows(group);
    const int j0 = w.j0, j1 = w.j1;
    // Q fragments: rows lane / 4 and lane / 4 + 8, elements 2 (lane % 4) (+ 1, + 8, + 9)
    uint32_t qf[8][4];
    int lim[2];
    int64_t row_of[2];
    int head_of[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = r0 + 8 * j;
      const int f = f0 + min(r, rows - 1);
      const int i = f / group;
      lim[j] = r < rows ? seq.limit(i) : 0;
      row_of[j] = seq.row0 + i;
      head_of[j] = head * group + f - i * group;
      const T* qp = q + row_of[j] * q_stride + (int64_t)head_of[j] * PG_HD + c2;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        qf[k][j] = *reinterpret_cast<const uint32_t*>(qp + k * 16);
        qf[k][j + 2] = *reinterpret_cast<const uint32_t*>(qp + k * 16 + 8);
      }
    }
    const int lim_min = seq.limit(f0 / group);

    float o[16][4];
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    // the running maximum, less P_UP, and sum
    float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};
    float l_over[2] = {0.f, 0.f};  // what l's roundings have added to it
    bool odd_v = false;  // an infinity or NaN was taken out of V

    for (int jb = j0; ok && jb < j1; ++jb, ++g) {
      const int stage = g % PR_STAGES;
      const int key0 = jb * PR_BLOCK;
      ok = __all_sync(0xffffffffu,
                      paged_wait<LOADS>(&full[stage], (g / PR_STAGES) & 1, &sh.failed));
      if (!ok) break;
      const uint32_t kb = smem_u32(ring + stage * PR_STAGE_BYTES), vb = kb + 4096;
      const bool absent = sh.absent[warp][stage] != 0;
      float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      {
        const int row = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int chunk = (k & 3) * 2 + ((lane >> 3) & 1);
          uint32_t kf[4];
          ldmatrix_x4(kf, kb + (k >> 2) * 2048 + row * 128 + ((chunk ^ (row & 7)) << 4));
          H::mma(s[0], qf[k], kf[0], kf[1]);
          H::mma(s[1], qf[k], kf[2], kf[3]);
        }
      }
      if (absent || key0 + PR_BLOCK > lim_min) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (absent || key0 + n * 8 + c2 + (j & 1) >= lim[j >> 1]) s[n][j] = -CUDART_INF_F;
      }
      float base[2], corr[2];
      bool grew = false;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float mx = fmaf(quad_max(fmaxf(fmaxf(s[0][2 * j], s[0][2 * j + 1]),
                                             fmaxf(s[1][2 * j], s[1][2 * j + 1]))),
                              scale_log2, -H::P_UP);
        const float mn = fmaxf(m[j], mx);
        base[j] = mn == -CUDART_INF_F ? 0.f : mn;
        grew |= mn > m[j];
        corr[j] = exp2_mufu(m[j] - base[j]);  // 0 for a row that had seen nothing
        m[j] = mn;
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          l[j] *= corr[j];
          l_over[j] *= corr[j];
        }
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          o[n][0] *= corr[0];
          o[n][1] *= corr[0];
          o[n][2] *= corr[1];
          o[n][3] *= corr[1];
        }
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = exp2_mufu(fmaf(s[n][j], scale_log2, -base[j >> 1]));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float term =
            (s[0][2 * j] + s[0][2 * j + 1]) + (s[1][2 * j] + s[1][2 * j + 1]) - l_over[j];
        const float sum = l[j] + term;
        l_over[j] = (sum - l[j]) - term;
        l[j] = sum;
      }
      // P rounds to the cache's type (the matrix instruction takes one type for both sides): at
      // most half a step of each weight, the size of the output's own rounding (fp16: or 2^-40 of
      // the largest weight).
      const uint32_t pf[4] = {H::pack(s[0][0], s[0][1]), H::pack(s[0][2], s[0][3]),
                              H::pack(s[1][0], s[1][1]), H::pack(s[1][2], s[1][3])};
      uint32_t v_mask[2] = {0xffffffffu, 0xffffffffu};
      const bool v_whole = key0 + PR_BLOCK <= lim_min;  // every row sees every slot
      if (!v_whole) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int key = key0 + c2 + 8 * j;
          v_mask[j] = (key < seq.end ? 0xffffu : 0u) | (key + 1 < seq.end ? 0xffff0000u : 0u);
        }
      }
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int row = lane & 15, chunk = (n & 3) * 2 + (lane >> 4);
        uint32_t vf[4];
        ldmatrix_x4_trans(vf, vb + (n >> 2) * 2048 + row * 128 + ((chunk ^ (row & 7)) << 4));
        if (!v_whole) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            vf[j] &= v_mask[j & 1];
            const uint32_t bad = H::not_finite(vf[j]);
            odd_v |= bad != 0;
            vf[j] &= ~bad;
          }
        }
        H::mma(o[2 * n], pf, vf[0], vf[1]);
        H::mma(o[2 * n + 1], pf, vf[2], vf[3]);
      }
      __syncwarp();  // every lane has read the stage
      if (lane == 0 && more) {
        issue(next_id);
        if (more) next_id = id_of(ahead, next_j);
      }
    }
    if (__any_sync(0xffffffffu, odd_v)) {
      for (int key = max(j0, lim_min / PR_BLOCK) * PR_BLOCK;
           key < min(j1 * PR_BLOCK, seq.end); ++key) {
        const int id = kv.page_id(w.b, key);
        if (id < 0) continue;
        const T* v = static_cast<const T*>(kv.v) + (int64_t)kv.page_row(id, head, key) * PG_HD + c2;
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          const uint32_t x = *reinterpret_cast<const uint32_t*>(v + n * 8);
          const float2 odd = H::unpack(x & H::not_finite(x));
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (key < lim[j]) {
              o[n][2 * j] += odd.x;
              o[n][2 * j + 1] += odd.y;
            }
        }
      }
    }
    // ---- the segment's output
    const bool whole = w.whole();
    const int part = 2 * worker + (first_segment ? 0 : 1);
    if (lane == 0 && !whole && j0 == 0)  // begins here, goes on in the next shares
      parts.join[worker] = w.join(sh.table, worker, part, group);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      l[j] = quad_sum(l[j]);
      const int r = r0 + 8 * j;
      if (!ok) l[j] = CUDART_NAN_F;  // a wait ran out, here or in a segment before
      const float inv = l[j] == 0.f ? 0.f : 1.0f / l[j];  // a row that sees nothing: 0
      const float row_lse =
          l[j] == 0.f ? -CUDART_INF_F : m[j] + H::P_UP + log2f(l[j] * exp2f(-H::P_UP));
      if (r < rows) {
        if (whole) {
          T* po = out + row_of[j] * out_stride + (int64_t)head_of[j] * PG_HD + c2;
#pragma unroll
          for (int n = 0; n < 16; ++n)
            *reinterpret_cast<uint32_t*>(po + n * 8) =
                H::pack(o[n][2 * j] * inv, o[n][2 * j + 1] * inv);
          if (lse && c2 == 0) lse[row_of[j] * heads + head_of[j]] = row_lse;
        } else {
          float* po = parts.o + ((int64_t)part * PR_ROWS + r) * PG_HD + c2;
#pragma unroll
          for (int n = 0; n < 16; ++n)
            *reinterpret_cast<float2*>(po + n * 8) =
                make_float2(o[n][2 * j] * inv, o[n][2 * j + 1] * inv);
          if (c2 == 0) parts.lse[part * PR_ROWS + r] = row_lse;
        }
      }
    }
    first_segment = false;
    __syncwarp();
    go_on = false;
    if (lane == 0) go_on = w.next(kv, group);
    go_on = __any_sync(0xffffffffu, go_on);
  } while (go_on);
  if (!ok && lane == 0) {
    for (uint32_t x = g; x < loaded; ++x)
      paged_drain<LOADS>(&full[x % PR_STAGES], (x / PR_STAGES) & 1);
    paged_report_timeout();
  }
}

// Joins the parts of the tiles that begin in a worker's share and go on behind it:
// out = sum_p 2^(lse_p - lse) o_p, lse = log2 sum_p 2^lse_p. Block (x, y) looks after workers
// k * gridDim.x + x, k < 8, and the rows y, y + gridDim.y, ...: warp k after worker k's tile
// where the parts are few, all warps after one where they are many.
template <typename T>
__global__ void __launch_bounds__(PR_WARPS * 32)
    paged_rows_join_kernel(const ShareParts parts, int heads, int group, T* __restrict__ out,
                           int64_t out_stride, float* __restrict__ lse) {
  using H = Half16<T>;
  constexpr int FEW = 8;
  __shared__ float sm_m[PR_WARPS], sm_l[PR_WARPS];
  __shared__ float4 sm_o[PR_WARPS][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  // parts p0, p0 + step, ... of a row
  auto merge = [&](const ShareJoin& jn, int worker, int r, int p0, int step, float& m, float& l,
                   float4& o) {
    m = -CUDART_INF_F;
    for (int p = p0 + lane * step; p < jn.count; p += 32 * step)
      m = fmaxf(m, parts.lse[share_part(jn, worker, p) * PR_ROWS + r]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    const float base = m == -CUDART_INF_F ? 0.f : m;
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int p = p0; p < jn.count; p += step) {
      const int64_t at = (int64_t)share_part(jn, worker, p) * PR_ROWS + r;
      const float c = exp2_mufu(parts.lse[at] - base);
      const float4 x = *reinterpret_cast<const float4*>(parts.o + at * PG_HD + lane * 4);
      l += c;
      o.x = fmaf(c, x.x, o.x);
      o.y = fmaf(c, x.y, o.y);
      o.z = fmaf(c, x.z, o.z);
      o.w = fmaf(c, x.w, o.w);
    }
  };
  auto write = [&](const ShareJoin& jn, int r, float m, float l, const float4& o) {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const int f = jn.f0 + r, i = f / group, h = jn.head * group + f - i * group;
    const int64_t row = (int64_t)jn.row0 + i;
    uint2 y;
    y.x = H::pack(o.x * inv, o.y * inv);
    y.y = H::pack(o.z * inv, o.w * inv);
    *reinterpret_cast<uint2*>(out + row * out_stride + (int64_t)h * PG_HD + lane * 4) = y;
    if (lse && lane == 0) lse[row * heads + h] = l == 0.f ? -CUDART_INF_F : m + log2f(l);
  };
  float m, l;
  float4 o;
  const int counts = lane < PR_WARPS ? parts.join[lane * gridDim.x + blockIdx.x].count : 0;
  const int mine = __shfl_sync(0xffffffffu, counts, warp);
  if (mine > 0 && mine <= FEW) {
    const int worker = warp * gridDim.x + blockIdx.x;
    const ShareJoin jn = parts.join[worker];
    for (int r = blockIdx.y; r < jn.rows; r += gridDim.y) {
      merge(jn, worker, r, 0, 1, m, l, o);
      write(jn, r, m, l, o);
    }
  }
  for (unsigned many = __ballot_sync(0xffffffffu, counts > FEW); many; many &= many - 1) {
    const int worker = (__ffs(many) - 1) * gridDim.x + blockIdx.x;
    const ShareJoin jn = parts.join[worker];
    for (int r = blockIdx.y; r < jn.rows; r += gridDim.y) {
      merge(jn, worker, r, warp, PR_WARPS, m, l, o);
      if (lane == 0) {
        sm_m[warp] = m;
        sm_l[warp] = l;
      }
      sm_o[warp][lane] = o;
      __syncthreads();
      if (warp == 0) {
        m = sm_m[0];
#pragma unroll
        for (int k = 1; k < PR_WARPS; ++k) m = fmaxf(m, sm_m[k]);
        const float base = m == -CUDART_INF_F ? 0.f : m;
        l = 0.f;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < PR_WARPS; ++k) {
          const float c = exp2_mufu(sm_m[k] - base);
          const float4 x = sm_o[k][lane];
          l = fmaf(c, sm_l[k], l);
          o.x = fmaf(c, x.x, o.x);
          o.y = fmaf(c, x.y, o.y);
          o.z = fmaf(c, x.z, o.z);
          o.w = fmaf(c, x.w, o.w);
        }
        write(jn, r, m, l, o);
      }
      __syncthreads();
    }
  }
}

// ------------------------------------------------------------------ attention weights
// w_k += sum_r 2^(s_rk - lse_r) over the rows that see slot k, for at most 16 query rows per key
// head (one tile, so a slot has one worker). The slots are the matrix instruction's rows here
// (S^T = K Q^T) and the query rows its columns, so a slot's sum stays in the lanes of a quad.
// The dot product may take the head's elements in any order: lane c of a quad takes the
// 16-byte pieces c, c + 4, ... of both operands, so a quad reads whole 64-byte runs and K goes
// to registers directly. Bound by the reads of K: a warp is a worker as in the attention
// kernel, with one block of 16 slots on its way while it works on another (K in registers: 128 of
// them, and a few spills). 16 x up to 4097 slots, 32 / 8 heads, f16, 83 MB: 19.1 us, 4.3 TB/s.
constexpr int PW_WARPS = 8;  // two CTAs per SM
struct PwShared {
  PrShares::Walk walk[PW_WARPS];
  ShareTable table;
};

template <typename T>
__global__ void __launch_bounds__(PW_WARPS * 32, 2)
    paged_weights_kernel(const PagedKV kv, const T* __restrict__ q, int64_t q_stride, int heads,
                         float scale_log2, const float* __restrict__ lse,
                         float* __restrict__ weights) {
  using H = Half16<T>;
  __shared__ PwShared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = heads / kv.kv_heads;
  PrShares::Walk& w = sh.walk[warp];
  if (!PrShares::begin(kv, group, sh.table, gridDim.x * PW_WARPS, warp * gridDim.x + blockIdx.x, w))
    return;
  __syncwarp();
  const int r0 = lane >> 2, c = lane & 3;
  const T* k_pool = static_cast<const T*>(kv.k);
  bool go_on;
  do {
    const PagedSeq seq = w.seq;
    const int b = w.b, head = w.head, rows = w.rows(group), j1 = w.j1;
    // Q: row lane / 4 of each half of the tile's rows; and of this lane's columns 2 c + e the
    // log-sum-exp and limit (no slot for the columns behind the last row)
    uint4 qf[2][4];
    float x[2][2];
    int lim[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int f = min(h * 8 + r0, rows - 1), i = f / group;
      const T* qp = q + (seq.row0 + i) * q_stride + (int64_t)(head * group + f - i * group) * PG_HD;
#pragma unroll
      for (int p = 0; p < 4; ++p) qf[h][p] = *reinterpret_cast<const uint4*>(qp + p * 32 + c * 8);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int fc = h * 8 + 2 * c + e, ic = min(fc, rows - 1) / group;
        const int g = min(fc, rows - 1) - ic * group;
        x[h][e] = -__ldg(lse + (int64_t)(seq.row0 + ic) * heads + head * group + g);
        lim[h][e] = fc < rows ? seq.limit(ic) : 0;
      }
    }
    // rows of the cache of the next 32 blocks, a lane each
    int first = w.j0, at = -1;
    auto look_up = [&]() {
      const int key = (first + lane) * PR_BLOCK;
      const int id = first + lane < j1 && key < seq.end ? kv.page_id(b, key) : -1;
      at = id >= 0 ? kv.page_row(id, head, key) : -1;
    };
    auto load = [&](int row, uint4 (&k)[2][4]) {
      if (row < 0) return;  // a page outside the pool
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int p = 0; p < 4; ++p)
          k[j][p] = *reinterpret_cast<const uint4*>(k_pool + (int64_t)(row + r0 + 8 * j) * PG_HD +
                                                    p * 32 + c * 8);
    };
    auto use = [&](int jb, int row, const uint4 (&k)[2][4]) {
      if (row < 0) return;
      const int key0 = jb * PR_BLOCK;
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h * 8 >= rows) break;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const uint32_t a0[4] = {k[0][p].x, k[1][p].x, k[0][p].y, k[1][p].y};
          const uint32_t a1[4] = {k[0][p].z, k[1][p].z, k[0][p].w, k[1][p].w};
          H::mma(s, a0, qf[h][p].x, qf[h][p].y);
          H::mma(s, a1, qf[h][p].z, qf[h][p].w);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (key0 + r0 + 8 * j < lim[h][e])
              sum[j] += exp2_mufu(fmaf(s[2 * j + e], scale_log2, x[h][e]));
      }
      sum[0] = quad_sum(sum[0]);
      sum[1] = quad_sum(sum[1]);
      const int mine = r0 + 8 * c;  // lanes c = 0, 1 write a slot each
      if (c < 2 && key0 + mine < seq.end) atomicAdd(weights + row + mine, c ? sum[1] : sum[0]);
    };
    uint4 ka[2][4], kb[2][4];
    look_up();
    int row_a = __shfl_sync(0xffffffffu, at, 0), row_b = -1;
    load(row_a, ka);
    for (int jb = first; jb < j1; jb += 2) {
      if (jb + 1 < j1) {
        if (jb + 1 - first >= 32) {
          first = jb + 1;
          look_up();
        }
        row_b = __shfl_sync(0xffffffffu, at, jb + 1 - first);
        load(row_b, kb);
      }
      use(jb, row_a, ka);
      if (jb + 1 < j1) {
        if (jb + 2 < j1) {
          if (jb + 2 - first >= 32) {
            first = jb + 2;
            look_up();
          }
          row_a = __shfl_sync(0xffffffffu, at, jb + 2 - first);
          load(row_a, ka);
        }
        use(jb + 1, row_b, kb);
      }
    }
    __syncwarp();
    go_on = false;
    if (lane == 0) go_on = w.next(kv, group);
    go_on = __any_sync(0xffffffffu, go_on);
  } while (go_on);
}

}  // namespace cb
