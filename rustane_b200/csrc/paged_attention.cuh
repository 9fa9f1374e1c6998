// Attention of new tokens over a paged cache, for few query rows per key head (a decode
// step), and the attention weight that every slot got from a step.
//
// The query rows of one key head in one sequence, n tokens x `group` heads (row f = token
// f / group, head f % group), are cut into tiles of 16: the m16n8k16 matrix instruction's
// rows. Per tile
//   s_rk = scale log2(e) q_r . k_k,  m = max_k s, l = sum_k 2^(s - m),
//   o_r = sum_k 2^(s_rk - m) v_k / l
// with the running maximum and sum (32 bits) of an online softmax. K and V are read once per
// 16 rows, so for a decode step the kernel is bound by the reads of the cache.
#pragma once
#include "paged_common.cuh"

namespace cb {

constexpr int PR_ROWS = 16;    // query rows of a tile
constexpr int PR_WARPS = 4;
constexpr int PR_STAGES = 3;   // blocks of 16 keys in flight per warp
constexpr int PR_BLOCK = 16;   // keys of a block
constexpr int PR_STAGE_BYTES = 2 * PR_BLOCK * PG_HD * 2;  // K and V
constexpr int PR_RING = PR_WARPS * PR_STAGES * PR_STAGE_BYTES;
constexpr int PR_SMEM = PR_RING + 256 + 1024;

// Where the parts of a split row go: part (row * heads + head) * splits + split.
struct PagedParts {
  float* o;    // [rows * heads * splits][128] normalised within the part
  float* lse;  // [rows * heads * splits] base-2 log-sum-exp of the part
  int splits;
  int keys;    // keys of a split, a multiple of 16
};

// Sum over the four lanes of a quad (the columns of an accumulator row).
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}

// Grid: ((tile * kv_heads) + key head) * splits + split. Each warp takes every fourth block
// of 16 keys of the CTA's part through a ring of its own, filled by TMA (128-byte swizzle,
// so the ldmatrix reads of eight rows meet no bank twice); the warps' results are joined in
// shared memory. With several splits the parts are joined by paged_combine_kernel.
template <typename T>
__global__ void __launch_bounds__(PR_WARPS * 32, 2)
    paged_rows_kernel(const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const PagedKV kv,
                      const T* __restrict__ q, int64_t q_stride, int heads, float scale_log2,
                      T* __restrict__ out, int64_t out_stride, float* __restrict__ lse,
                      const PagedParts parts) {
  using H = Half16<T>;
  extern __shared__ uint8_t pr_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(pr_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + PR_RING);
  __shared__ int failed;
  __shared__ float sm_m[PR_WARPS][PR_ROWS], sm_l[PR_WARPS][PR_ROWS];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = heads / kv.kv_heads;
  const int split = blockIdx.x % parts.splits;
  const int rest = blockIdx.x / parts.splits;
  const int head = rest % kv.kv_heads;
  const PagedTile t = paged_find_tile<PR_ROWS>(kv, group, rest / kv.kv_heads);
  if (t.b < 0) return;
  const PagedSeq seq = t.seq;
  const int f0 = t.tile * PR_ROWS;
  const int rows = min(PR_ROWS, seq.n * group - f0);
  const int tile_end = max(0, seq.limit((f0 + rows - 1) / group));  // slots that any row sees
  const int k0 = split * parts.keys;
  const int k1 = min(tile_end, k0 + parts.keys);
  if (split > 0 && k0 >= k1) return;  // a part that the join does not ask for

  if (threadIdx.x == 0) {
    failed = 0;
    for (int i = 0; i < PR_WARPS * PR_STAGES; ++i) mbar_init(&bars[i], 1);
    fence_mbar_init();
  }
  __syncthreads();

  const int blocks = (max(0, k1 - k0) + PR_BLOCK - 1) / PR_BLOCK;
  const int mine = blocks > warp ? (blocks - warp + PR_WARPS - 1) / PR_WARPS : 0;
  uint8_t* ring = smem + warp * PR_STAGES * PR_STAGE_BYTES;
  uint64_t* full = bars + warp * PR_STAGES;
  auto key_of = [&](int i) { return k0 + (warp + i * PR_WARPS) * PR_BLOCK; };
  auto id_of = [&](int i) { return i < mine ? kv.page_id(t.b, key_of(i)) : -1; };
  auto load = [&](int i, int id) {
    if (lane == 0) {
      const int stage = i % PR_STAGES;
      // rows behind the matrix read as zero (a page outside the pool)
      const int row = id >= 0 ? kv.page_row(id, head, key_of(i)) : kv.cache_rows();
      uint8_t* dst = ring + stage * PR_STAGE_BYTES;
      mbar_arrive_expect_tx(&full[stage], PR_STAGE_BYTES);
      tma_load_2d(dst, &tmK, &full[stage], 0, row);
      tma_load_2d(dst + 2048, &tmK, &full[stage], 64, row);
      tma_load_2d(dst + 4096, &tmV, &full[stage], 0, row);
      tma_load_2d(dst + 6144, &tmV, &full[stage], 64, row);
    }
  };
  // page ids of the next blocks: ids[0] of the block at hand, the last one is loaded one
  // step before it is needed
  int ids[PR_STAGES + 1];
#pragma unroll
  for (int i = 0; i <= PR_STAGES; ++i) ids[i] = id_of(i);
#pragma unroll
  for (int i = 0; i < PR_STAGES; ++i)
    if (i < mine) load(i, ids[i]);

  // Q fragments: rows lane / 4 and lane / 4 + 8, elements 2 (lane % 4) (+ 1, + 8, + 9)
  const int r0 = lane >> 2, c2 = (lane & 3) * 2;
  uint32_t qf[8][4];
  int lim[2];
  const T* qp[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = r0 + 8 * j;
    const int f = f0 + min(r, rows - 1);
    const int i = f / group;
    lim[j] = r < rows ? seq.limit(i) : 0;
    qp[j] = q + (int64_t)(seq.row0 + i) * q_stride + (int64_t)(head * group + f - i * group) * PG_HD;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
#pragma unroll
    for (int a = 0; a < 4; ++a)
      qf[k][a] = *reinterpret_cast<const uint32_t*>(qp[a & 1] + k * 16 + c2 + (a >> 1) * 8);
  }
  const int lim_min = seq.limit(f0 / group);

  float o[16][4];
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
  float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};

  for (int i = 0; i < mine; ++i) {
    const int stage = i % PR_STAGES;
    const int key0 = key_of(i);
    if (!mbar_wait(&full[stage], (i / PR_STAGES) & 1, &failed)) break;
    const uint32_t kb = smem_u32(ring + stage * PR_STAGE_BYTES), vb = kb + 4096;
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
    const bool all_seen = ids[0] >= 0 && key0 + PR_BLOCK <= lim_min;
    if (!all_seen) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (ids[0] < 0 || key0 + n * 8 + c2 + (j & 1) >= lim[j >> 1]) s[n][j] = -CUDART_INF_F;
    }
    float base[2], corr[2];
    bool grew = false;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float mx = quad_max(fmaxf(fmaxf(s[0][2 * j], s[0][2 * j + 1]),
                                      fmaxf(s[1][2 * j], s[1][2 * j + 1]))) * scale_log2;
      const float mn = fmaxf(m[j], mx);
      base[j] = mn == -CUDART_INF_F ? 0.f : mn;
      grew |= mn > m[j];
      corr[j] = exp2_mufu(m[j] - base[j]);  // 0 for a row that had seen nothing
      m[j] = mn;
    }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int j = 0; j < 2; ++j) l[j] *= corr[j];
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
      for (int j = 0; j < 4; ++j) {
        s[n][j] = exp2_mufu(fmaf(s[n][j], scale_log2, -base[j >> 1]));
        l[j >> 1] += s[n][j];
      }
    // P rounds to the cache's type (the matrix instruction takes one type for both sides):
    // at most half a step of each weight, the size of the output's own rounding.
    const uint32_t pf[4] = {H::pack(s[0][0], s[0][1]), H::pack(s[0][2], s[0][3]),
                            H::pack(s[1][0], s[1][1]), H::pack(s[1][2], s[1][3])};
    // slots behind the sequence may hold anything, and 0 x NaN is not 0: their V reads as 0
    uint32_t v_mask[2] = {0xffffffffu, 0xffffffffu};
    const bool v_whole = key0 + PR_BLOCK <= seq.end;
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
        for (int j = 0; j < 4; ++j) vf[j] &= v_mask[j & 1];
      }
      H::mma(o[2 * n], pf, vf[0], vf[1]);
      H::mma(o[2 * n + 1], pf, vf[2], vf[3]);
    }
    __syncwarp();  // every lane has read the stage
    if (i + PR_STAGES < mine) load(i + PR_STAGES, ids[PR_STAGES]);
#pragma unroll
    for (int j = 0; j < PR_STAGES; ++j) ids[j] = ids[j + 1];
    ids[PR_STAGES] = id_of(i + PR_STAGES + 1);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) l[j] = quad_sum(l[j]);

  // ---- join the warps: [warp][row][128] over the ring (whose last load has arrived)
  __syncthreads();
  float* sm_o = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = r0 + 8 * j;
    if ((lane & 3) == 0) {
      sm_m[warp][r] = m[j];
      sm_l[warp][r] = l[j];
    }
#pragma unroll
    for (int n = 0; n < 16; ++n)
      *reinterpret_cast<float2*>(sm_o + (warp * PR_ROWS + r) * PG_HD + n * 8 + c2) =
          make_float2(o[n][2 * j], o[n][2 * j + 1]);
  }
  __syncthreads();
  const int d = threadIdx.x;  // one thread per element
  for (int r = 0; r < rows; ++r) {
    float mx = sm_m[0][r];
#pragma unroll
    for (int w = 1; w < PR_WARPS; ++w) mx = fmaxf(mx, sm_m[w][r]);
    const float base = mx == -CUDART_INF_F ? 0.f : mx;
    float sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < PR_WARPS; ++w) {
      const float c = exp2_mufu(sm_m[w][r] - base);
      sum = fmaf(c, sm_l[w][r], sum);
      acc = fmaf(c, sm_o[(w * PR_ROWS + r) * PG_HD + d], acc);
    }
    const float res = sum == 0.f ? 0.f : acc / sum;  // a row that sees nothing: 0
    const float row_lse = sum == 0.f ? -CUDART_INF_F : mx + log2f(sum);
    const int f = f0 + r, i = f / group;
    const int64_t at = (int64_t)(seq.row0 + i);
    const int h = head * group + f - i * group;
    if (parts.splits == 1) {
      out[at * out_stride + (int64_t)h * PG_HD + d] = H::from(res);
      if (lse && d == 0) lse[at * heads + h] = row_lse;
    } else {
      const int64_t p = (at * heads + h) * parts.splits + split;
      parts.o[p * PG_HD + d] = res;
      if (d == 0) parts.lse[p] = row_lse;
    }
  }
}

// Joins the parts of every row: out = sum_s 2^(lse_s - lse) o_s, lse = log2 sum_s 2^lse_s.
// One warp per (row, head). A tile has as many parts as its last row's slots need.
constexpr int PC_WARPS = 4;
template <typename T>
__global__ void __launch_bounds__(PC_WARPS * 32)
    paged_combine_kernel(const PagedKV kv, int heads, const PagedParts parts,
                         T* __restrict__ out, int64_t out_stride, float* __restrict__ lse) {
  using H = Half16<T>;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * PC_WARPS + (threadIdx.x >> 5);
  if (w >= (int64_t)kv.rows * heads) return;
  const int r = (int)(w / heads), h = (int)(w - (int64_t)r * heads);
  int started = 0;
  for (int base = 0; base <= kv.batch; base += 32) {
    const bool before = base + lane <= kv.batch && __ldg(kv.row_start + base + lane) <= r;
    started += __popc(__ballot_sync(0xffffffffu, before));
  }
  const int b = started - 1;
  if (b < 0 || b >= kv.batch) return;  // padding
  const PagedSeq seq = paged_seq(kv, b);
  const int i = r - seq.row0;
  if (i < 0 || i >= seq.n) return;
  const int group = heads / kv.kv_heads;
  const int f = i * group + h % group;
  const int last = min((f / PR_ROWS + 1) * PR_ROWS, seq.n * group) - 1;
  const int tile_end = max(0, seq.limit(last / group));
  const int n = min(parts.splits, max(1, (tile_end + parts.keys - 1) / parts.keys));

  const float* pl = parts.lse + w * parts.splits;
  const float* po = parts.o + w * parts.splits * PG_HD + lane * 4;
  float mx = -CUDART_INF_F;
  for (int s = lane; s < n; s += 32) mx = fmaxf(mx, pl[s]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
  const float base = mx == -CUDART_INF_F ? 0.f : mx;
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < n; s0 += 32) {
    // max and sum both skip NaN of a maximum; a NaN part makes its weight and the row NaN
    const float mine = s0 + lane < n ? exp2_mufu(pl[s0 + lane] - base) : 0.f;
    const int m = min(32, n - s0);
#pragma unroll 4
    for (int s = 0; s < m; ++s) {
      const float c = __shfl_sync(0xffffffffu, mine, s);
      const float4 x = *reinterpret_cast<const float4*>(po + (int64_t)(s0 + s) * PG_HD);
      sum += c;
      acc.x = fmaf(c, x.x, acc.x);
      acc.y = fmaf(c, x.y, acc.y);
      acc.z = fmaf(c, x.z, acc.z);
      acc.w = fmaf(c, x.w, acc.w);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  uint2 w2;
  w2.x = H::pack(acc.x * inv, acc.y * inv);
  w2.y = H::pack(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(out + (int64_t)r * out_stride + (int64_t)h * PG_HD + lane * 4) = w2;
  if (lse && lane == 0) lse[w] = sum == 0.f ? -CUDART_INF_F : mx + log2f(sum);
}

// ------------------------------------------------------------------ attention weights
// w_k += sum_r 2^(s_rk - lse_r) over the rows that see slot k. The slots are the matrix
// instruction's rows here (S^T = K Q^T), so a slot's sum stays in the lanes of one quad. A
// warp keeps 16 slots' K in registers and walks the query rows eight at a time.
// The dot product may take the head's elements in any order: lane c of a quad takes the
// 16-byte pieces c, c + 4, ... of both operands, so a quad reads whole 64-byte runs and no
// shared memory is needed.
constexpr int PW_WARPS = 4;
constexpr int PW_KEYS = PW_WARPS * 16;  // slots of a CTA

// Grid: ((sequence * blocks of PW_KEYS slots) + block) * kv_heads + key head.
template <typename T>
__global__ void __launch_bounds__(PW_WARPS * 32)
    paged_weights_kernel(const PagedKV kv, const T* __restrict__ q, int64_t q_stride, int heads,
                         float scale_log2, const float* __restrict__ lse,
                         float* __restrict__ weights, int blocks) {
  using H = Half16<T>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = heads / kv.kv_heads;
  const int head = blockIdx.x % kv.kv_heads;
  const int rest = blockIdx.x / kv.kv_heads;
  const int b = rest / blocks;
  const PagedSeq seq = paged_seq(kv, b);
  const int key0 = (rest % blocks) * PW_KEYS + warp * 16;
  if (seq.n == 0 || key0 >= seq.end || key0 >= seq.limit(seq.n - 1)) return;
  const int id = kv.page_id(b, key0);  // a page holds whole blocks of 16
  if (id < 0) return;
  const int row = kv.page_row(id, head, key0);
  const int r0 = lane >> 2, c = lane & 3;

  uint4 kf[2][4];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int p = 0; p < 4; ++p)
      kf[j][p] = *reinterpret_cast<const uint4*>(
          static_cast<const T*>(kv.k) + (int64_t)(row + r0 + 8 * j) * PG_HD + p * 32 + c * 8);

  // the first token that sees key0; the ones before it add nothing
  const int i0 = max(0, key0 - seq.past);
  const int f_end = seq.n * group;
  float sum[2] = {0.f, 0.f};
  for (int f0 = i0 * group; f0 < f_end; f0 += 8) {
    const int f = min(f0 + r0, f_end - 1);
    const int i = f / group;
    const T* qp = q + (int64_t)(seq.row0 + i) * q_stride + (int64_t)(head * group + f - i * group) * PG_HD;
    uint4 qf[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) qf[p] = *reinterpret_cast<const uint4*>(qp + p * 32 + c * 8);
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t a0[4] = {kf[0][p].x, kf[1][p].x, kf[0][p].y, kf[1][p].y};
      const uint32_t a1[4] = {kf[0][p].z, kf[1][p].z, kf[0][p].w, kf[1][p].w};
      H::mma(s, a0, qf[p].x, qf[p].y);
      H::mma(s, a1, qf[p].z, qf[p].w);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {  // this lane's two query rows
      const int fq = f0 + 2 * c + j;
      if (fq < f_end) {
        const int iq = fq / group;
        const float x = __ldg(lse + (int64_t)(seq.row0 + iq) * heads + head * group + fq - iq * group);
        const int lim = seq.limit(iq);
        if (key0 + r0 < lim) sum[0] += exp2_mufu(fmaf(s[j], scale_log2, -x));
        if (key0 + r0 + 8 < lim) sum[1] += exp2_mufu(fmaf(s[2 + j], scale_log2, -x));
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    sum[j] = quad_sum(sum[j]);
    if (c == 0 && key0 + r0 + 8 * j < seq.end) atomicAdd(weights + row + r0 + 8 * j, sum[j]);
  }
}

}  // namespace cb
