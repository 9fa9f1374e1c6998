// Attention weight that every slot of a paged cache got from a chunk of new tokens, on the
// 5th-generation tensor cores: w_k += sum_r 2^(s_rk - lse_r), for many query rows.
//
// The slots are the rows of the product (S^T = K Q^T): a thread owns one slot, reads the
// scores of all query rows of a step from its own TMEM lane and adds up, so the sum needs no
// exchange and its order is fixed. A CTA keeps the K of 512 slots of one key head (four tiles
// of 128, one warpgroup each) and walks the query rows in steps of whole tokens, at most 128
// rows: every Q step that is loaded serves all tiles, and while one tile's scores are made
// the other warpgroups add up theirs. 640 threads:
//   warp 0       TMA producer: K once, then the Q steps (two buffers)
//   warp 1       TMEM owner; issues S^T (128 x 128 x 128), one buffer per tile
//   warps 2, 3   copy the steps' log-sum-exps and limits to shared memory
//   warps 4-19   the sums
// The exponentials are the bound (half of the flops of an attention, as many exponentials):
// 16 a clock and SM, 4096 cycles per 512 slots and 128 rows against the products' 2048, so a
// quarter of them goes to the FMA pipes. (Two tiles a CTA with two buffers each left two warps
// per scheduler and took 1.4 times as long; steps of 64 rows with two CTAs an SM likewise: a
// step costs a warp some 60 instructions whatever its rows.)
// 3 chunks of up to 1024 on 8192 slots, 32 / 8 heads, bf16: 151 us, 0.71 PFLOP/s. A step of 512
// slots and 128 rows takes 2.6 us, about 4800 cycles: 3100 of MUFU, 2900 issue slots of each
// scheduler, 2048 of products, which its four warps of sums overlap only in part; and 296 CTAs of
// unequal length on 148 SMs leave a tail of 12 %.
#pragma once
#include "paged_attention_tc.cuh"

namespace cb {

constexpr int WT_TILES = 4;
constexpr int WT_KEYS = WT_TILES * 128;  // slots of a CTA
constexpr int WT_ROWS = 128;        // query rows of a step, at most
constexpr int WT_THREADS = 640;
constexpr int WT_Q_BUFS = 2;
constexpr int WT_Q_BYTES = WT_ROWS * PG_HD * 2;
constexpr int WT_L_BUFS = 4;
constexpr int WT_K_OFF = 0;         // [tile][half of the head][128 slots][128 B]
constexpr int WT_Q_OFF = WT_TILES * 32768;  // [buffer][half][128 rows][128 B]
constexpr int WT_L_OFF = WT_Q_OFF + WT_Q_BUFS * WT_Q_BYTES;  // [buffer]: -lse [128], limit [128]
constexpr int WT_BAR_OFF = WT_L_OFF + WT_L_BUFS * WT_ROWS * 8;
constexpr int WT_SMEM = WT_BAR_OFF + 256 + 1024;
constexpr uint32_t WT_TMEM_COLS = 512;  // 128 columns per tile

// 3-D tiled TMA load without a cache hint.
__device__ __forceinline__ void tma_load_3d_plain(void* smem_dst, const CUtensorMap* map,
                                                  uint64_t* bar, int32_t c0, int32_t c1,
                                                  int32_t c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// Grid: ((sequence * blocks of WT_KEYS slots) + block) * kv_heads + key head. tmQ: q as
// [rows][heads][128] in boxes of step_tokens x group x 64.
template <typename T, bool LOADS>
__global__ void __launch_bounds__(WT_THREADS, 1)
    paged_weights_tile_kernel(const __grid_constant__ CUtensorMap tmK,
                              const __grid_constant__ CUtensorMap tmQ, const PagedKV kv, int heads,
                              float scale_log2, const float* __restrict__ lse,
                              float* __restrict__ weights, int blocks, int box_rows,
                              int step_tokens) {
  extern __shared__ uint8_t wt_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(wt_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + WT_BAR_OFF);
  uint64_t* k_full = bars;
  uint64_t* q_full = bars + 1;    // [2]
  uint64_t* q_empty = bars + 3;   // [2]
  uint64_t* l_full = bars + 5;    // [4]
  uint64_t* l_empty = bars + 9;   // [4]
  uint64_t* s_full = bars + 13;   // [tile]
  uint64_t* s_empty = bars + 17;  // [tile]
  uint64_t* drain = bars + 21;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 24);
  int* failed = reinterpret_cast<int*>(bars + 25);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = heads / kv.kv_heads;
  const int head = blockIdx.x % kv.kv_heads;
  const int rest = blockIdx.x / kv.kv_heads;
  const int b = rest / blocks;
  const int key0 = (rest % blocks) * WT_KEYS;
  const PagedSeq seq = paged_seq(kv, b);
  if (seq.n == 0 || key0 >= seq.limit(seq.n - 1)) return;  // no query sees these slots
  const int tiles = min(WT_TILES, (seq.limit(seq.n - 1) - key0 + 127) / 128);
  const int i0 = max(0, key0 - seq.past);  // the first token that sees one of them
  const int steps = (seq.n - i0 + step_tokens - 1) / step_tokens;
  const int step_rows = step_tokens * group;

  if (threadIdx.x == 0) {
    mbar_init(k_full, 1);
    for (int i = 0; i < WT_Q_BUFS; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < WT_L_BUFS; ++i) {
      mbar_init(&l_full[i], 1);
      mbar_init(&l_empty[i], 4 * tiles);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 4);
    }
    mbar_init(drain, 1);
    *failed = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmQ);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, WT_TMEM_COLS);
    tmem_relinquish();
  }
  // Rows behind a step's (where 128 is no multiple of the group) are 0 and count with a
  // log-sum-exp of infinity, weight 0. (The masks count for them all the same: 0 times a key's
  // infinity is NaN. 3 x 1024 on 8192 slots, 8 key heads of 5 and 7: 367 and 502 us, without
  // these masks 356 and 486.)
  for (int i = threadIdx.x; i < WT_Q_BUFS * 2 * (WT_ROWS - step_rows) * 8; i += WT_THREADS) {
    const int half = i / ((WT_ROWS - step_rows) * 8), in_half = i - half * (WT_ROWS - step_rows) * 8;
    *reinterpret_cast<uint4*>(smem + WT_Q_OFF + half * (WT_Q_BYTES / 2) + step_rows * 128 +
                              in_half * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ---------------- producer
    if (LOADS && lane == 0) mbar_arrive_expect_tx(k_full, 32768 * tiles);
    __syncwarp();
    for (int s = 0; LOADS && s < tiles; ++s) {
      const int k = key0 + s * 128;
      const int id = pt_step_id<128>(kv, b, k, seq.end, box_rows, lane);
      const int part = lane >> 1, half = lane & 1;
      if (part * box_rows < 128) {
        const int row = id >= 0 ? kv.page_row(id, head, k + part * box_rows) : kv.cache_rows();
        tma_load_2d(smem + WT_K_OFF + s * 32768 + half * 16384 + part * box_rows * 128, &tmK, k_full,
                    half * 64, row);
      }
    }
    if (LOADS && lane == 0) {
      int j = 0;
      for (; j < steps; ++j) {
        const int buf = j % WT_Q_BUFS;
        if (!paged_wait<LOADS>(&q_empty[buf], ((j / WT_Q_BUFS) & 1) ^ 1u, failed)) break;
        uint8_t* dst = smem + WT_Q_OFF + buf * WT_Q_BYTES;
        const int row = seq.row0 + i0 + j * step_tokens;
        mbar_arrive_expect_tx(&q_full[buf], step_rows * 256);
        tma_load_3d_plain(dst, &tmQ, &q_full[buf], 0, head * group, row);
        tma_load_3d_plain(dst + WT_Q_BYTES / 2, &tmQ, &q_full[buf], 64, head * group, row);
      }
      // what is still on its way (in a CTA that ends as it should it has been used by then)
      paged_drain<LOADS>(k_full, 0);
      for (int x = max(0, j - WT_Q_BUFS); x < j; ++x)
        paged_drain<LOADS>(&q_full[x % WT_Q_BUFS], (x / WT_Q_BUFS) & 1);
    }
  } else if (warp == 1) {
    // ---------------- matrix instructions
    constexpr uint32_t idesc = pt_idesc<T>(WT_ROWS, false);
    const uint32_t leader = pt_elect();
    const uint32_t t0 = __shfl_sync(0xffffffffu, tmem, 0);
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
      const bool there = __all_sync(0xffffffffu, paged_wait<LOADS>(bar, parity, failed));
      tc_fence_after();
      return there;
    };
    const uint32_t k_desc = pt_desc_k(smem_u32(smem + WT_K_OFF));
    const uint32_t q_desc = pt_desc_k(smem_u32(smem + WT_Q_OFF));
    bool ok = wait(k_full, 0);
    for (int j = 0; ok && j < steps; ++j) {
      const int buf = j % WT_Q_BUFS;
      if (!(ok = wait(&q_full[buf], (j / WT_Q_BUFS) & 1))) break;
      for (int s = 0; ok && s < tiles; ++s) {
        if (!(ok = wait(&s_empty[s], (j & 1) ^ 1u))) break;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t k_off = s * (32768 >> 4) + (k >> 2) * (16384 >> 4) + (k & 3) * 2;
          const uint32_t q_off = buf * (WT_Q_BYTES >> 4) + (k >> 2) * (WT_Q_BYTES >> 5) + (k & 3) * 2;
          pt_mma_ss(leader, t0 + s * 128, k_desc + k_off, q_desc + q_off, idesc,
                    k != 0);
        }
        pt_commit(leader, &s_full[s]);
      }
      pt_commit(leader, &q_empty[buf]);
    }
    pt_commit(leader, drain);
    paged_drain<LOADS>(drain, 0);
  } else if (warp < 4) {
    // ---------------- log-sum-exps and limits of the steps' rows: a warp takes every other
    // step and loads its next one before it waits for the buffer (one step after another,
    // the loads' latency was the kernel's pace)
    float x[4];
    int lim[4];
    auto load = [&](int j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = lane + 32 * e;
        const int tok = c / group, i = i0 + j * step_tokens + tok;
        const bool valid = c < step_rows && i < seq.n;
        x[e] = valid ? -__ldg(lse + (int64_t)(seq.row0 + i) * heads + head * group + c - tok * group)
                     : -CUDART_INF_F;
        lim[e] = valid ? seq.limit(i) : 0;
      }
    };
    if (warp - 2 < steps) load(warp - 2);
    for (int j = warp - 2; j < steps; j += 2) {
      const int buf = j % WT_L_BUFS;
      float y[4];
      int lm[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = x[e];
        lm[e] = lim[e];
      }
      if (j + 2 < steps) load(j + 2);
      if (!__all_sync(0xffffffffu, paged_wait<LOADS>(&l_empty[buf], ((j / WT_L_BUFS) & 1) ^ 1u,
                                                     failed)))
        break;
      float* dst = reinterpret_cast<float*>(smem + WT_L_OFF + buf * WT_ROWS * 8);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        dst[lane + 32 * e] = y[e];
        reinterpret_cast<int*>(dst)[WT_ROWS + lane + 32 * e] = lm[e];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&l_full[buf]);
    }
  } else if (warp >= 4 && (warp - 4) >> 2 < tiles) {
    // ---------------- sums: thread = slot
    const int s = (warp - 4) >> 2, quad = warp & 3;
    const int key = key0 + s * 128 + quad * 32 + lane;
    const uint32_t t_s = tmem + s * 128 + ((uint32_t)(quad * 32) << 16);
    const float2 sc2 = make_float2(scale_log2, scale_log2);
    float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    bool ok = true;
    for (int j = 0; j < steps; ++j) {
      const int buf = j % WT_L_BUFS;
      const int first = i0 + j * step_tokens;
      // whole steps whose rows all see the tile's slots need no masks, in 32 rows without padding
      const bool whole = first + step_tokens <= seq.n && key0 + s * 128 + 128 <= seq.limit(first);
      const int unmasked = whole ? step_rows / 32 : 0;
      const float4* nl = reinterpret_cast<const float4*>(smem + WT_L_OFF + buf * WT_ROWS * 8);
      const int4* lim = reinterpret_cast<const int4*>(nl + WT_ROWS / 4);
      ok = __all_sync(0xffffffffu, paged_wait<LOADS>(&l_full[buf], (j / WT_L_BUFS) & 1, failed) &&
                                       paged_wait<LOADS>(&s_full[s], j & 1, failed));
      if (!ok) break;
      tc_fence_after();
      uint32_t u[2][32];  // 32 query rows at a time, the next ones on their way
      tmem_ld_32x32b_x32(t_s, u[0]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t(&w)[32] = u[c & 1];
        tmem_ld_wait_regs(u[c & 1]);
        if (c < 3) {
          tmem_ld_32x32b_x32(t_s + (c + 1) * 32, u[(c + 1) & 1]);
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[s]);
        }
        if (c < unmasked) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 y = nl[c * 8 + e / 4];
            float2 a = ffma2(make_float2(__uint_as_float(w[e]), __uint_as_float(w[e + 1])), sc2,
                             make_float2(y.x, y.y));
            float2 d = ffma2(make_float2(__uint_as_float(w[e + 2]), __uint_as_float(w[e + 3])), sc2,
                             make_float2(y.z, y.w));
            a.x = exp2_mufu(a.x);
            a.y = exp2_mufu(a.y);
            if (e % 8 == 0) {  // a quarter of the exponentials on the FMA pipes
              d = exp2_poly2(d);
            } else {
              d.x = exp2_mufu(d.x);
              d.y = exp2_mufu(d.y);
            }
            acc[0] = fadd2(acc[0], a);
            acc[1] = fadd2(acc[1], d);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 y = nl[c * 8 + e / 4];
            const int4 m = lim[c * 8 + e / 4];
            acc[0].x += key < m.x ? exp2_mufu(fmaf(__uint_as_float(w[e]), scale_log2, y.x)) : 0.f;
            acc[0].y += key < m.y ? exp2_mufu(fmaf(__uint_as_float(w[e + 1]), scale_log2, y.y)) : 0.f;
            acc[1].x += key < m.z ? exp2_mufu(fmaf(__uint_as_float(w[e + 2]), scale_log2, y.z)) : 0.f;
            acc[1].y += key < m.w ? exp2_mufu(fmaf(__uint_as_float(w[e + 3]), scale_log2, y.w)) : 0.f;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&l_empty[buf]);
    }
    if (!ok) acc[0].x = CUDART_NAN_F;  // a wait ran out
    if (key < seq.limit(seq.n - 1)) {
      const int id = kv.page_id(b, key);
      if (id >= 0)
        atomicAdd(weights + kv.page_row(id, head, key),
                  (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *failed != 0) paged_report_timeout();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, WT_TMEM_COLS);
  }
}

}  // namespace cb
