// Attention of a chunk of new tokens over a paged cache on the 5th-generation tensor cores
// (tcgen05, TMEM): the mathematics of paged_attention.cuh for many query rows per key head.
//
// A CTA takes 256 query rows of one key head in one sequence as two tiles of 128 (A and B)
// and walks the keys in steps of 128. Both tiles use every K and V step that is loaded: with
// one tile per load the L2 would have to deliver a byte per 128 flops, 13 TB/s at the tensor
// cores' rate. 384 threads:
//   warp 0       TMA producer: K and V steps, two buffers each; a page of the step per lane
//                and half of the head (128-byte swizzle)
//   warp 1       TMEM owner (512 columns); lane 0 issues the matrix instructions:
//                  S = Q K^T  (128 x 128 x 128) and O += P V  (P read from TMEM)
//                in the order PV_A(j) S_A(j+1) PV_B(j) S_B(j+1): while one tile's products
//                run, the other tile's softmax does
//   warps 4-7    softmax of tile A, one thread per query row: 128 scores of a step in
//   warps 8-11   registers (tile B likewise), running maximum and sum in 32 bits, P written
//                over S. O in TMEM is rescaled only when the maximum has grown by 2^8 (P stays
//                below 2^8, which both types hold).
// A tile's S(j+1) is issued behind its PV(j), so "S(j+1) is full" also says that O may be
// rescaled and that P(j) is no longer read: no further barriers are needed.
#pragma once
#include "paged_attention.cuh"

namespace cb {

constexpr int PT_SUB = 128;            // rows of a tile
constexpr int PT_ROWS = 2 * PT_SUB;    // query rows of a CTA
constexpr int PT_KEYS = 128;           // keys of a step
constexpr int PT_THREADS = 384;
constexpr int PT_Q_OFF = 0;            // [tile][half of the head][128 rows][128 B]
constexpr int PT_K_OFF = 65536;        // [buffer][half][128 keys][128 B]
constexpr int PT_V_OFF = 131072;
constexpr int PT_BAR_OFF = 196608;
constexpr int PT_SMEM = PT_BAR_OFF + 256 + 1024;
constexpr uint32_t PT_TMEM_COLS = 512;  // S_A, S_B, O_A, O_B: 128 columns each
constexpr float PT_RESCALE = 8.0f;

template <typename T>
__device__ __forceinline__ constexpr uint32_t pt_idesc(bool b_mn) {
  // A and B formats: 0 = fp16, 1 = bf16
  const uint32_t fmt = sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? (1u << 7) | (1u << 10) : 0u;
  return (b_mn ? umma_idesc_f16_bmn(128, 128) : umma_idesc_f16(128, 128)) | fmt;
}

// Loads the Q rows f0 + r (r = 0 .. 127) of a key head into a K-major swizzled tile, one
// thread per row; rows behind the sequence's last are zero.
template <typename T>
__device__ __forceinline__ void pt_load_q(uint8_t* tile, const T* __restrict__ q, int64_t q_stride,
                                          const PagedSeq& seq, int head, int group, int f, int r) {
  const int i = f / group;
  uint4 x[16];
  if (i < seq.n) {
    const uint4* src = reinterpret_cast<const uint4*>(
        q + (int64_t)(seq.row0 + i) * q_stride + (int64_t)(head * group + f - i * group) * PG_HD);
#pragma unroll
    for (int c = 0; c < 16; ++c) x[c] = __ldg(src + c);
  } else {
#pragma unroll
    for (int c = 0; c < 16; ++c) x[c] = make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int c = 0; c < 16; ++c)
    *reinterpret_cast<uint4*>(tile + (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = x[c];
}

// Producer side of a step: the lanes of a warp load the pages of keys key0 .. key0 + 127 into
// a [half][128][128 B] buffer (box_rows keys each; absent pages and slots behind the table
// read as zero). id: the lane's page id of this step.
__device__ __forceinline__ void pt_load_step(const CUtensorMap* map, uint8_t* dst, uint64_t* bar,
                                             const PagedKV& kv, int head, int key0, int id,
                                             int box_rows, int lane) {
  if (lane == 0) mbar_arrive_expect_tx(bar, 32768);
  __syncwarp();
  const int part = lane >> 1, half = lane & 1;
  if (part * box_rows < PT_KEYS) {
    const int row = id >= 0 ? kv.page_row(id, head, key0 + part * box_rows) : kv.cache_rows();
    tma_load_2d(dst + half * 16384 + part * box_rows * 128, map, bar, half * 64, row);
  }
}
__device__ __forceinline__ int pt_step_id(const PagedKV& kv, int b, int key0, int end,
                                          int box_rows, int lane) {
  const int key = key0 + (lane >> 1) * box_rows;
  return (lane >> 1) * box_rows < PT_KEYS && key < end ? kv.page_id(b, key) : -1;
}

template <typename T>
__global__ void __launch_bounds__(PT_THREADS, 1)
    paged_tile_kernel(const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const PagedKV kv,
                      const T* __restrict__ q, int64_t q_stride, int heads, float scale_log2,
                      T* __restrict__ out, int64_t out_stride, float* __restrict__ lse,
                      const PagedParts parts, int box_rows) {
  using H = Half16<T>;
  extern __shared__ uint8_t pt_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(pt_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + PT_BAR_OFF);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;   // [2]
  uint64_t* k_empty = bars + 3;  // [2]
  uint64_t* v_full = bars + 5;   // [2]
  uint64_t* v_empty = bars + 7;  // [2]
  uint64_t* s_full = bars + 9;   // [2] tile A, tile B
  uint64_t* p_full = bars + 11;  // [2]
  uint64_t* o_full = bars + 13;  // [2]
  uint64_t* drain = bars + 15;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
  int* failed = reinterpret_cast<int*>(bars + 17);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = heads / kv.kv_heads;
  const int split = blockIdx.x % parts.splits;
  const int rest = blockIdx.x / parts.splits;
  const int head = rest % kv.kv_heads;
  const PagedTile t = paged_find_tile<PT_ROWS>(kv, group, rest / kv.kv_heads);
  if (t.b < 0) return;
  const PagedSeq seq = t.seq;
  const int f0 = t.tile * PT_ROWS;
  const int rows = min(PT_ROWS, seq.n * group - f0);
  const int k0 = split * parts.keys;
  // steps of each tile: up to the last slot that its last row sees
  int n_sub[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int last = min(rows, (s + 1) * PT_SUB) - 1;
    const int end = last < s * PT_SUB ? 0 : seq.limit((f0 + last) / group);
    n_sub[s] = (max(0, min(end - k0, parts.keys)) + PT_KEYS - 1) / PT_KEYS;
  }
  const int n = max(n_sub[0], n_sub[1]);
  if (split > 0 && n == 0) return;  // a part that the join does not ask for

  if (threadIdx.x == 0) {
    mbar_init(q_full, 8);
    mbar_init(drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    *failed = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, PT_TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ---------------- producer
    const int end = min(seq.end, k0 + n * PT_KEYS);
    int id = pt_step_id(kv, t.b, k0, end, box_rows, lane);
    for (int j = 0; j < n; ++j) {
      const int key0 = k0 + j * PT_KEYS, buf = j & 1;
      const uint32_t free_parity = ((j >> 1) & 1) ^ 1u;
      const int next = j + 1 < n ? pt_step_id(kv, t.b, key0 + PT_KEYS, end, box_rows, lane) : -1;
      if (!mbar_wait(&k_empty[buf], free_parity, failed)) break;
      pt_load_step(&tmK, smem + PT_K_OFF + buf * 32768, &k_full[buf], kv, head, key0, id, box_rows,
                   lane);
      if (!mbar_wait(&v_empty[buf], free_parity, failed)) break;
      pt_load_step(&tmV, smem + PT_V_OFF + buf * 32768, &v_full[buf], kv, head, key0, id, box_rows,
                   lane);
      id = next;
    }
  } else if (warp == 1) {
    if (lane == 0 && n > 0) {
      // ---------------- matrix instructions
      constexpr uint32_t idesc_s = pt_idesc<T>(false), idesc_pv = pt_idesc<T>(true);
      const uint32_t q_addr = smem_u32(smem + PT_Q_OFF);
      const uint32_t k_addr = smem_u32(smem + PT_K_OFF);
      const uint32_t v_addr = smem_u32(smem + PT_V_OFF);
      auto issue_s = [&](int s, int j) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {  // head dim in steps of 16
          const uint32_t off = (uint32_t)((k >> 2) * 16384 + (k & 3) * 32);
          umma_f16_ss(tmem + s * 128, sw128_kmajor_desc(q_addr + s * 32768 + off),
                      sw128_kmajor_desc(k_addr + (j & 1) * 32768 + off), idesc_s, k != 0);
        }
        umma_commit(&s_full[s]);
      };
      auto issue_pv = [&](int s, int j) {
#pragma unroll
        for (int k = 0; k < 8; ++k)  // keys in steps of 16 (8 packed columns of P)
          umma_f16_ts(tmem + 256 + s * 128, tmem + s * 128 + k * 8,
                      sw128_mnmajor_desc(v_addr + (j & 1) * 32768 + k * 2048, 16384), idesc_pv,
                      (j | k) != 0);
      };
      bool ok = mbar_wait(q_full, 0, failed) && mbar_wait(&k_full[0], 0, failed);
      tc_fence_after();
      if (ok) {
        for (int s = 0; s < 2; ++s)
          if (n_sub[s] > 0) issue_s(s, 0);
        umma_commit(&k_empty[0]);
      }
      for (int j = 0; ok && j < n; ++j) {
        const int buf = j & 1;
        bool k_ready = false;
        ok = mbar_wait(&v_full[buf], (j >> 1) & 1, failed);
        for (int s = 0; ok && s < 2; ++s) {
          if (j >= n_sub[s]) continue;
          if (!(ok = mbar_wait(&p_full[s], j & 1, failed))) break;
          tc_fence_after();
          issue_pv(s, j);
          if (s == 1 || j >= n_sub[1]) umma_commit(&v_empty[buf]);
          if (j + 1 < n_sub[s]) {
            if (!k_ready && !(ok = mbar_wait(&k_full[buf ^ 1], ((j + 1) >> 1) & 1, failed))) break;
            k_ready = true;
            tc_fence_after();
            issue_s(s, j + 1);
          } else {
            umma_commit(&o_full[s]);
          }
        }
        if (ok && j + 1 < n) umma_commit(&k_empty[buf ^ 1]);
      }
      umma_commit(drain);  // nothing is in flight when TMEM is given back
      mbar_wait(drain, 0, failed);
    }
  } else if (warp >= 4) {
    // ---------------- softmax: thread = query row r of tile s
    const int s = (warp - 4) >> 2, quad = warp & 3;
    const int r = quad * 32 + lane;
    const int f = f0 + s * PT_SUB + r;
    uint8_t* q_tile = smem + PT_Q_OFF + s * 32768;
    pt_load_q(q_tile, q, q_stride, seq, head, group, f, r);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);

    const int i = f / group;
    const bool valid = i < seq.n;
    const int lim = valid ? seq.limit(i) : 0;
    // every row of the tile sees the slots below this
    const int lim_all = s * PT_SUB + PT_SUB <= rows ? seq.limit((f0 + s * PT_SUB) / group) : 0;
    const int n_s = s == 0 ? n_sub[0] : n_sub[1];
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t t_s = tmem + s * 128 + lane_off, t_o = tmem + 256 + s * 128 + lane_off;
    float m = -CUDART_INF_F, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n_s; ++j) {
      const int key0 = k0 + j * PT_KEYS;
      // absent pages of this step, a bit per 16 keys
      bool gone = false;
      if (lane < PT_KEYS / 16 && key0 + lane * 16 < seq.end)
        gone = kv.page_id(t.b, key0 + lane * 16) < 0;
      const uint32_t absent = __ballot_sync(0xffffffffu, gone);
      if (!mbar_wait(&s_full[s], j & 1, failed)) { ok = false; break; }
      tc_fence_after();
      uint32_t u[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(t_s + c * 32, u[c]);
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_wait_regs(u[c]);
      if (absent || key0 + PT_KEYS > lim_all) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (key0 + c * 32 + e >= lim || (absent >> (c * 2 + e / 16) & 1u))
              u[c][e] = 0xff800000u;  // -inf
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx[c] = __uint_as_float(u[c][0]);
#pragma unroll
        for (int e = 1; e < 31; e += 2)
          mx[c] = fmax3(mx[c], __uint_as_float(u[c][e]), __uint_as_float(u[c][e + 1]));
        mx[c] = fmaxf(mx[c], __uint_as_float(u[c][31]));
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale_log2;
      float corr = 1.0f;
      bool need = false;
      if (j == 0) {
        m = top;
      } else if (top > m + PT_RESCALE) {  // also when nothing was seen so far (m = -inf)
        corr = exp2_mufu(m - top);
        m = top;
        l *= corr;
        need = true;
      }
      if (__any_sync(0xffffffffu, need)) {
#pragma unroll 1
        for (int c = 0; c < 8; ++c) {
          uint32_t o[16];
          tmem_ld_32x32b_x16(t_o + c * 16, o);
          tmem_ld_wait_regs16(o);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
          tmem_st_32x32b_x16(t_o + c * 16, o);
        }
      }
      const float base = m == -CUDART_INF_F ? 0.f : m;
      const float2 sc2 = make_float2(scale_log2, scale_log2), nb2 = make_float2(-base, -base);
      float2 sum[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        sum[c] = make_float2(0.f, 0.f);
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float2 x = ffma2(make_float2(__uint_as_float(u[c][2 * e]), __uint_as_float(u[c][2 * e + 1])),
                           sc2, nb2);
          x.x = exp2_mufu(x.x);
          x.y = exp2_mufu(x.y);
          sum[c] = fadd2(sum[c], x);
          // P rounds to the cache's type: at most half a step of each weight, the size of the
          // output's own rounding
          p[e] = H::pack(x.x, x.y);
        }
        tmem_st_32x32b_x16(t_s + c * 16, p);
      }
      sum[0] = fadd2(fadd2(sum[0], sum[1]), fadd2(sum[2], sum[3]));
      l += sum[0].x + sum[0].y;
      if (key0 + PT_KEYS > seq.end) {
        // slots behind the sequence may hold anything, and 0 x NaN is not 0: zero their V
        const int row0 = seq.end - key0;  // 1 .. 127
        if (!mbar_wait(&v_full[j & 1], (j >> 1) & 1, failed)) { ok = false; break; }
        uint8_t* v = smem + PT_V_OFF + (j & 1) * 32768;
        if (r >= row0) {
#pragma unroll
          for (int c = 0; c < 16; ++c)
            *reinterpret_cast<uint4*>(v + (c >> 3) * 16384 + r * 128 + (c & 7) * 16) =
                make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[s]);
    }
    // ---------------- the tile's output
    const int h = head * group + f - i * group;
    const int64_t row = (int64_t)seq.row0 + i;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const float row_lse = l == 0.f ? -CUDART_INF_F : m + log2f(l);
    if (ok && n_s > 0) ok = mbar_wait(&o_full[s], 0, failed);
    tc_fence_after();
    if (ok) {
      if (parts.splits > 1) {
        const int64_t part = (row * heads + h) * parts.splits + split;
        if (valid) parts.lse[part] = row_lse;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          if (n_s > 0) {
            tmem_ld_32x32b_x32(t_o + c * 32, o);
            tmem_ld_wait_regs(o);
          }
          if (valid) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
              if (n_s > 0 && l != 0.f)
                x = make_float4(__uint_as_float(o[4 * e]) * inv, __uint_as_float(o[4 * e + 1]) * inv,
                                __uint_as_float(o[4 * e + 2]) * inv,
                                __uint_as_float(o[4 * e + 3]) * inv);
              *reinterpret_cast<float4*>(parts.o + part * PG_HD + c * 32 + e * 4) = x;
            }
          }
        }
      } else {
        if (lse && valid) lse[row * heads + h] = row_lse;
        // through the Q tile (no S reads it any more), so that half a warp writes a whole row
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          if (n_s > 0) {
            tmem_ld_32x32b_x32(t_o + c * 32, o);
            tmem_ld_wait_regs(o);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (n_s > 0 && l != 0.f) {
              w.x = H::pack(__uint_as_float(o[8 * e]) * inv, __uint_as_float(o[8 * e + 1]) * inv);
              w.y = H::pack(__uint_as_float(o[8 * e + 2]) * inv, __uint_as_float(o[8 * e + 3]) * inv);
              w.z = H::pack(__uint_as_float(o[8 * e + 4]) * inv, __uint_as_float(o[8 * e + 5]) * inv);
              w.w = H::pack(__uint_as_float(o[8 * e + 6]) * inv, __uint_as_float(o[8 * e + 7]) * inv);
            }
            const int chunk = c * 4 + e;
            *reinterpret_cast<uint4*>(q_tile + (chunk >> 3) * 16384 + r * 128 +
                                      (((chunk & 7) ^ (r & 7)) << 4)) = w;
          }
        }
        __syncwarp();
        const int chunk = lane & 15;
        for (int rr = quad * 32 + (lane >> 4); rr < quad * 32 + 32; rr += 2) {
          const int ff = f0 + s * PT_SUB + rr, ii = ff / group;
          if (ii >= seq.n) break;
          const uint4 w = *reinterpret_cast<const uint4*>(
              q_tile + (chunk >> 3) * 16384 + rr * 128 + (((chunk & 7) ^ (rr & 7)) << 4));
          *reinterpret_cast<uint4*>(out + ((int64_t)seq.row0 + ii) * out_stride +
                                    (int64_t)(head * group + ff - ii * group) * PG_HD + chunk * 8) = w;
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, PT_TMEM_COLS);
  }
}

}  // namespace cb
