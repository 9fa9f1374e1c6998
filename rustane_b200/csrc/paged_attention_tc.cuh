// Attention of a chunk of new tokens over a paged cache on the 5th-generation tensor cores
// (tcgen05, TMEM): the mathematics of paged_attention.cuh for many query rows per key head.
//
// A CTA takes 256 query rows of one key head in one sequence as two tiles of 128 (A and B)
// and walks the keys in steps of 128. Both tiles use every K and V step that is loaded: with
// one tile per load the L2 would have to deliver a byte per 128 flops, 13 TB/s at the tensor
// cores' rate. 384 threads:
//   warp 0       TMA producer: K and V steps, two buffers each; a page of the step per lane
//                and half of the head (128-byte swizzle)
//   warp 1       TMEM owner (512 columns); issues the matrix instructions:
//                  S = Q K^T  (128 x 128 x 128) and O += P V  (P read from TMEM)
//                in the order PV_A(j) S_A(j+1) PV_B(j) S_B(j+1): while one tile's products
//                run, the other tile's softmax does. PV starts when the first 64 keys' P are
//                there, beside the exponentials of the others.
//   warps 4-7    softmax of tile A, one thread per query row: 128 scores of a step in
//   warps 8-11   registers (tile B likewise), running maximum and sum in 32 bits, P written
//                over S. O in TMEM is rescaled only when the maximum has grown by 2^8 (P stays
//                below 2^8, or in fp16, whose small weights are taken 2^7 up, below 2^15).
// A tile's S(j+1) is issued behind its PV(j), so "S(j+1) is full" also says that O may be
// rescaled and that P(j) is no longer read. Steps of 64 keys with two S buffers a tile, and
// two threads per row, hide the products' latency as well, but a step costs a warp some sixty
// instructions whatever its keys: both were slower. Where there are at most 128 rows, tile B
// rests: to give it the same rows and every other step won 3 % when tried and was not kept.
//
// Measured (bf16): 2 x 2048 new tokens on 16384 slots, 40 / 8 heads, 1.29 TFLOP: 1.18 to 1.31 ms
// on different GPUs, 980 to 1090 TFLOP/s at the power cap's 1.57 GHz. 8 chunks of up to 512 on
// 2048 (f16, 12 / 12 heads): 51.8 us; at most 16 steps a tile do not hide a tile's own cost (its
// Q, the pipeline's start, its output), and the join (alone and cold) takes 10 us.
//
// Infinities and NaN in V of slots that not every row sees are taken out and added afterwards to
// the rows that see them (see paged_attention.cuh).
//
// The work is handed out in equal shares (paged_shares.cuh), a share to a CTA; paged_join_kernel
// joins the tiles that are cut.
#pragma once
#include "paged_shares.cuh"

namespace cb {

constexpr int PT_SUB = 128;            // rows of a tile
constexpr int PT_ROWS = 2 * PT_SUB;    // query rows of a CTA
constexpr int PT_KEYS = 128;           // keys of a step
constexpr int PT_BUFS = 2;             // K steps, and V steps, in flight
constexpr int PT_STEP_BYTES = PT_KEYS * PG_HD * 2;
constexpr int PT_THREADS = 384;
constexpr int PT_Q_OFF = 0;            // [tile][half of the head][128 rows][128 B]
constexpr int PT_K_OFF = 65536;        // [buffer][half][128 keys][128 B]
constexpr int PT_V_OFF = PT_K_OFF + PT_BUFS * PT_STEP_BYTES;
constexpr int PT_BAR_OFF = PT_V_OFF + PT_BUFS * PT_STEP_BYTES;
constexpr int PT_SHARE_OFF = PT_BAR_OFF + 256;
constexpr int PT_SMEM = PT_SHARE_OFF + SHARE_CHUNK * 8 + 64 + PT_THREADS / 32 * 80 + 1024;
constexpr uint32_t PT_TMEM_COLS = 512;  // S_A, S_B, O_A, O_B: 128 columns each
constexpr float PT_RESCALE = 8.0f;
// Binary places that P is taken up: what PT_RESCALE leaves of the type's.
template <typename T>
constexpr float PT_UP = Half16<T>::P_UP > 0.0f ? Half16<T>::P_UP - PT_RESCALE : 0.0f;

template <typename T>
__device__ __forceinline__ constexpr uint32_t pt_idesc(int n, bool b_mn) {
  // A and B formats: 0 = fp16, 1 = bf16
  const uint32_t fmt = __is_same(T, __nv_bfloat16) ? (1u << 7) | (1u << 10) : 0u;
  return (b_mn ? umma_idesc_f16_bmn(128, n) : umma_idesc_f16(128, n)) | fmt;
}

// Matrix instructions are issued by a whole warp with one lane's predicate, not by a branch
// of one lane: the operands are warp-uniform then, and the descriptors (their low words;
// the high word is the same for all) move on by additions. From a one-lane branch an
// instruction took about 130 cycles to issue, twice its time in the tensor cores.
constexpr uint32_t PT_DESC_HI = 64u | (1u << 14) | (2u << 29);  // 1024-byte groups, 128-byte swizzle
__device__ __forceinline__ uint32_t pt_desc_k(uint32_t smem_addr) {  // K-major
  return ((smem_addr & 0x3FFFFu) >> 4) | (1u << 16);
}
__device__ __forceinline__ uint32_t pt_desc_mn(uint32_t smem_addr, uint32_t lbo_bytes) {
  return ((smem_addr & 0x3FFFFu) >> 4) | ((lbo_bytes >> 4) << 16);
}
__device__ __forceinline__ uint32_t pt_elect() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(is));
  return is;
}
__device__ __forceinline__ void pt_mma_ss(uint32_t leader, uint32_t d, uint32_t a_lo, uint32_t b_lo,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 a, {%2, %4};\n\tmov.b64 b, {%3, %4};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], a, b, %5, p;\n\t}" ::"r"(leader),
      "r"(d), "r"(a_lo), "r"(b_lo), "r"(PT_DESC_HI), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void pt_mma_ts(uint32_t leader, uint32_t d, uint32_t a_tmem,
                                          uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 b, {%3, %4};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], b, %5, p;\n\t}" ::"r"(leader),
      "r"(d), "r"(a_tmem), "r"(b_lo), "r"(PT_DESC_HI), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void pt_commit(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}" ::"r"(
          leader),
      "r"(smem_u32(bar))
      : "memory");
}

// Loads a warp's 32 query rows f0 + r (r = first .. first + 31) of a key head into a K-major
// swizzled tile; rows behind the sequence's last are zero. Half a warp takes a row, so a load
// meets whole lines.
template <typename T>
__device__ __forceinline__ void pt_load_q(uint8_t* tile, const T* __restrict__ q, int64_t q_stride,
                                          const PagedSeq& seq, int head, int group, int f0,
                                          int first, int lane) {
  const int c = lane & 15;
  int r = first + (lane >> 4);
  int i = (f0 + r) / group, g = f0 + r - i * group;
#pragma unroll 2
  for (int it = 0; it < 16; ++it) {
    uint8_t* dst = tile + (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
    if (i < seq.n)
      cp_async_16(smem_u32(dst), q + (int64_t)(seq.row0 + i) * q_stride +
                                     (int64_t)(head * group + g) * PG_HD + c * 8);
    else
      *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
    r += 2;
    g += 2;
    while (g >= group) {  // two rows on
      g -= group;
      ++i;
    }
  }
  cp_async_commit();
  cp_async_wait<0>();
}

// Producer side of a step: the lanes of a warp load the pages of KEYS keys from key0 on into
// a [half][KEYS][128 B] buffer (box_rows keys each; absent pages and slots behind the table
// read as zero). id: the lane's page id of this step.
template <int KEYS>
__device__ __forceinline__ void pt_load_step(const CUtensorMap* map, uint8_t* dst, uint64_t* bar,
                                             const PagedKV& kv, int head, int key0, int id,
                                             int box_rows, int lane) {
  if (lane == 0) mbar_arrive_expect_tx(bar, KEYS * 256);
  __syncwarp();
  const int part = lane >> 1, half = lane & 1;
  if (part * box_rows < KEYS) {
    const int row = id >= 0 ? kv.page_row(id, head, key0 + part * box_rows) : kv.cache_rows();
    tma_load_2d(dst + half * KEYS * 128 + part * box_rows * 128, map, bar, half * 64, row);
  }
}
template <int KEYS>
__device__ __forceinline__ int pt_step_id(const PagedKV& kv, int b, int key0, int end,
                                          int box_rows, int lane) {
  const int key = key0 + (lane >> 1) * box_rows;
  return (lane >> 1) * box_rows < KEYS && key < end ? kv.page_id(b, key) : -1;
}

// A tile counts three steps for its Q, its pipeline's start and its output (ragged prompts: 58.6
// us with two, 51.6 with three, 53.8 with four).
using PtShares = PagedShares<PT_ROWS, PT_KEYS, 3, 5>;

struct PtShared {  // at PT_SHARE_OFF
  PtShares::Walk walk[PT_THREADS / 32];  // every warp's (registers are for the scores)
  ShareTable table;
};
static_assert(sizeof(PtShared) <= PT_SMEM - 1024 - PT_SHARE_OFF, "shared memory");

// Parts: o [2 gridDim][128][256 rows], lse [2 gridDim][256].
template <typename T, bool LOADS>
__global__ void __launch_bounds__(PT_THREADS, 1)
    paged_tile_kernel(const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const PagedKV kv,
                      const T* __restrict__ q, int64_t q_stride, int heads, float scale_log2,
                      T* __restrict__ out, int64_t out_stride, float* __restrict__ lse,
                      const ShareParts parts, int box_rows) {
  using H = Half16<T>;
  extern __shared__ uint8_t pt_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(pt_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + PT_BAR_OFF);
  PtShared& sh = *reinterpret_cast<PtShared*>(smem + PT_SHARE_OFF);
  uint64_t* k_full = bars;        // [2]
  uint64_t* k_empty = bars + 2;   // [2]
  uint64_t* v_full = bars + 4;    // [2]
  uint64_t* v_empty = bars + 6;   // [2]
  uint64_t* s_full = bars + 8;    // [tile]
  uint64_t* p_full = bars + 10;   // [tile][first, last 64 keys]
  uint64_t* o_full = bars + 14;   // [tile]
  uint64_t* q_full = bars + 16;
  uint64_t* drain = bars + 17;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 18);
  int* failed = reinterpret_cast<int*>(bars + 19);
  uint32_t* absent_of = reinterpret_cast<uint32_t*>(bars + 20);  // [4] absent pages of a step
  volatile uint32_t* odd_v = absent_of + 4;  // infinities or NaN were taken out of V

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = heads / kv.kv_heads;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 8);
    mbar_init(drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&o_full[i], 1);
    }
    *failed = 0;
    *odd_v = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  PtShares::Walk& w = sh.walk[warp];
  pdl_launch_dependents();  // (the join; it waits for this kernel's end)
  const bool some_work = PtShares::begin(kv, group, sh.table, gridDim.x, blockIdx.x, w);
  if (threadIdx.x == 0) parts.join[blockIdx.x].count = 0;  // (set below where a tile goes on)
  if (!some_work) return;
  if (warp == 1) {
    tmem_alloc(tmem_slot, PT_TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  auto next_segment = [&]() -> bool {  // the whole warp
    __syncwarp();
    bool more = false;
    if (lane == 0) more = w.next(kv, group);
    return __any_sync(0xffffffffu, more);
  };
  // steps of the segment's two tiles, from j0 on
  auto sub_steps = [&](int s) {
    const int f = w.tile * PT_ROWS + s * PT_SUB, rows = w.seq.n * group;
    if (f >= rows) return 0;
    const int end = w.seq.limit((min(f + PT_SUB, rows) - 1) / group);
    // the tile whose rows see nothing keeps the one step it has
    const int n = max(w.steps == 1 ? 1 : 0, (end + PT_KEYS - 1) / PT_KEYS);
    return max(0, min(n, w.j1) - w.j0);
  };

  // 128 x 72 + 256 x 216 registers of the 384 x 168 that the block was launched with
  if (warp < 4) {
    regs_dec<72>();
    if (warp == 0) {
      // ---------------- producer
      uint32_t g = 0;               // steps loaded
      uint32_t k_of = 0, v_of = 0;  // of K and of V
      bool ok = LOADS;
      if (LOADS) do {
        const int n = w.j1 - w.j0;
        const int b = w.b, head = w.head, end = w.seq.end, first = w.j0 * PT_KEYS;
        int id = pt_step_id<PT_KEYS>(kv, b, first, end, box_rows, lane);
        for (int j = 0; ok && j < n; ++j, ++g) {
          const int key0 = first + j * PT_KEYS, buf = g % PT_BUFS;
          const uint32_t free_parity = ((g / PT_BUFS) & 1) ^ 1u;
          const int next =
              j + 1 < n ? pt_step_id<PT_KEYS>(kv, b, key0 + PT_KEYS, end, box_rows, lane) : -1;
          // absent pages, a bit per 16 keys. (Four steps' words are kept: a step's is written
          // when S of two steps before is done, which the softmax of the one four before
          // precedes.)
          const int part = lane >> 1;
          const bool gone = (lane & 1) == 0 && part * box_rows < PT_KEYS &&
                            key0 + part * box_rows < end && id < 0;
          uint32_t absent = 0;
          for (uint32_t parts_gone = __ballot_sync(0xffffffffu, gone); parts_gone;
               parts_gone &= parts_gone - 1)
            absent |= ((1u << (box_rows / 16)) - 1) << ((__ffs(parts_gone) - 1) / 2 * (box_rows / 16));
          ok = __all_sync(0xffffffffu, paged_wait<LOADS>(&k_empty[buf], free_parity, failed));
          if (!ok) break;
          if (lane == 0) absent_of[g & 3] = absent;
          pt_load_step<PT_KEYS>(&tmK, smem + PT_K_OFF + buf * PT_STEP_BYTES, &k_full[buf], kv, head,
                                key0, id, box_rows, lane);
          k_of = g + 1;
          ok = __all_sync(0xffffffffu, paged_wait<LOADS>(&v_empty[buf], free_parity, failed));
          if (!ok) break;
          pt_load_step<PT_KEYS>(&tmV, smem + PT_V_OFF + buf * PT_STEP_BYTES, &v_full[buf], kv, head,
                                key0, id, box_rows, lane);
          v_of = g + 1;
          id = next;
        }
      } while (ok && next_segment());
      // the last steps' loads (of a CTA that ends as it should they have long been used)
      for (uint32_t x = k_of < PT_BUFS ? 0 : k_of - PT_BUFS; x < k_of; ++x)
        paged_drain<LOADS>(&k_full[x % PT_BUFS], (x / PT_BUFS) & 1);
      for (uint32_t x = v_of < PT_BUFS ? 0 : v_of - PT_BUFS; x < v_of; ++x)
        paged_drain<LOADS>(&v_full[x % PT_BUFS], (x / PT_BUFS) & 1);
    } else if (warp == 1) {
      // ---------------- matrix instructions
      constexpr uint32_t idesc_s = pt_idesc<T>(PT_KEYS, false), idesc_pv = pt_idesc<T>(128, true);
      const uint32_t leader = pt_elect();
      const uint32_t t0 = __shfl_sync(0xffffffffu, tmem, 0);
      auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        const bool there = __all_sync(0xffffffffu, paged_wait<LOADS>(bar, parity, failed));
        tc_fence_after();
        return there;
      };
      const uint32_t q_desc = pt_desc_k(smem_u32(smem + PT_Q_OFF));
      const uint32_t k_desc = pt_desc_k(smem_u32(smem + PT_K_OFF));
      const uint32_t v_desc = pt_desc_mn(smem_u32(smem + PT_V_OFF), PT_KEYS * 128);
      auto issue_s = [&](int s, uint32_t g) {
        const uint32_t a = q_desc + s * (32768 >> 4);
        const uint32_t b = k_desc + (g % PT_BUFS) * (PT_STEP_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {  // head dim in steps of 16
          const uint32_t off = (k >> 2) * (16384 >> 4) + (k & 3) * 2;
          pt_mma_ss(leader, t0 + s * 128, a + off, b + off, idesc_s, k != 0);
        }
        pt_commit(leader, &s_full[s]);
      };
      auto issue_pv = [&](int s, uint32_t& gp, uint32_t g, bool first) -> bool {
        const uint32_t b = v_desc + (g % PT_BUFS) * (PT_STEP_BYTES >> 4);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (!wait(&p_full[s * 2 + half], gp & 1)) return false;
#pragma unroll
          for (int k = half * 4; k < half * 4 + 4; ++k)  // keys in steps of 16 (8 columns of P)
            pt_mma_ts(leader, t0 + 256 + s * 128, t0 + s * 128 + k * 8, b + k * (2048 >> 4),
                      idesc_pv, !first || k != 0);
        }
        ++gp;
        return true;
      };
      uint32_t g = 0, seg = 0, gpA = 0, gpB = 0;  // steps, segments, P of tiles A and B
      bool ok = true;
      do {
        const int n = __shfl_sync(0xffffffffu, w.j1 - w.j0, 0);
        const int nA = __shfl_sync(0xffffffffu, sub_steps(0), 0);
        const int nB = __shfl_sync(0xffffffffu, sub_steps(1), 0);
        if (!(ok = wait(q_full, seg & 1))) break;
        if (!(ok = wait(&k_full[g % PT_BUFS], (g / PT_BUFS) & 1))) break;
        if (nA > 0) issue_s(0, g);
        if (nB > 0) issue_s(1, g);
        pt_commit(leader, &k_empty[g % PT_BUFS]);
        for (int j = 0; ok && j < n; ++j) {
          const uint32_t h = g + j;
          if (!(ok = wait(&v_full[h % PT_BUFS], (h / PT_BUFS) & 1))) break;
          if (j < nA) {
            if (!(ok = issue_pv(0, gpA, h, j == 0))) break;
            if (j >= nB) pt_commit(leader, &v_empty[h % PT_BUFS]);
            if (j + 1 < nA) {
              if (!(ok = wait(&k_full[(h + 1) % PT_BUFS], ((h + 1) / PT_BUFS) & 1))) break;
              issue_s(0, h + 1);
            } else {
              pt_commit(leader, &o_full[0]);
            }
          }
          if (j < nB) {
            if (!(ok = issue_pv(1, gpB, h, j == 0))) break;
            pt_commit(leader, &v_empty[h % PT_BUFS]);
            if (j + 1 < nB) {
              if (!(ok = wait(&k_full[(h + 1) % PT_BUFS], ((h + 1) / PT_BUFS) & 1))) break;
              issue_s(1, h + 1);
            } else {
              pt_commit(leader, &o_full[1]);
            }
          }
          if (j + 1 < n) pt_commit(leader, &k_empty[(h + 1) % PT_BUFS]);
        }
        // also for a tile without steps in this segment: no tile's warps run ahead of the
        // others by a segment
        if (ok && nA == 0) pt_commit(leader, &o_full[0]);
        if (ok && nB == 0) pt_commit(leader, &o_full[1]);
        g += n;
        ++seg;
      } while (ok && next_segment());
      pt_commit(leader, drain);  // nothing is in flight when TMEM is given back
      paged_drain<LOADS>(drain, 0);
    }
  } else {
    regs_inc<216>();
    // ---------------- softmax: thread = query row r of tile s
    const int s = (warp - 4) >> 2, quad = warp & 3;
    const int r = quad * 32 + lane;
    uint8_t* q_tile = smem + PT_Q_OFF + s * 32768;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t t_s = tmem + s * 128 + lane_off, t_o = tmem + 256 + s * 128 + lane_off;
    uint32_t g0 = 0;       // steps of the segments before
    uint32_t gs = 0;       // S taken of this tile
    uint32_t seg = 0;      // segments before this one
    bool ok = true;
    do {
      const PagedSeq seq = w.seq;
      const int key_first = w.j0 * PT_KEYS;
      const int f_sub = w.tile * PT_ROWS + s * PT_SUB, f = f_sub + r;
      pt_load_q(q_tile, q, q_stride, seq, w.head, group, f_sub, quad * 32, lane);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);

      const int i = f / group;
      const bool valid = i < seq.n;
      // (rows behind the sequence's last are zero and need no mask: nobody reads their output)
      const int lim = valid ? seq.limit(i) : 0x7fffffff;
      // every row of the tile sees the slots below this
      const int lim_all = seq.limit(f_sub / group);
      const int n_s = sub_steps(s);
      float m = -CUDART_INF_F, l = 0.f;  // the running maximum, less PT_UP, and sum
      for (int j = 0; j < n_s; ++j, ++gs) {
        const int key0 = key_first + j * PT_KEYS;
        ok = __all_sync(0xffffffffu, paged_wait<LOADS>(&s_full[s], gs & 1, failed));
        if (!ok) break;
        tc_fence_after();
        uint32_t u[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(t_s + c * 32, u[c]);
        const uint32_t absent = absent_of[(g0 + j) & 3];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_wait_regs(u[c]);
        if (absent || key0 + PT_KEYS > lim_all) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            // a bit for each key that this row sees
            const int seen = min(max(lim - key0 - c * 32, 0), 32);
            uint32_t bits = seen == 32 ? 0xffffffffu : (1u << seen) - 1;
            if (absent >> (c * 2) & 1u) bits &= 0xffff0000u;
            if (absent >> (c * 2 + 1) & 1u) bits &= 0x0000ffffu;
            if (__all_sync(0xffffffffu, bits == 0xffffffffu)) continue;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(bits >> e & 1u)) u[c][e] = 0xff800000u;  // -inf
          }
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
        const float top =
            fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), scale_log2, -PT_UP<T>);
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
        if (key0 + PT_KEYS > lim_all) {
          // not every row sees every slot of this step: V of slots behind the sequence reads as
          // 0, infinities and NaN of the others too (a thread per slot)
          const uint32_t g = g0 + j;
          ok = __all_sync(0xffffffffu,
                          paged_wait<LOADS>(&v_full[g % PT_BUFS], (g / PT_BUFS) & 1, failed));
          if (!ok) break;
          uint8_t* v = smem + PT_V_OFF + (g % PT_BUFS) * PT_STEP_BYTES + r * 128;
          if (r >= seq.end - key0) {
#pragma unroll 4
            for (int c = 0; c < 16; ++c)
              *reinterpret_cast<uint4*>(v + (c >> 3) * 16384 + ((c & 7) ^ (r & 7)) * 16) =
                  make_uint4(0, 0, 0, 0);
          } else {
            uint32_t any = 0;
#pragma unroll 4
            for (int c = 0; c < 16; ++c) {
              const uint4 x = *reinterpret_cast<const uint4*>(  // (eight rows meet no bank twice)
                  v + (c >> 3) * 16384 + ((c & 7) ^ (r & 7)) * 16);
              any |= H::not_finite(x.x) | H::not_finite(x.y) | H::not_finite(x.z) | H::not_finite(x.w);
            }
            if (any) {
              *odd_v = 1;  // before the values go: the other tile's warps read the same V
              __threadfence_block();
#pragma unroll 1
              for (int c = 0; c < 64; ++c) {
                uint32_t* x = reinterpret_cast<uint32_t*>(v + (c >> 5) * 16384) + (c & 31);
                *x &= ~H::not_finite(*x);
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        const float base = m == -CUDART_INF_F ? 0.f : m;
        const float2 sc2 = make_float2(scale_log2, scale_log2), nb2 = make_float2(-base, -base);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float2 x = ffma2(make_float2(__uint_as_float(u[c][2 * e]), __uint_as_float(u[c][2 * e + 1])),
                             sc2, nb2);
            x.x = exp2_mufu(x.x);
            x.y = exp2_mufu(x.y);
            sum[e & 1] = fadd2(sum[e & 1], x);
            // P rounds to the cache's type: at most half a step of each weight, the size of
            // the output's own rounding (fp16: or 2^-32 of the largest weight, over 2^20
            // slots less than that rounding)
            p[e] = H::pack(x.x, x.y);
          }
          tmem_st_32x32b_x16(t_s + c * 16, p);
          if (c & 1) {  // 64 keys' P are there
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[s * 2 + (c >> 1)]);
          }
        }
        sum[0] = fadd2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
      }
      // ---------------- the segment's output
      const int h = w.head * group + f - i * group;
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      const float row_lse =
          l == 0.f ? -CUDART_INF_F : m + PT_UP<T> + log2f(l * exp2f(-PT_UP<T>));
      const bool some = n_s > 0 && l != 0.f;
      if (ok) ok = __all_sync(0xffffffffu, paged_wait<LOADS>(&o_full[s], seg & 1, failed));
      if (!ok) break;
      tc_fence_after();
      if (*odd_v && n_s > 0) {
        // O += the infinities and NaN that this row sees, of all slots that either tile may
        // have taken them out of (added twice they are what they were). All of the warp takes
        // part: the TMEM accesses are its.
        const int lim_tile = seq.limit(w.tile * PT_ROWS / group);
        for (int key = max(key_first, lim_tile / PT_KEYS * PT_KEYS);
             key < min(w.j1 * PT_KEYS, seq.end); ++key) {
          const int id = kv.page_id(w.b, key);
          if (id < 0) continue;
          const uint4* v = reinterpret_cast<const uint4*>(
              static_cast<const T*>(kv.v) + (int64_t)kv.page_row(id, w.head, key) * PG_HD);
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            const uint4 x0 = v[c * 2], x1 = v[c * 2 + 1];
            uint32_t x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w}, odd = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              x[e] &= H::not_finite(x[e]);
              odd |= x[e];
            }
            if (!odd) continue;  // the same in all lanes
            uint32_t o[16];
            tmem_ld_32x32b_x16(t_o + c * 16, o);
            tmem_ld_wait_regs16(o);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 y = H::unpack(x[e]);
              if (key < lim) {
                o[2 * e] = __float_as_uint(__uint_as_float(o[2 * e]) + y.x);
                o[2 * e + 1] = __float_as_uint(__uint_as_float(o[2 * e + 1]) + y.y);
              }
            }
            tmem_st_32x32b_x16(t_o + c * 16, o);
            tmem_st_wait();
          }
        }
      }
      if (!w.whole()) {
        const int part = 2 * blockIdx.x + (seg == 0 ? 0 : 1);
        if (valid) parts.lse[part * PT_ROWS + s * PT_SUB + r] = row_lse;
        // [128][256 rows]: a warp's store is one line
        float* po = parts.o + (int64_t)part * PG_HD * PT_ROWS + s * PT_SUB + r;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(t_o + c * 32, o);
          tmem_ld_wait_regs(o);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            po[e * PT_ROWS] = some ? __uint_as_float(o[e]) * inv : 0.f;
          po += 32 * PT_ROWS;
        }
        if (w.j0 == 0 && threadIdx.x == 128)  // begins here, goes on in the next shares
          parts.join[blockIdx.x] = w.join(sh.table, blockIdx.x, part, group);
      } else {
        if (lse && valid) lse[((int64_t)seq.row0 + i) * heads + h] = row_lse;
        // through the Q tile (no S reads it any more), so that half a warp writes a whole row
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(t_o + c * 32, o);
          tmem_ld_wait_regs(o);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint4 y = make_uint4(0, 0, 0, 0);
            if (some) {
              y.x = H::pack(__uint_as_float(o[8 * e]) * inv, __uint_as_float(o[8 * e + 1]) * inv);
              y.y = H::pack(__uint_as_float(o[8 * e + 2]) * inv, __uint_as_float(o[8 * e + 3]) * inv);
              y.z = H::pack(__uint_as_float(o[8 * e + 4]) * inv, __uint_as_float(o[8 * e + 5]) * inv);
              y.w = H::pack(__uint_as_float(o[8 * e + 6]) * inv, __uint_as_float(o[8 * e + 7]) * inv);
            }
            const int chunk = c * 4 + e;
            *reinterpret_cast<uint4*>(q_tile + (chunk >> 3) * 16384 + r * 128 +
                                      (((chunk & 7) ^ (r & 7)) << 4)) = y;
          }
        }
        __syncwarp();
        const int chunk = lane & 15;
        int rr = quad * 32 + (lane >> 4);
        int ii = (f_sub + rr) / group, gg = f_sub + rr - ii * group;
#pragma unroll 2
        for (int it = 0; it < 16; ++it) {
          if (ii < seq.n) {
            const uint4 y = *reinterpret_cast<const uint4*>(
                q_tile + (chunk >> 3) * 16384 + rr * 128 + (((chunk & 7) ^ (rr & 7)) << 4));
            *reinterpret_cast<uint4*>(out + ((int64_t)seq.row0 + ii) * out_stride +
                                      (int64_t)(w.head * group + gg) * PG_HD + chunk * 8) = y;
          }
          rr += 2;
          gg += 2;
          while (gg >= group) {
            gg -= group;
            ++ii;
          }
        }
        __syncwarp();  // the next Q goes over it
      }
      tc_fence_before();
      g0 += w.j1 - w.j0;
      ++seg;
    } while (next_segment());
    if (!ok) {
      // a wait ran out: NaN for the rows of this segment and of all behind it
      tmem_st_wait();
      do {
        const int f = w.tile * PT_ROWS + s * PT_SUB + r, i = f / group;
        const bool valid = i < w.seq.n;
        if (!w.whole()) {  // (the join gives a row NaN for one such part)
          const int part = 2 * blockIdx.x + (seg == 0 ? 0 : 1);
          if (valid) parts.lse[part * PT_ROWS + s * PT_SUB + r] = CUDART_NAN_F;
          if (w.j0 == 0 && threadIdx.x == 128)
            parts.join[blockIdx.x] = w.join(sh.table, blockIdx.x, part, group);
        } else if (valid) {
          const int64_t row = (int64_t)w.seq.row0 + i;
          const int h = w.head * group + f - i * group;
          if (lse) lse[row * heads + h] = CUDART_NAN_F;
          for (int c = 0; c < PG_HD / 8; ++c)
            reinterpret_cast<uint4*>(out + row * out_stride + (int64_t)h * PG_HD)[c] =
                make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
        }
        ++seg;
      } while (next_segment());
    }
    tc_fence_before();
  }
  __syncthreads();
  if (threadIdx.x == 0 && *failed != 0) paged_report_timeout();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, PT_TMEM_COLS);
  }
}

// Joins the parts of the tile that begins in share blockIdx.x and goes on behind it:
// out = sum_p 2^(lse_p - lse) o_p. A block takes 32 rows; a warp reads the parts of 32 rows
// at once (whole lines) and the block writes whole rows through shared memory.
constexpr int PJ_ROWS = 32;
constexpr int PJ_WARPS = 8;
template <typename T>
__global__ void __launch_bounds__(PJ_WARPS * 32)
    paged_join_kernel(const ShareParts parts, int heads, int group, T* __restrict__ out,
                      int64_t out_stride, float* __restrict__ lse) {
  using H = Half16<T>;
  pdl_wait();
  const ShareJoin jn = parts.join[blockIdx.x];
  const int r0 = blockIdx.y * PJ_ROWS;
  if (jn.count == 0 || r0 >= jn.rows) return;
  __shared__ float tile[PJ_ROWS][PG_HD + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = r0 + lane;
  auto part_of = [&](int p) { return share_part(jn, blockIdx.x, p); };
  float mx = -CUDART_INF_F;
  for (int p = 0; p < jn.count; ++p) mx = fmaxf(mx, parts.lse[part_of(p) * PT_ROWS + r]);
  const float base = mx == -CUDART_INF_F ? 0.f : mx;
  constexpr int PER = PG_HD / PJ_WARPS;
  float sum = 0.f, acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
  for (int p = 0; p < jn.count; ++p) {
    const int part = part_of(p);
    const float c = exp2_mufu(parts.lse[part * PT_ROWS + r] - base);
    const float* po = parts.o + ((int64_t)part * PG_HD + warp * PER) * PT_ROWS + r;
    sum += c;
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] = fmaf(c, po[e * PT_ROWS], acc[e]);
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
  for (int e = 0; e < PER; ++e) tile[lane][warp * PER + e] = acc[e] * inv;
  const int f = jn.f0 + r, i = f / group;
  if (lse && warp == 0 && r < jn.rows)
    lse[((int64_t)jn.row0 + i) * heads + jn.head * group + f - i * group] =
        sum == 0.f ? -CUDART_INF_F : mx + log2f(sum);
  __syncthreads();
  for (int rr = warp; rr < PJ_ROWS && r0 + rr < jn.rows; rr += PJ_WARPS) {
    const int ff = jn.f0 + r0 + rr, ii = ff / group;
    uint2 y;
    y.x = H::pack(tile[rr][lane * 4], tile[rr][lane * 4 + 1]);
    y.y = H::pack(tile[rr][lane * 4 + 2], tile[rr][lane * 4 + 3]);
    *reinterpret_cast<uint2*>(out + ((int64_t)jn.row0 + ii) * out_stride +
                              (int64_t)(jn.head * group + ff - ii * group) * PG_HD + lane * 4) = y;
  }
}

}  // namespace cb
