// Rotary positions: pair i of a head at position p is turned by the angle a = p f_i,
//   (x0, x1) -> (x0 cos a - x1 sin a, x1 cos a + x0 sin a),
// its gradient by -a. Both kernels move 2 + 2 bytes an element and do little else, so they
// are bound by memory. A thread owns four pairs of a head (eight elements: two 8-byte
// pieces, adjacent for interleaved pairs and rot_dim / 2 apart for half pairs) at one token
// and walks heads with them: an angle is formed once for all of a thread's heads, both
// elements of a pair meet in one thread (so a tensor can be rotated in place), and the lanes
// of a head read whole 32-byte sectors.
// The angle is formed in 64 bits as a fraction of a turn (at position 10^6 a 32-bit product
// would be off by 0.06 rad), reduced to [-1/2, 1/2] there, and only then rounded to 32 bits.
#pragma once
#include "paged_common.cuh"

namespace cb {

// cos and sin of pairs 4u .. 4u + 3 at position p, times amp (sin times amp_sin).
__device__ __forceinline__ void rope_angles(const double* __restrict__ inv_freq, int u, int p,
                                            float amp, float amp_sin, float (&c)[4],
                                            float (&s)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double turns = (double)p * __ldg(inv_freq + 4 * u + j) * 0.15915494309189535;
    float sj, cj;
    sincospif(2.0f * (float)(turns - rint(turns)), &sj, &cj);
    c[j] = cj * amp;
    s[j] = sj * amp_sin;
  }
}

// The eight elements of unit u: a holds the first four, b the last four.
template <typename T>
__device__ __forceinline__ void rope_turn(uint2& a, uint2& b, const float (&c)[4],
                                          const float (&s)[4], bool half_layout) {
  using H = Half16<T>;
  const float2 a0 = H::unpack(a.x), a1 = H::unpack(a.y), b0 = H::unpack(b.x),
               b1 = H::unpack(b.y);
  if (half_layout) {
    a.x = H::pack(a0.x * c[0] - b0.x * s[0], a0.y * c[1] - b0.y * s[1]);
    a.y = H::pack(a1.x * c[2] - b1.x * s[2], a1.y * c[3] - b1.y * s[3]);
    b.x = H::pack(b0.x * c[0] + a0.x * s[0], b0.y * c[1] + a0.y * s[1]);
    b.y = H::pack(b1.x * c[2] + a1.x * s[2], b1.y * c[3] + a1.y * s[3]);
  } else {
    a.x = H::pack(a0.x * c[0] - a0.y * s[0], a0.y * c[0] + a0.x * s[0]);
    a.y = H::pack(a1.x * c[1] - a1.y * s[1], a1.y * c[1] + a1.x * s[1]);
    b.x = H::pack(b0.x * c[2] - b0.y * s[2], b0.y * c[2] + b0.x * s[2]);
    b.y = H::pack(b1.x * c[3] - b1.y * s[3], b1.y * c[3] + b1.x * s[3]);
  }
}

// Offsets of unit u's two pieces; units from rot / 8 on are not rotated.
__device__ __forceinline__ void rope_pieces(int u, int rot, bool half_layout, int& off_a,
                                            int& off_b) {
  const bool apart = half_layout && u < rot / 8;
  off_a = apart ? 4 * u : 8 * u;
  off_b = apart ? rot / 2 + 4 * u : 8 * u + 4;
}

constexpr int ROPE_THREADS = 256;

// Grid: every thread one (token, chunk of per_thread heads, unit), the unit fastest.
template <typename T>
__global__ void __launch_bounds__(ROPE_THREADS)
    rope_kernel(const T* x, int64_t x_stride, T* y, int64_t y_stride,  // y may be x
                const int* __restrict__ positions, const double* __restrict__ inv_freq, int rot,
                bool half_layout, float amp, float amp_sin, int tokens, int heads, int head_dim,
                int per_thread) {
  const int units = head_dim / 8;
  const int chunks = (heads + per_thread - 1) / per_thread;
  const int64_t idx = (int64_t)blockIdx.x * ROPE_THREADS + threadIdx.x;
  const int64_t rest = idx / units;
  const int u = (int)(idx - rest * units);
  const int64_t t = rest / chunks;
  if (t >= tokens) return;
  const int h0 = (int)(rest - t * chunks) * per_thread;
  const int h1 = min(heads, h0 + per_thread);
  int off_a, off_b;
  rope_pieces(u, rot, half_layout, off_a, off_b);
  const bool turn = u < rot / 8;
  const T* xp = x + t * x_stride;
  T* yp = y + t * y_stride;
  float c[4], s[4];
  if (turn) rope_angles(inv_freq, u, __ldg(positions + t), amp, amp_sin, c, s);
  for (int h = h0; h < h1; h += 4) {
    uint2 a[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (h + j >= h1) break;
      a[j] = *reinterpret_cast<const uint2*>(xp + (h + j) * head_dim + off_a);
      b[j] = *reinterpret_cast<const uint2*>(xp + (h + j) * head_dim + off_b);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (h + j >= h1) break;
      if (turn) rope_turn<T>(a[j], b[j], c, s, half_layout);
      *reinterpret_cast<uint2*>(yp + (h + j) * head_dim + off_a) = a[j];
      *reinterpret_cast<uint2*>(yp + (h + j) * head_dim + off_b) = b[j];
    }
  }
}

constexpr int APPEND_WARPS = 8;

// One warp per (row, chunk of per_warp heads): half a warp holds a head's 16 units. The
// row's heads are counted q first, then k, then v. rot = 0 when nothing is rotated.
template <typename T>
__global__ void __launch_bounds__(APPEND_WARPS * 32)
    paged_append_kernel(const PagedKV kv, const T* q, int64_t q_stride,
                        T* q_out, int64_t q_out_stride, int heads,  // q_out may be q
                        const T* __restrict__ k, int64_t k_stride, const T* __restrict__ v,
                        int64_t v_stride, const int* __restrict__ positions,
                        const double* __restrict__ inv_freq, int rot, bool half_layout, float amp,
                        float* __restrict__ weights, int* __restrict__ slot_positions,
                        int per_warp) {
  const int lane = threadIdx.x & 31;
  const int all = heads + 2 * kv.kv_heads;
  const int chunks = (all + per_warp - 1) / per_warp;
  const int64_t warp = (int64_t)blockIdx.x * APPEND_WARPS + (threadIdx.x >> 5);
  const int64_t r64 = warp / chunks;
  if (r64 >= kv.rows) return;
  const int r = (int)r64, chunk = (int)(warp - r64 * chunks);

  // the last sequence that starts at or before this row
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
  const int slot = seq.past + i;
  const int id = slot >= 0 && slot < seq.end ? kv.page_id(b, slot) : -1;
  const int p = positions ? __ldg(positions + r) : slot;

  if (chunk == 0 && id >= 0 && (weights || slot_positions)) {
    for (int h = lane; h < kv.kv_heads; h += 32) {
      const int at = kv.page_row(id, h, slot);
      if (weights) weights[at] = 0.f;
      if (slot_positions) slot_positions[at] = p;
    }
  }

  const int u = lane & 15;
  int off_a, off_b;
  rope_pieces(u, rot, half_layout, off_a, off_b);
  float c[4], s[4];
  if (u < rot / 8) rope_angles(inv_freq, u, p, amp, amp, c, s);
  const int h1 = min(all, (chunk + 1) * per_warp);
  for (int h0 = chunk * per_warp + (lane >> 4); h0 < h1; h0 += 8) {
    uint2 a[4], bb[4];
    const T* src[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int h = h0 + 2 * j;
      if (h >= h1) break;
      src[j] = h < heads ? q + r * q_stride + (int64_t)h * PG_HD
               : h < heads + kv.kv_heads
                   ? k + r * k_stride + (int64_t)(h - heads) * PG_HD
                   : v + r * v_stride + (int64_t)(h - heads - kv.kv_heads) * PG_HD;
      a[j] = *reinterpret_cast<const uint2*>(src[j] + off_a);
      bb[j] = *reinterpret_cast<const uint2*>(src[j] + off_b);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int h = h0 + 2 * j;
      if (h >= h1) break;
      const bool is_v = h >= heads + kv.kv_heads;
      if (u < rot / 8 && !is_v) rope_turn<T>(a[j], bb[j], c, s, half_layout);
      T* dst;
      if (h < heads) {
        dst = q_out + r * q_out_stride + (int64_t)h * PG_HD;
      } else {
        if (id < 0) continue;  // a page outside the pool, or a slot outside the sequence
        const int hk = is_v ? h - heads - kv.kv_heads : h - heads;
        dst = static_cast<T*>(is_v ? kv.v : kv.k) + (int64_t)kv.page_row(id, hk, slot) * PG_HD;
      }
      *reinterpret_cast<uint2*>(dst + off_a) = a[j];
      *reinterpret_cast<uint2*>(dst + off_b) = bb[j];
    }
  }
}

}  // namespace cb
