// Rotary positions: pair i of a head at position p is turned by the angle a = p f_i,
//   (x0, x1) -> (x0 cos a - x1 sin a, x1 cos a + x0 sin a),
// its gradient by -a. Both kernels move 2 + 2 bytes an element and are bound by memory as long
// as an angle (it costs about as much as moving ten elements) serves several heads. A thread
// owns PIECE pairs of a head at one token (two pieces of PIECE elements, adjacent for
// interleaved pairs and rot_dim / 2 apart for half pairs) and walks heads with them: an angle is
// formed once for all of a thread's heads, both elements of a pair meet in one thread (so a
// tensor can be rotated in place), and the next heads' loads are out while a head is turned.
// PIECE is 8 (16-byte accesses) where rot_dim and the head's size are multiples of 16, else 4.
// The angle is formed in 64 bits as a fraction of a turn (at position 10^6 a 32-bit product
// would be off by 0.06 rad), reduced to [-1/2, 1/2] there, and only then rounded to 32 bits.
// Measured: 16384 tokens x 12 heads of 128, interleaved, f16, 101 MB: 20.7 us, 4.9 TB/s (torch's
// copy of as much: 35 us); appending 12 prompts of up to 1000 tokens, 32 / 8 heads, bf16, 191 MB:
// 38.4 us, 5.0 TB/s; one token of 64 sequences: 3.7 us, a launch and three dependent reads.
#pragma once
#include "paged_common.cuh"

namespace cb {

template <int PIECE>
struct RopeUnit {
  static constexpr int WORDS = PIECE / 2;  // of a piece
  float c[PIECE], s[PIECE];                // cos and sin of its pairs
  int off_a, off_b;                        // of its pieces within the head
  bool turn;                               // false: these elements pass
  bool half_layout;

  __device__ __forceinline__ RopeUnit(int u, int rot, bool half) : half_layout(half) {
    turn = u < rot / (2 * PIECE);
    const bool apart = half && turn;
    off_a = apart ? PIECE * u : 2 * PIECE * u;
    off_b = apart ? rot / 2 + PIECE * u : 2 * PIECE * u + PIECE;
  }
  // The angles of unit u at position p; sin times amp_sin.
  __device__ __forceinline__ void angles(const double* __restrict__ inv_freq, int u, int p,
                                         float amp, float amp_sin) {
    if (!turn) return;
#pragma unroll
    for (int j = 0; j < PIECE; ++j) {
      const double turns = (double)p * __ldg(inv_freq + PIECE * u + j) * 0.15915494309189535;
      float sj, cj;
      sincospif(2.0f * (float)(turns - rint(turns)), &sj, &cj);
      c[j] = cj * amp;
      s[j] = sj * amp_sin;
    }
  }
  template <typename T>
  static __device__ __forceinline__ void load(const T* head, int off, uint32_t (&w)[WORDS]) {
    if constexpr (PIECE == 8) {
      const uint4 x = *reinterpret_cast<const uint4*>(head + off);
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(head + off);
      w[0] = x.x, w[1] = x.y;
    }
  }
  template <typename T>
  static __device__ __forceinline__ void store(T* head, int off, const uint32_t (&w)[WORDS]) {
    if constexpr (PIECE == 8)
      *reinterpret_cast<uint4*>(head + off) = make_uint4(w[0], w[1], w[2], w[3]);
    else
      *reinterpret_cast<uint2*>(head + off) = make_uint2(w[0], w[1]);
  }
  template <typename T>
  __device__ __forceinline__ void rotate(uint32_t (&a)[WORDS], uint32_t (&b)[WORDS]) const {
    using H = Half16<T>;
    if (half_layout) {  // pair j: element j of both pieces
#pragma unroll
      for (int k = 0; k < WORDS; ++k) {
        const float2 x = H::unpack(a[k]), y = H::unpack(b[k]);
        a[k] = H::pack(x.x * c[2 * k] - y.x * s[2 * k], x.y * c[2 * k + 1] - y.y * s[2 * k + 1]);
        b[k] = H::pack(y.x * c[2 * k] + x.x * s[2 * k], y.y * c[2 * k + 1] + x.y * s[2 * k + 1]);
      }
    } else {  // pair j: word j of the two pieces one after the other
#pragma unroll
      for (int k = 0; k < WORDS; ++k) {
        const float2 x = H::unpack(a[k]), y = H::unpack(b[k]);
        const int j = WORDS + k;
        a[k] = H::pack(x.x * c[k] - x.y * s[k], x.y * c[k] + x.x * s[k]);
        b[k] = H::pack(y.x * c[j] - y.y * s[j], y.y * c[j] + y.x * s[j]);
      }
    }
  }
};

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_BATCH = 2;  // heads whose loads are out together

// Grid: every thread one (token, chunk of per_thread heads, unit), the unit fastest.
template <typename T, int PIECE>
__global__ void __launch_bounds__(ROPE_THREADS)
    rope_kernel(const T* x, int64_t x_stride, T* y, int64_t y_stride,  // y may be x
                const int* __restrict__ positions, const double* __restrict__ inv_freq, int rot,
                bool half_layout, float amp, float amp_sin, int tokens, int heads, int head_dim,
                int per_thread) {
  using Unit = RopeUnit<PIECE>;
  const int units = head_dim / (2 * PIECE);
  const int chunks = (heads + per_thread - 1) / per_thread;
  const int64_t idx = (int64_t)blockIdx.x * ROPE_THREADS + threadIdx.x;
  const int64_t rest = idx / units;
  const int u = (int)(idx - rest * units);
  const int64_t t = rest / chunks;
  if (t >= tokens) return;
  const int h0 = (int)(rest - t * chunks) * per_thread;
  const int h1 = min(heads, h0 + per_thread);
  Unit unit(u, rot, half_layout);
  const T* xp = x + t * x_stride;
  T* yp = y + t * y_stride;
  uint32_t a[2][ROPE_BATCH][Unit::WORDS], b[2][ROPE_BATCH][Unit::WORDS];
  auto load = [&](int h, int buf) {
#pragma unroll
    for (int j = 0; j < ROPE_BATCH; ++j) {
      if (h + j >= h1) break;
      Unit::load(xp + (h + j) * head_dim, unit.off_a, a[buf][j]);
      Unit::load(xp + (h + j) * head_dim, unit.off_b, b[buf][j]);
    }
  };
  auto finish = [&](int h, int buf) {
#pragma unroll
    for (int j = 0; j < ROPE_BATCH; ++j) {
      if (h + j >= h1) break;
      if (unit.turn) unit.template rotate<T>(a[buf][j], b[buf][j]);
      Unit::store(yp + (h + j) * head_dim, unit.off_a, a[buf][j]);
      Unit::store(yp + (h + j) * head_dim, unit.off_b, b[buf][j]);
    }
  };
  load(h0, 0);
  unit.angles(inv_freq, u, __ldg(positions + t), amp, amp_sin);
  for (int h = h0; h < h1; h += 2 * ROPE_BATCH) {
    load(h + ROPE_BATCH, 1);
    finish(h, 0);
    load(h + 2 * ROPE_BATCH, 0);
    finish(h + ROPE_BATCH, 1);
  }
}

constexpr int APPEND_WARPS = 8;

// One warp per (row, chunk of per_warp heads): a head's units lie side by side in the warp, so
// it takes 32 / units heads at once. The row's heads are counted q first, then k, then v.
// rot = 0 when nothing is rotated.
template <typename T, int PIECE>
__global__ void __launch_bounds__(APPEND_WARPS * 32)
    paged_append_kernel(const PagedKV kv, const T* q, int64_t q_stride,
                        T* q_out, int64_t q_out_stride, int heads,  // q_out may be q
                        const T* __restrict__ k, int64_t k_stride, const T* __restrict__ v,
                        int64_t v_stride, const int* __restrict__ positions,
                        const double* __restrict__ inv_freq, int rot, bool half_layout, float amp,
                        float* __restrict__ weights, int* __restrict__ slot_positions,
                        int per_warp) {
  using Unit = RopeUnit<PIECE>;
  constexpr int UNITS = PG_HD / (2 * PIECE), AT_ONCE = 32 / UNITS;
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

  const int u = lane % UNITS;
  Unit unit(u, rot, half_layout);
  const int h1 = min(all, (chunk + 1) * per_warp);
  uint32_t wa[2][Unit::WORDS], wb[2][Unit::WORDS];
  auto load = [&](int h, int buf) {
    if (h >= h1) return;
    const T* src = h < heads ? q + r * q_stride + (int64_t)h * PG_HD
                   : h < heads + kv.kv_heads
                       ? k + r * k_stride + (int64_t)(h - heads) * PG_HD
                       : v + r * v_stride + (int64_t)(h - heads - kv.kv_heads) * PG_HD;
    Unit::load(src, unit.off_a, wa[buf]);
    Unit::load(src, unit.off_b, wb[buf]);
  };
  auto finish = [&](int h, int buf) {
    if (h >= h1) return;
    const bool is_v = h >= heads + kv.kv_heads;
    if (unit.turn && !is_v) unit.template rotate<T>(wa[buf], wb[buf]);
    T* dst;
    if (h < heads) {
      dst = q_out + r * q_out_stride + (int64_t)h * PG_HD;
    } else {
      if (id < 0) return;  // a page outside the pool, or a slot outside the sequence
      const int hk = is_v ? h - heads - kv.kv_heads : h - heads;
      dst = static_cast<T*>(is_v ? kv.v : kv.k) + (int64_t)kv.page_row(id, hk, slot) * PG_HD;
    }
    Unit::store(dst, unit.off_a, wa[buf]);
    Unit::store(dst, unit.off_b, wb[buf]);
  };
  const int h0 = chunk * per_warp + lane / UNITS;
  load(h0, 0);
  unit.angles(inv_freq, u, p, amp, amp);
  for (int h = h0; h < h1; h += 2 * AT_ONCE) {
    load(h + AT_ONCE, 1);
    finish(h, 0);
    load(h + 2 * AT_ONCE, 0);
    finish(h + AT_ONCE, 1);
  }
}

}  // namespace cb
