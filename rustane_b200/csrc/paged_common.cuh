// What the paged-cache kernels share: the descriptor as they get it, the sequences of a
// step, and the two 16-bit types.
//
// Every value that a kernel reads from device memory (lengths, row starts, page ids) is
// held to the host's bounds here, so no value of them can lead outside the caller's arrays.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <stdint.h>

#include "ptx.cuh"

namespace cb {

constexpr int PG_HD = 128;  // head dim

struct PagedKV {
  void* k;
  void* v;
  const int* table;
  const int* len;
  const int* row_start;
  int pages, kv_heads, page_size, page_shift;
  int batch, table_stride, max_len, rows, max_new;

  // Row of the cache as a [pages * kv_heads * page_size][128] matrix, or -1 for a slot of a
  // page outside the pool. slot < max_len (<= table_stride * page_size, checked on the host).
  __device__ __forceinline__ int page_id(int b, int slot) const {
    const int id = __ldg(table + (size_t)b * table_stride + (slot >> page_shift));
    return (unsigned)id < (unsigned)pages ? id : -1;
  }
  __device__ __forceinline__ int page_row(int id, int head, int slot) const {
    return (id * kv_heads + head) * page_size + (slot & (page_size - 1));
  }
  __device__ __forceinline__ int cache_rows() const { return pages * kv_heads * page_size; }
};

// One sequence's part of a step. Token i < n sees the slots below limit(i).
struct PagedSeq {
  int row0;  // first row of its new tokens
  int n;     // new tokens that are processed (at most max_new)
  int past;  // slots in front of its new tokens (negative: len is below the new tokens)
  int end;   // slots in use, at most max_len

  __device__ __forceinline__ int limit(int i) const { return min(past + i + 1, end); }
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedKV& kv, int b) {
  const int lo = min(max(__ldg(kv.row_start + b), 0), kv.rows);
  const int hi = min(max(__ldg(kv.row_start + b + 1), lo), kv.rows);
  const int len = min(max(__ldg(kv.len + b), 0), 0x3fffffff);
  return PagedSeq{lo, min(hi - lo, kv.max_new), len - (hi - lo), min(len, kv.max_len)};
}

// Every wait of these kernels is bounded. One that runs out ends its CTA's work: what the CTA had
// still to write becomes NaN (never what the arrays held before), its copies in flight are
// waited for, and it is counted in the device's word, which cb_paged_check_device_error reads
// (rows kernel: a count per warp). LOADS = false is the self-test: nothing is ever loaded, so
// the waits run out, after 1 ms.
__device__ int paged_expired;

template <bool LOADS>
__device__ __forceinline__ bool paged_wait(uint64_t* bar, uint32_t parity, int* failed) {
  return mbar_wait_for(bar, parity, failed, LOADS ? CB_WAIT_LIMIT_NS : 1000000ull);
}
// Before a CTA ends: for what is still on its way, also after another wait has run out.
template <bool LOADS>
__device__ __forceinline__ void paged_drain(uint64_t* bar, uint32_t parity) {
  paged_wait<LOADS>(bar, parity, nullptr);
}
__device__ __forceinline__ void paged_report_timeout() {
  atomicAdd(&paged_expired, 1);
}

// Programmatic dependent launch, in its two halves: a kernel lets the next one on the stream
// start (it then waits in pdl_wait for this one's end and memory).
__device__ __forceinline__ void pdl_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// 2^x of two numbers on the FMA pipes, for kernels whose exponentials keep the MUFU busy
// (16 results a clock and SM). x = n + f with n the nearest whole number: 2^f on [-1/2, 1/2] by
// the polynomial of degree 5 with the least largest relative error (Remez's exchange; 2.8e-7, with
// 32-bit steps 3.4e-7, where ex2.approx has 2.4e-7), times 2^n built in the exponent field.
// Results below 2^-126 are 0, as ex2.approx.ftz's; NaN stays NaN. n ends at 127: up to 2^128 the
// polynomial is taken on to f = 1, where it is off by 7e-5, and behind that it overflows.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 fmul2_ftz(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;"
      : "=l"(r)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 exp2_poly2(float2 x) {
  constexpr float MAGIC = 12582912.0f;  // 1.5 x 2^23: adding it rounds to a whole number
  // n = -127 makes an exponent field of 0, exactly 0
  x.x = max_nan(x.x, -127.0f);
  x.y = max_nan(x.y, -127.0f);
  float2 t = fadd2(x, make_float2(MAGIC, MAGIC));
  t.x = min_nan(t.x, MAGIC + 127.0f);
  t.y = min_nan(t.y, MAGIC + 127.0f);
  const float2 n = fadd2(t, make_float2(-MAGIC, -MAGIC));
  const float2 f = ffma2(n, make_float2(-1.0f, -1.0f), x);
  auto both = [](float c) { return make_float2(c, c); };
  float2 p = ffma2(both(1.301088603e-03f), f, both(9.678628296e-03f));
  p = ffma2(p, f, both(5.551895499e-02f));
  p = ffma2(p, f, both(2.402208745e-01f));
  p = ffma2(p, f, both(6.931457520e-01f));
  p = ffma2(p, f, both(1.0f));
  const float2 scale = make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                                   __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u));
  return fmul2_ftz(p, scale);
}

// ------------------------------------------------------------------ the 16-bit types
template <typename T>
struct Half16;
template <>
struct Half16<__half> {
  // P of an attention is taken that many binary places up, as far as the type goes: fp16's
  // normal range ends at 2^-14, and weights below it lose up to 2^-25 each of the largest one,
  // which over a long cache adds up to more than an output's rounding.
  static constexpr float P_UP = 15.0f;
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_half2(lo, hi); }
  static __device__ __forceinline__ __half from(float x) { return __float2half_rn(x); }
  // Of two packed values, 0xffff in the halves that are infinite or NaN.
  static __device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    const uint32_t all_ones = ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
    return (all_ones >> 15) * 0xffffu;
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    mma_16816(d, a, b0, b1);
  }
};
template <>
struct Half16<__nv_bfloat16> {
  static constexpr float P_UP = 0.0f;  // (normal down to 2^-126)
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
  static __device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    const uint32_t all_ones = ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
    return (all_ones >> 15) * 0xffffu;
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

}  // namespace cb
