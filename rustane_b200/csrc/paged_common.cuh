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

// The sequence and tile of a flat tile index, when the n * group query rows of each sequence
// are cut into tiles of M. The whole warp calls it; b = -1 when there are fewer tiles.
struct PagedTile {
  int b, tile;
  PagedSeq seq;
};
template <int M>
__device__ __forceinline__ PagedTile paged_find_tile(const PagedKV& kv, int group, int t) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int base = 0; base < kv.batch; base += 32) {
    PagedSeq s{0, 0, 0, 0};
    if (base + lane < kv.batch) s = paged_seq(kv, base + lane);
    const int tiles = (s.n * group + M - 1) / M;
    int incl = tiles;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += up;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + incl > t);
    if (past) {
      const int src = __ffs(past) - 1;
      PagedTile r;
      r.b = base + src;
      r.tile = t - before - __shfl_sync(0xffffffffu, incl - tiles, src);
      r.seq.row0 = __shfl_sync(0xffffffffu, s.row0, src);
      r.seq.n = __shfl_sync(0xffffffffu, s.n, src);
      r.seq.past = __shfl_sync(0xffffffffu, s.past, src);
      r.seq.end = __shfl_sync(0xffffffffu, s.end, src);
      return r;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return PagedTile{-1, 0, PagedSeq{0, 0, 0, 0}};
}

// ------------------------------------------------------------------ the 16-bit types
template <typename T>
struct Half16;
template <>
struct Half16<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_half2(lo, hi); }
  static __device__ __forceinline__ __half from(float x) { return __float2half_rn(x); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    mma_16816(d, a, b0, b1);
  }
};
template <>
struct Half16<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
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
