// C entry points of the paged KV cache and of the rotary embedding (include/cuda_bridge.h,
// "Serving from a paged KV cache"). Each call checks its arguments on the host, holds what
// only the device knows to the descriptor's bounds in the kernels, and enqueues its kernels
// without allocating or synchronising.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <limits>
#include <type_traits>

#include "cuda_bridge.h"
#include "paged_attention.cuh"
#include "paged_attention_tc.cuh"
#include "paged_common.cuh"
#include "paged_evict.cuh"
#include "paged_rope.cuh"
#include "paged_weights_tc.cuh"
#include "tensor_map.h"

using namespace cb;

namespace {

constexpr int PG_SMS = 148;  // of a B200: the plans below are made for it, without a GPU
constexpr int64_t INT_LIMIT = std::numeric_limits<int32_t>::max();

// ------------------------------------------------------------------------ checks
bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

constexpr float LOG2_E = 1.4426950408889634f;
// The kernels take scale * log2(e), which has to be finite too.
bool scale_ok(float scale) { return scale > 0.0f && std::isfinite(scale * LOG2_E); }

bool dtype_ok(int32_t d) { return d == CB_DTYPE_F16 || d == CB_DTYPE_BF16; }

// Sizes of a descriptor (no pointers).
bool kv_sizes_ok(const cb_paged_kv* kv) {
  if (!kv || !dtype_ok(kv->dtype)) return false;
  if (kv->page_size != 16 && kv->page_size != 32 && kv->page_size != 64 && kv->page_size != 128)
    return false;
  if (kv->pages <= 0 || kv->kv_heads <= 0 || kv->batch <= 0 || kv->table_stride <= 0 ||
      kv->max_len <= 0 || kv->rows < 0 || kv->max_new < 0 || kv->max_new > kv->rows)
    return false;
  if (kv->max_len > (int64_t)kv->table_stride * kv->page_size) return false;
  // cache rows are TMA coordinates (a tile's worth of head room)
  return (double)kv->pages * kv->kv_heads * kv->page_size < (double)(INT_LIMIT - 1024) &&
         kv->batch < INT_LIMIT - 64 && kv->max_len < INT_LIMIT / 2;
}

bool kv_pointers_ok(const cb_paged_kv* kv, bool rows_needed) {
  if (!kv->k || !kv->v || !kv->table || !kv->len || (rows_needed && !kv->row_start)) return false;
  return aligned(kv->k, 16) && aligned(kv->v, 16) && aligned(kv->table, 4) &&
         aligned(kv->len, 4) && aligned(kv->row_start, 4);
}

bool heads_ok(const cb_paged_kv* kv, int32_t heads) {
  return heads > 0 && heads % kv->kv_heads == 0 && heads / kv->kv_heads <= 128 &&
         (int64_t)kv->rows * heads <= INT_LIMIT &&
         (int64_t)kv->max_new * heads <= INT_LIMIT;
}

// A token array: [rows][width] elements of two bytes. One without rows may be null, as that of
// an empty tensor. No memory has 2^60 elements: the bytes up to its end fit 64 bits.
bool array_ok(const void* p, int64_t rows, int64_t stride, int64_t width) {
  if (rows == 0) return true;
  return p && aligned(p, 16) && stride >= width && stride % 8 == 0 &&
         stride <= (int64_t(1) << 40) && (double)rows * (double)stride < 0x1p60;
}

// Whether two token arrays share an element. Columns of one wider array do not.
bool arrays_overlap(const void* a, int64_t a_stride, int64_t a_width, const void* b,
                    int64_t b_stride, int64_t b_width, int64_t rows) {
  const int64_t pa = reinterpret_cast<intptr_t>(a), pb = reinterpret_cast<intptr_t>(b);
  const int64_t ea = pa + ((rows - 1) * a_stride + a_width) * 2;
  const int64_t eb = pb + ((rows - 1) * b_stride + b_width) * 2;
  if (ea <= pb || eb <= pa) return false;
  if (a_stride != b_stride) return true;
  const int64_t s = a_stride * 2, off = ((pb - pa) % s + s) % s;
  return !(off >= a_width * 2 && off + b_width * 2 <= s);
}

bool ranges_overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const int64_t pa = reinterpret_cast<intptr_t>(a), pb = reinterpret_cast<intptr_t>(b);
  return pa < pb + b_bytes && pb < pa + a_bytes;
}

// What a call reads or writes, from its first to its last byte; a token array by its rows.
struct Span {
  const void* p;
  int64_t bytes;
};
Span token_span(const void* p, int64_t rows, int64_t stride, int64_t width) {
  return Span{p, ((rows - 1) * stride + width) * 2};
}
Span meta_span(const void* p, const cb_paged_kv* kv) {  // [pages][kv_heads][page_size]
  return Span{p, (int64_t)kv->pages * kv->kv_heads * kv->page_size * 4};
}
Span pool_span(const void* p, const cb_paged_kv* kv) {
  return Span{p, (int64_t)kv->pages * kv->kv_heads * kv->page_size * PG_HD * 2};
}
Span table_span(const cb_paged_kv* kv) {
  return Span{kv->table, (int64_t)kv->batch * kv->table_stride * 4};
}
Span len_span(const cb_paged_kv* kv) { return Span{kv->len, kv->batch * 4ll}; }
Span row_start_span(const cb_paged_kv* kv) { return Span{kv->row_start, (kv->batch + 1ll) * 4}; }

// Whether an output meets another output or an input (those of one call; null ones are absent).
bool outputs_meet(std::initializer_list<Span> outputs, std::initializer_list<Span> inputs) {
  auto meet = [](const Span& a, const Span& b) {
    return a.p && b.p && ranges_overlap(a.p, a.bytes, b.p, b.bytes);
  };
  for (const Span* o = outputs.begin(); o != outputs.end(); ++o) {
    for (const Span* x = o + 1; x != outputs.end(); ++x)
      if (meet(*o, *x)) return true;
    for (const Span& x : inputs)
      if (meet(*o, x)) return true;
  }
  return false;
}

// The current device is a B200 and every (non-null) pointer is memory of it.
cb_status check_device(std::initializer_list<const void*> pointers) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();  // not the next call's error
    return CB_ERR_CUDA;
  }
  static std::atomic<uint64_t> known{0};  // bit per device that was found to be one
  if (dev >= 64 || !(known.load(std::memory_order_relaxed) >> dev & 1)) {
    int major = 0, minor = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev) != cudaSuccess) {
      cudaGetLastError();
      return CB_ERR_CUDA;
    }
    if (major != 10 || minor != 0) return CB_ERR_UNSUPPORTED;
    if (dev < 64) known.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
  }
  for (const void* p : pointers) {
    if (!p) continue;
    cudaPointerAttributes a;
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
      cudaGetLastError();
      return CB_ERR_INVALID_ARG;
    }
    if (!(a.type == cudaMemoryTypeDevice && a.device == dev) && a.type != cudaMemoryTypeManaged)
      return CB_ERR_INVALID_ARG;
  }
  return CB_OK;
}

PagedKV device_kv(const cb_paged_kv* kv) {
  PagedKV d;
  d.k = kv->k;
  d.v = kv->v;
  d.table = kv->table;
  d.len = kv->len;
  d.row_start = kv->row_start;
  d.pages = kv->pages;
  d.kv_heads = kv->kv_heads;
  d.page_size = kv->page_size;
  d.page_shift = kv->page_size == 16 ? 4 : kv->page_size == 32 ? 5 : kv->page_size == 64 ? 6 : 7;
  d.batch = kv->batch;
  d.table_stride = kv->table_stride;
  d.max_len = kv->max_len;
  d.rows = kv->rows;
  d.max_new = kv->max_new;
  return d;
}

cb_status status_of(cudaError_t e) {
  if (e == cudaSuccess) return CB_OK;
  cudaGetLastError();
  return CB_ERR_CUDA;
}

// Dynamic shared memory above 48 KB is asked for once per kernel and device.
template <typename F>
cudaError_t allow_smem(F* kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && (done.load(std::memory_order_acquire) >> dev & 1)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(uint64_t(1) << dev, std::memory_order_release);
  return e;
}

// The cache as a [rows][128] matrix in boxes of box_rows x 64 elements, 128-byte swizzle.
// (Both types are two bytes and out-of-range rows read as zero bytes: one element type does.)
bool make_cache_map(CUtensorMap* map, const void* ptr, const cb_paged_kv* kv, uint32_t box_rows) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[2] = {(cuuint64_t)PG_HD, (cuuint64_t)kv->pages * kv->kv_heads * kv->page_size};
  cuuint64_t strides[1] = {PG_HD * 2};
  cuuint32_t box[2] = {64, box_rows};
  cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(ptr), dims, strides, box,
             estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ------------------------------------------------------------------- attention plan
// Bounds of a step's work in tiles of `rows` query rows and steps of `keys` slots (the device
// knows how much there is): no more tiles than the rows need with one ragged tile per sequence,
// and no more than batch x those of the longest.
double step_bound(const cb_paged_kv* kv, int group, int rows, int keys) {
  const int64_t tiles =
      std::min<int64_t>(kv->batch * ceil_div((int64_t)kv->max_new * group, rows),
                        ceil_div((int64_t)kv->rows * group, rows) + kv->batch);
  return (double)tiles * kv->kv_heads * ceil_div(kv->max_len, keys);
}
// Shares count units of 32 bits: every step, and up to three for each tile (which has a step).
bool shares_ok(double steps) { return steps * 4 < (double)INT_LIMIT; }

struct AttentionPlan {
  bool tc;          // the tcgen05 kernel, else the 16-row one
  double steps;     // at most
  int ctas;         // one per SM, or as many as there can be steps
  size_t workers;   // with a share each
  size_t rows;      // query rows of a tile: of a part
  size_t bytes() const {
    return workers * (2 * rows * (PG_HD + 1) * sizeof(float) + sizeof(ShareJoin));
  }
};

// More than 16 query rows per key head go to the tcgen05 kernel. Both sides measured (us, the L2
// flushed before each call; bf16, 8 key heads):
//                rows per key head     8    16    24    32    64   128
//   4 x 8192 slots,  16-row kernel    47    49    66    68   100   160
//                    tcgen05          53    53    55    53    55    55
//   32 x 2048 slots, 16-row kernel    74    78   119   121   199   360
//                    tcgen05          82    84    86    86    88    88
AttentionPlan plan_attention(const cb_paged_kv* kv, int32_t heads) {
  AttentionPlan p;
  const int group = heads / kv->kv_heads;
  p.tc = (int64_t)kv->max_new * group > PR_ROWS;
  p.rows = p.tc ? PT_ROWS : PR_ROWS;
  p.steps = step_bound(kv, group, (int)p.rows, p.tc ? PT_KEYS : PR_BLOCK);
  p.ctas = (int)std::max(1.0, std::min<double>(PG_SMS, p.steps));
  p.workers = (size_t)p.ctas * (p.tc ? 1 : PR_WARPS);
  return p;
}

// A kernel that may start before the one in front of it on the stream has ended (it waits for
// that itself).
template <typename... Params, typename... Args>
cudaError_t launch_pdl(void (*kernel)(Params...), dim3 grid, int threads, cudaStream_t st,
                       Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

template <typename T, bool LOADS>
cb_status launch_attention(const cb_paged_kv* kv, const T* q, int64_t q_stride, int32_t heads,
                           float scale, T* out, int64_t out_stride, float* lse, float* workspace,
                           cudaStream_t st) {
  const AttentionPlan p = plan_attention(kv, heads);
  if (!shares_ok(p.steps)) return CB_ERR_UNSUPPORTED;
  const int box = p.tc ? std::min(kv->page_size, PT_KEYS) : PR_BLOCK;
  const int group = heads / kv->kv_heads;
  CUtensorMap tk, tv;
  if (!make_cache_map(&tk, kv->k, kv, box) || !make_cache_map(&tv, kv->v, kv, box))
    return CB_ERR_UNSUPPORTED;
  const PagedKV d = device_kv(kv);
  const float scale_log2 = scale * LOG2_E;
  float* part_lse = workspace + p.workers * 2 * p.rows * PG_HD;
  const ShareParts parts{workspace, part_lse,
                         reinterpret_cast<ShareJoin*>(part_lse + p.workers * 2 * p.rows)};
  cudaError_t e;
  if (p.tc) {
    static std::atomic<uint64_t> done{0};
    if ((e = allow_smem(paged_tile_kernel<T, LOADS>, PT_SMEM, done)) != cudaSuccess)
      return status_of(e);
    paged_tile_kernel<T, LOADS><<<p.ctas, PT_THREADS, PT_SMEM, st>>>(
        tk, tv, d, q, q_stride, heads, scale_log2, out, out_stride, lse, parts, box);
    if ((e = cudaPeekAtLastError()) != cudaSuccess) return status_of(e);
    e = launch_pdl(paged_join_kernel<T>, dim3(p.ctas, PT_ROWS / PJ_ROWS), PJ_WARPS * 32, st, parts,
                   heads, group, out, out_stride, lse);
  } else {
    static std::atomic<uint64_t> done{0};
    if ((e = allow_smem(paged_rows_kernel<T, LOADS>, PR_SMEM, done)) != cudaSuccess)
      return status_of(e);
    paged_rows_kernel<T, LOADS><<<p.ctas, PR_WARPS * 32, PR_SMEM, st>>>(
        tk, tv, d, q, q_stride, heads, scale_log2, out, out_stride, lse, parts);
    if ((e = cudaPeekAtLastError()) != cudaSuccess) return status_of(e);
    const int tile_rows = (int)std::min<int64_t>(PR_ROWS, (int64_t)kv->max_new * group);
    e = launch_pdl(paged_rows_join_kernel<T>, dim3(p.ctas, tile_rows), PR_WARPS * 32, st, parts,
                   heads, group, out, out_stride, lse);
  }
  return status_of(e);
}

// q as a [rows][heads][128] array in boxes of tokens x group x 64, 128-byte swizzle.
bool make_q_map(CUtensorMap* map, const void* q, int64_t q_stride, int heads, int rows, int group,
                int tokens) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[3] = {(cuuint64_t)PG_HD, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t strides[2] = {PG_HD * 2, (cuuint64_t)q_stride * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)tokens};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(q), dims, strides, box,
             estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool LOADS>
cb_status launch_weights(const cb_paged_kv* kv, const T* q, int64_t q_stride, int32_t heads,
                         float scale, const float* lse, float* weights, cudaStream_t st) {
  const int group = heads / kv->kv_heads;
  const PagedKV d = device_kv(kv);
  const float scale_log2 = scale * LOG2_E;
  if ((int64_t)kv->max_new * group <= PR_ROWS) {
    // two CTAs per SM; no more than there are blocks of slots
    const double blocks = step_bound(kv, group, PR_ROWS, PR_BLOCK);
    if (!shares_ok(blocks)) return CB_ERR_UNSUPPORTED;
    const int ctas = (int)std::max(1.0, std::min(2.0 * PG_SMS, blocks));
    paged_weights_kernel<T><<<ctas, PW_WARPS * 32, 0, st>>>(d, q, q_stride, heads, scale_log2, lse,
                                                           weights);
    return status_of(cudaPeekAtLastError());
  }
  const int blocks = (int)ceil_div(kv->max_len, WT_KEYS);
  const int64_t grid = (int64_t)kv->batch * blocks * kv->kv_heads;
  if (grid > INT_LIMIT) return CB_ERR_UNSUPPORTED;
  const int box = std::min(kv->page_size, 128), tokens = WT_ROWS / group;
  CUtensorMap tk, tq;
  if (!make_cache_map(&tk, kv->k, kv, box) ||
      !make_q_map(&tq, q, q_stride, heads, kv->rows, group, tokens))
    return CB_ERR_UNSUPPORTED;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(paged_weights_tile_kernel<T, LOADS>, WT_SMEM, done);
  if (e != cudaSuccess) return status_of(e);
  paged_weights_tile_kernel<T, LOADS><<<(unsigned)grid, WT_THREADS, WT_SMEM, st>>>(
      tk, tq, d, heads, scale_log2, lse, weights, blocks, box, tokens);
  return status_of(cudaPeekAtLastError());
}

// ---------------------------------------------------------------------- evict plan
template <int THREADS, int PER>
cudaError_t launch_evict(const PagedKV& kv, const EvictArgs& a, int ctas, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)kv.batch * kv.kv_heads * ctas));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, paged_evict_kernel<THREADS, PER>, kv, a, ctas);
}

// Calls f with a value of the 16-bit type and the piece size as a type.
template <typename F>
void with_type(int32_t dtype, int piece, F&& f) {
  using P4 = std::integral_constant<int, 4>;
  using P8 = std::integral_constant<int, 8>;
  if (dtype == CB_DTYPE_F16) {
    if (piece == 8) f(__half(), P8()); else f(__half(), P4());
  } else {
    if (piece == 8) f(__nv_bfloat16(), P8()); else f(__nv_bfloat16(), P4());
  }
}

}  // namespace

extern "C" {

cb_status cb_rope_frequencies(int32_t rot_dim, const cb_rope_scaling* scaling, double* inv_freq,
                              float* amplitude) {
  if (!scaling || !inv_freq || rot_dim <= 0 || rot_dim % 8 != 0) return CB_ERR_INVALID_ARG;
  const cb_rope_scaling& s = *scaling;
  if (!(s.base > 1.0) || !std::isfinite(s.base)) return CB_ERR_INVALID_ARG;
  if (s.kind < CB_ROPE_SCALE_NONE || s.kind > CB_ROPE_SCALE_PARTS) return CB_ERR_INVALID_ARG;
  if (s.kind != CB_ROPE_SCALE_NONE && (!(s.factor >= 1.0) || !std::isfinite(s.factor)))
    return CB_ERR_INVALID_ARG;
  double base = s.base;
  if (s.kind == CB_ROPE_SCALE_BASE) base *= std::pow(s.factor, (double)rot_dim / (rot_dim - 2));
  if (!std::isfinite(base)) return CB_ERR_INVALID_ARG;
  double lo = 0.0, hi = 0.0;
  if (s.kind == CB_ROPE_SCALE_PARTS) {
    if (!(s.original_len > 0.0) || !(s.slow_turns > 0.0) || !(s.fast_turns >= s.slow_turns) ||
        !std::isfinite(s.original_len) || !std::isfinite(s.fast_turns))
      return CB_ERR_INVALID_ARG;
    // the pair that turns `turns` times within original_len: p f = 2 pi turns
    const double two_pi = 6.283185307179586;
    auto pair = [&](double turns) {
      return rot_dim * std::log(s.original_len / (turns * two_pi)) / (2.0 * std::log(base));
    };
    lo = std::max(0.0, std::floor(pair(s.fast_turns)));
    hi = std::min(rot_dim - 1.0, std::ceil(pair(s.slow_turns)));
  }
  for (int i = 0; i < rot_dim / 2; ++i) {
    double f = std::pow(base, -2.0 * i / rot_dim);
    if (s.kind == CB_ROPE_SCALE_LINEAR) f /= s.factor;
    if (s.kind == CB_ROPE_SCALE_PARTS) {
      const double ramp = std::min(1.0, std::max(0.0, (i - lo) / std::max(hi - lo, 0.001)));
      f = f / s.factor * ramp + f * (1.0 - ramp);
    }
    inv_freq[i] = f;
  }
  if (amplitude)
    *amplitude = s.kind == CB_ROPE_SCALE_PARTS ? (float)(0.1 * std::log(s.factor) + 1.0) : 1.0f;
  return CB_OK;
}

static bool rope_config_ok(const cb_rope_config* r, int32_t head_dim) {
  return r && r->inv_freq && aligned(r->inv_freq, 8) && r->rot_dim > 0 && r->rot_dim % 8 == 0 &&
         r->rot_dim <= head_dim &&
         (r->layout == CB_ROPE_HALF || r->layout == CB_ROPE_INTERLEAVED) &&
         std::isfinite(r->amplitude);
}

cb_status cb_rope(const cb_rope_config* rope, int32_t dtype, const void* x, int64_t x_stride,
                  void* y, int64_t y_stride, const int32_t* positions, int32_t tokens,
                  int32_t heads, int32_t head_dim, int32_t inverse, void* stream) {
  if (!dtype_ok(dtype) || head_dim <= 0 || head_dim % 8 != 0 || head_dim > 512 || heads <= 0 ||
      tokens < 0 || inverse < 0 || inverse > 1 || !rope_config_ok(rope, head_dim))
    return CB_ERR_INVALID_ARG;
  const int64_t width = (int64_t)heads * head_dim;
  if ((tokens > 0 && !positions) || !aligned(positions, 4) || width > INT_LIMIT ||
      !array_ok(x, tokens, x_stride, width) || !array_ok(y, tokens, y_stride, width))
    return CB_ERR_INVALID_ARG;
  if (tokens == 0) return CB_OK;
  if (!(x == y && x_stride == y_stride) &&
      arrays_overlap(x, x_stride, width, y, y_stride, width, tokens))
    return CB_ERR_INVALID_ARG;
  if (outputs_meet({token_span(y, tokens, y_stride, width)},
                   {Span{positions, tokens * 4ll}, Span{rope->inv_freq, rope->rot_dim * 4ll}}))
    return CB_ERR_INVALID_ARG;
  const cb_status s = check_device({x, y, positions, rope->inv_freq});
  if (s != CB_OK) return s;
  const int piece = rope->rot_dim % 16 == 0 && head_dim % 16 == 0 ? 8 : 4;
  // Heads of a thread: as many as leave half of the GPU's threads busy.
  const int64_t units = (int64_t)tokens * (head_dim / (2 * piece));
  const int64_t chunks_wanted = std::max<int64_t>(1, ceil_div((int64_t)PG_SMS * 1024, units));
  const int per_thread = (int)std::max<int64_t>(1, heads / std::min<int64_t>(heads, chunks_wanted));
  const int64_t blocks = ceil_div(units * ceil_div(heads, per_thread), ROPE_THREADS);
  if (blocks > INT_LIMIT) return CB_ERR_UNSUPPORTED;
  auto launch = [&](auto type, auto piece_of) {
    using T = decltype(type);
    rope_kernel<T, decltype(piece_of)::value>
        <<<(unsigned)blocks, ROPE_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(x), x_stride, static_cast<T*>(y), y_stride, positions,
            rope->inv_freq, rope->rot_dim, rope->layout == CB_ROPE_HALF, rope->amplitude,
            inverse ? -rope->amplitude : rope->amplitude, tokens, heads, head_dim, per_thread);
  };
  with_type(dtype, piece, launch);
  return status_of(cudaPeekAtLastError());
}

cb_status cb_paged_append(const cb_paged_kv* kv, const cb_rope_config* rope, int32_t heads,
                          const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride,
                          const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                          const int32_t* positions, float* weights, int32_t* slot_positions,
                          void* stream) {
  if (!kv_sizes_ok(kv) || !kv_pointers_ok(kv, true)) return CB_ERR_INVALID_ARG;
  if (rope && !rope_config_ok(rope, PG_HD)) return CB_ERR_INVALID_ARG;
  if (!q != !q_out || (q && !heads_ok(kv, heads))) return CB_ERR_INVALID_ARG;
  if (!q) heads = 0;
  const int64_t q_width = (int64_t)heads * PG_HD, kv_width = (int64_t)kv->kv_heads * PG_HD;
  const int64_t rows = kv->rows;
  if (q && (!array_ok(q, rows, q_stride, q_width) || !array_ok(q_out, rows, q_out_stride, q_width)))
    return CB_ERR_INVALID_ARG;
  if (!array_ok(k, rows, k_stride, kv_width) || !array_ok(v, rows, v_stride, kv_width) ||
      !aligned(positions, 4) || !aligned(weights, 4) || !aligned(slot_positions, 4))
    return CB_ERR_INVALID_ARG;
  if (rows == 0 || kv->max_new == 0) return CB_OK;
  if (q && !(q == q_out && q_stride == q_out_stride) &&
      arrays_overlap(q, q_stride, q_width, q_out, q_out_stride, q_width, rows))
    return CB_ERR_INVALID_ARG;
  if (q && (arrays_overlap(q_out, q_out_stride, q_width, k, k_stride, kv_width, rows) ||
            arrays_overlap(q_out, q_out_stride, q_width, v, v_stride, kv_width, rows)))
    return CB_ERR_INVALID_ARG;
  const Span q_out_span = q ? token_span(q_out, rows, q_out_stride, q_width) : Span{};
  const Span inv_freq{rope ? rope->inv_freq : nullptr, rope ? rope->rot_dim * 4ll : 0};
  const Span read[] = {table_span(kv), len_span(kv), row_start_span(kv),
                       Span{positions, rows * 4}, inv_freq};
  const Span tokens[] = {q ? token_span(q, rows, q_stride, q_width) : Span{},
                         token_span(k, rows, k_stride, kv_width),
                         token_span(v, rows, v_stride, kv_width)};
  const Span written[] = {pool_span(kv->k, kv), pool_span(kv->v, kv)};
  if (outputs_meet({q_out_span, meta_span(weights, kv), meta_span(slot_positions, kv)},
                   {read[0], read[1], read[2], read[3], read[4], written[0], written[1]}) ||
      outputs_meet({meta_span(weights, kv), meta_span(slot_positions, kv)},
                   {tokens[0], tokens[1], tokens[2]}) ||
      outputs_meet({written[0]}, {read[0], read[1], read[2], read[3], read[4]}) ||
      outputs_meet({written[1]}, {read[0], read[1], read[2], read[3], read[4]}))
    return CB_ERR_INVALID_ARG;
  const cb_status s =
      check_device({kv->k, kv->v, kv->table, kv->len, kv->row_start, rope ? rope->inv_freq : nullptr,
                    q, q_out, k, v, positions, weights, slot_positions});
  if (s != CB_OK) return s;
  const int all = heads + 2 * kv->kv_heads;
  const int rot = rope ? rope->rot_dim : 0;
  const int piece = rot % 16 == 0 ? 8 : 4;
  const int at_once = 32 / (PG_HD / (2 * piece));
  // Heads of a warp: as many as leave the GPU's warps three quarters busy (they share their
  // angles), a whole number of loads.
  const int64_t chunks_wanted = std::max<int64_t>(1, ceil_div((int64_t)PG_SMS * 48, rows));
  const int64_t heads_wanted = all / std::min<int64_t>(all, chunks_wanted);
  const int per_warp = (int)std::max<int64_t>(1, heads_wanted / at_once) * at_once;
  const int64_t blocks = ceil_div(rows * ceil_div(all, per_warp), APPEND_WARPS);
  if (blocks > INT_LIMIT) return CB_ERR_UNSUPPORTED;
  const PagedKV d = device_kv(kv);
  auto launch = [&](auto type, auto piece_of) {
    using T = decltype(type);
    paged_append_kernel<T, decltype(piece_of)::value>
        <<<(unsigned)blocks, APPEND_WARPS * 32, 0, static_cast<cudaStream_t>(stream)>>>(
            d, static_cast<const T*>(q), q_stride, static_cast<T*>(q_out), q_out_stride, heads,
            static_cast<const T*>(k), k_stride, static_cast<const T*>(v), v_stride, positions,
            rope ? rope->inv_freq : nullptr, rot, rope && rope->layout == CB_ROPE_HALF,
            rope ? rope->amplitude : 1.0f, weights, slot_positions, per_warp);
  };
  with_type(kv->dtype, piece, launch);
  return status_of(cudaPeekAtLastError());
}

cb_status cb_paged_attention_workspace(const cb_paged_kv* kv, int32_t heads, size_t* bytes) {
  if (!bytes || !kv_sizes_ok(kv) || !heads_ok(kv, heads)) return CB_ERR_INVALID_ARG;
  *bytes = plan_attention(kv, heads).bytes();
  return CB_OK;
}

}  // extern "C"

template <bool LOADS>
static cb_status paged_attention(const cb_paged_kv* kv, const void* q, int64_t q_stride,
                                 int32_t heads, float scale, void* out, int64_t out_stride,
                                 float* lse, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  if (!kv_sizes_ok(kv) || !kv_pointers_ok(kv, true) || !heads_ok(kv, heads))
    return CB_ERR_INVALID_ARG;
  const int64_t width = (int64_t)heads * PG_HD;
  if (!scale_ok(scale) || !array_ok(q, kv->rows, q_stride, width) ||
      !array_ok(out, kv->rows, out_stride, width) || !aligned(lse, 4) || !aligned(workspace, 16))
    return CB_ERR_INVALID_ARG;
  const size_t need = plan_attention(kv, heads).bytes();
  if (!workspace || workspace_bytes < need) return CB_ERR_INVALID_ARG;
  if (kv->rows == 0 || kv->max_new == 0) return CB_OK;
  if (arrays_overlap(q, q_stride, width, out, out_stride, width, kv->rows))
    return CB_ERR_INVALID_ARG;
  const Span lse_span{lse, (int64_t)kv->rows * heads * 4}, ws_span{workspace, (int64_t)need};
  const Span q_span = token_span(q, kv->rows, q_stride, width);
  if (outputs_meet({token_span(out, kv->rows, out_stride, width), lse_span, ws_span},
                   {pool_span(kv->k, kv), pool_span(kv->v, kv), table_span(kv), len_span(kv),
                    row_start_span(kv)}) ||
      outputs_meet({lse_span, ws_span}, {q_span}))
    return CB_ERR_INVALID_ARG;
  const cb_status s = check_device({kv->k, kv->v, kv->table, kv->len, kv->row_start, q, out, lse,
                                    workspace});
  if (s != CB_OK) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* ws = static_cast<float*>(workspace);
  if (kv->dtype == CB_DTYPE_F16)
    return launch_attention<__half, LOADS>(kv, static_cast<const __half*>(q), q_stride, heads,
                                           scale, static_cast<__half*>(out), out_stride, lse, ws,
                                           st);
  if constexpr (LOADS)
    return launch_attention<__nv_bfloat16, true>(kv, static_cast<const __nv_bfloat16*>(q), q_stride,
                                                 heads, scale, static_cast<__nv_bfloat16*>(out),
                                                 out_stride, lse, ws, st);
  return CB_ERR_UNSUPPORTED;
}

template <bool LOADS>
static cb_status paged_weights(const cb_paged_kv* kv, const void* q, int64_t q_stride,
                               int32_t heads, float scale, const float* lse, float* weights,
                               void* stream) {
  if (!kv_sizes_ok(kv) || !kv_pointers_ok(kv, true) || !heads_ok(kv, heads))
    return CB_ERR_INVALID_ARG;
  if (!scale_ok(scale) || !array_ok(q, kv->rows, q_stride, (int64_t)heads * PG_HD) ||
      (kv->rows > 0 && !lse) || !weights || !aligned(lse, 4) || !aligned(weights, 4))
    return CB_ERR_INVALID_ARG;
  if (kv->rows == 0 || kv->max_new == 0) return CB_OK;
  if (outputs_meet({meta_span(weights, kv)},
                   {pool_span(kv->k, kv), table_span(kv), len_span(kv), row_start_span(kv),
                    token_span(q, kv->rows, q_stride, (int64_t)heads * PG_HD),
                    Span{lse, (int64_t)kv->rows * heads * 4}}))
    return CB_ERR_INVALID_ARG;
  const cb_status s =
      check_device({kv->k, kv->table, kv->len, kv->row_start, q, lse, weights});
  if (s != CB_OK) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (kv->dtype == CB_DTYPE_F16)
    return launch_weights<__half, LOADS>(kv, static_cast<const __half*>(q), q_stride, heads, scale,
                                         lse, weights, st);
  if constexpr (LOADS)
    return launch_weights<__nv_bfloat16, true>(kv, static_cast<const __nv_bfloat16*>(q), q_stride,
                                               heads, scale, lse, weights, st);
  return CB_ERR_UNSUPPORTED;
}

extern "C" {

cb_status cb_paged_attention(const cb_paged_kv* kv, const void* q, int64_t q_stride,
                             int32_t heads, float scale, void* out, int64_t out_stride,
                             float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  return paged_attention<true>(kv, q, q_stride, heads, scale, out, out_stride, lse, workspace,
                               workspace_bytes, stream);
}

cb_status cb_paged_attention_weights(const cb_paged_kv* kv, const void* q, int64_t q_stride,
                                     int32_t heads, float scale, const float* lse,
                                     float* weights, void* stream) {
  return paged_weights<true>(kv, q, q_stride, heads, scale, lse, weights, stream);
}

cb_status cb_paged_check_device_error(int32_t* expired, void* stream) {
  if (!expired) return CB_ERR_INVALID_ARG;
  cb_status s = check_device({});
  if (s != CB_OK) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  *expired = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(expired, paged_expired, sizeof(int32_t), 0,
                                            cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && *expired != 0) {
    const int none = 0;
    e = cudaMemcpyToSymbolAsync(paged_expired, &none, sizeof(none), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    s = CB_ERR_DEVICE_TIMEOUT;
  }
  return e == cudaSuccess ? s : status_of(e);
}

cb_status cb_selftest_paged_timeout(const cb_paged_kv* kv, const void* q, int64_t q_stride,
                                    int32_t heads, float scale, void* out, int64_t out_stride,
                                    float* lse, float* weights, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  const cb_status s = paged_weights<false>(kv, q, q_stride, heads, scale, lse, weights, stream);
  if (s != CB_OK) return s;
  return paged_attention<false>(kv, q, q_stride, heads, scale, out, out_stride, lse, workspace,
                                workspace_bytes, stream);
}

static size_t evict_list(const cb_paged_kv* kv, int32_t budget) {
  return (size_t)std::min(budget, kv->max_len);
}

cb_status cb_paged_evict_workspace(const cb_paged_kv* kv, int32_t budget, size_t* bytes) {
  if (!bytes || !kv_sizes_ok(kv) || budget <= 0) return CB_ERR_INVALID_ARG;
  *bytes = (size_t)kv->batch * kv->kv_heads * 2 * evict_list(kv, budget) * sizeof(int32_t);
  return CB_OK;
}

cb_status cb_paged_evict(const cb_paged_kv* kv, const float* weights, float* weights_out,
                         const int32_t* positions, int32_t* positions_out,
                         const int32_t* next_position, int32_t budget, int32_t sinks,
                         int32_t recent, int32_t* len_out, void* workspace,
                         size_t workspace_bytes, void* stream) {
  if (!kv_sizes_ok(kv) || !kv_pointers_ok(kv, false)) return CB_ERR_INVALID_ARG;
  if (!weights || !weights_out || !positions || !positions_out || !next_position || !len_out ||
      !workspace || budget <= 0 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
    return CB_ERR_INVALID_ARG;
  if (!aligned(weights, 4) || !aligned(weights_out, 4) || !aligned(positions, 4) ||
      !aligned(positions_out, 4) || !aligned(next_position, 4) || !aligned(len_out, 4) ||
      !aligned(workspace, 16))
    return CB_ERR_INVALID_ARG;
  size_t need = 0;
  cb_paged_evict_workspace(kv, budget, &need);
  if (workspace_bytes < need) return CB_ERR_INVALID_ARG;
  const Span w_in = meta_span(weights, kv), p_in = meta_span(positions, kv);
  const Span w_out = meta_span(weights_out, kv), p_out = meta_span(positions_out, kv);
  const Span lens_out{len_out, kv->batch * 4ll}, ws{workspace, (int64_t)need};
  const Span next{next_position, kv->batch * 4ll};
  if ((weights != weights_out && outputs_meet({w_out}, {w_in})) ||
      (positions != positions_out && outputs_meet({p_out}, {p_in})) ||
      outputs_meet({w_out}, {p_in}) || outputs_meet({p_out}, {w_in}) ||
      outputs_meet({lens_out, ws}, {w_in, p_in}) ||
      outputs_meet({w_out, p_out, lens_out, ws},
                   {len_span(kv), table_span(kv), next, pool_span(kv->k, kv),
                    pool_span(kv->v, kv)}) ||
      outputs_meet({pool_span(kv->k, kv)}, {w_in, p_in, len_span(kv), table_span(kv), next}) ||
      outputs_meet({pool_span(kv->v, kv)}, {w_in, p_in, len_span(kv), table_span(kv), next}))
    return CB_ERR_INVALID_ARG;
  if (kv->max_len > EV_MAX_LEN) return CB_ERR_UNSUPPORTED;
  const cb_status s = check_device({kv->k, kv->v, kv->table, kv->len, weights, weights_out,
                                    positions, positions_out, next_position, len_out, workspace});
  if (s != CB_OK) return s;
  const int64_t items = (int64_t)kv->batch * kv->kv_heads;
  if (items * EV_MAX_CTAS > INT_LIMIT) return CB_ERR_UNSUPPORTED;
  const PagedKV d = device_kv(kv);
  const EvictArgs a{weights, weights_out, positions, positions_out, next_position, budget, sinks,
                    recent, len_out, static_cast<int*>(workspace), (int)evict_list(kv, budget)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // The smallest form that holds the longest sequence; long ones are spread over a cluster.
  const int n = kv->max_len;
  cudaError_t e;
  if (n <= 128 * 8)
    e = launch_evict<128, 8>(d, a, 1, st);
  else if (n <= 512 * 8)
    e = launch_evict<512, 8>(d, a, 1, st);
  else if (n <= 512 * 8 * 2)
    e = launch_evict<512, 8>(d, a, 2, st);
  else if (n <= 512 * 8 * 4)
    e = launch_evict<512, 8>(d, a, 4, st);
  else if (n <= 512 * 8 * 8)
    e = launch_evict<512, 8>(d, a, 8, st);
  else
    e = launch_evict<EV_MAX_THREADS, EV_MAX_PER_THREAD>(d, a, EV_MAX_CTAS, st);
  return status_of(e);
}

}  // extern "C"
