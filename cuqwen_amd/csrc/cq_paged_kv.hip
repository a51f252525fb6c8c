// Rows of K and V into and out of the pages of a paged KV cache (cq_kv_pages).
//
// What bounds it: the launch.  A step's rows of a batch are some ten KB, a prompt's
// chunk a few MB; the scattered stores of V (whose tiles keep 4 consecutive tokens of
// a dimension together) are written as 16-byte pieces where a block's tokens fill a
// tile, else as single elements.  2048 rows of 1.5B heads, fp16: 4.2 us (4.2 MB moved); 64
// scattered rows of 7B heads, int8: 2.4 us, and 3.5 to read them back.
#include "cq_attention.h"
#include "cq_pages.h"

#include <algorithm>

namespace cq {

namespace {

constexpr int kRowThreads = 256;

struct RowArgs {
  PageView pv;
  int64_t layer_off;        // layer * layer_stride
  const _Float16* x[2];     // store: K and V rows; load: unused
  _Float16* y[2];           // load
  int64_t row_stride;
  const int* slots;
  int n_tokens, n_kv;
  int n_slots;              // slots of the pool
};

// Element offset of slot `slot`'s page in head h.
__device__ __forceinline__ int64_t page_off(const RowArgs& a, int slot, int h) {
  return a.layer_off + (int64_t)(slot >> a.pv.shift) * a.pv.page_stride + (int64_t)h * a.pv.head_stride;
}
// Offsets within a page of one head (the layout functions with kv head 0).
__device__ __forceinline__ int in_page(int kind, int t, int d, int hd) {
  return (int)(kind ? kv_v_offset(0, t, d, 0, hd) : kv_k_offset(0, t, d, 0, hd));
}
__device__ __forceinline__ int in_page8(int kind, int t, int d, int hd) {
  return (int)(kind ? kv8_v_offset(0, t, d, 0, hd) : kv8_k_offset(0, t, d, 0, hd));
}

// fp16: block = (32 tokens, kv head, K or V).  K goes in its 16-byte pieces of 8
// dimensions; V through LDS, so that a piece's 8 keys meet.
template <int HD>
__global__ __launch_bounds__(kRowThreads) void store_rows_kernel(RowArgs a) {
  constexpr int P8 = HD / 8, PAD = HD + 8;
  __shared__ __align__(16) _Float16 tile[32 * PAD];
  __shared__ int slot[32], whole;
  const int t0 = blockIdx.x * 32, h = blockIdx.y, kind = blockIdx.z, n = min(32, a.n_tokens - t0);
  const int mask = (1 << a.pv.shift) - 1;
  _Float16* base = (_Float16*)a.pv.kv[kind];
  if (threadIdx.x < 32) slot[threadIdx.x] = threadIdx.x < n ? a.slots[t0 + threadIdx.x] : -1;
  const _Float16* x = a.x[kind] + (int64_t)t0 * a.row_stride + h * HD;
  constexpr int PER = 32 * P8 / kRowThreads;   // pieces per thread: 1 or 2
  h8_t v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = i * kRowThreads + threadIdx.x, t = c / P8, p = c % P8;
    v[i] = t < n ? *reinterpret_cast<const h8_t*>(x + (int64_t)t * a.row_stride + 8 * p) : h8_t{0, 0, 0, 0, 0, 0, 0, 0};
  }
  __syncthreads();
  if (kind == 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = i * kRowThreads + threadIdx.x, t = c / P8, p = c % P8, s = slot[t];
      if ((unsigned)s < (unsigned)a.n_slots) *reinterpret_cast<h8_t*>(base + page_off(a, s, h) + in_page(0, s & mask, 8 * p, HD)) = v[i];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = i * kRowThreads + threadIdx.x;
    *reinterpret_cast<h8_t*>(tile + c / P8 * PAD + 8 * (c % P8)) = v[i];
  }
  if (threadIdx.x < kWave) {
    const int s = slot[threadIdx.x & 31], s0 = slot[0];
    const bool all = __all(s0 >= 0 && (s0 & 31) == 0 && s == s0 + (int)(threadIdx.x & 31) && s < a.n_slots);
    if (threadIdx.x == 0) whole = all;
  }
  __syncthreads();
  if (whole) {   // one tile of one page
    _Float16* dst = base + page_off(a, slot[0], h) + in_page(1, slot[0] & mask, 0, HD);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = i * kRowThreads + threadIdx.x, dt = c / kWave, j = c % kWave / 16, dl = c % 16;
      h8_t o;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = tile[(e < 4 ? 4 * j + e : 12 + 4 * j + e) * PAD + dt * 16 + dl];
      *reinterpret_cast<h8_t*>(dst + c * 8) = o;
    }
    return;
  }
  for (int c = threadIdx.x; c < n * HD; c += kRowThreads) {
    const int t = c / HD, d = c % HD, s = slot[t];
    if ((unsigned)s < (unsigned)a.n_slots) base[page_off(a, s, h) + in_page(1, s & mask, d, HD)] = tile[t * PAD + d];
  }
}

// One-byte codes: a wave per (token, kv head, K or V) row, as the decode step
// quantizes its new row.
template <int HD, int F>
__global__ __launch_bounds__(kRowThreads) void store_rows8_kernel(RowArgs a) {
  constexpr int E = HD / kWave;
  const int lane = threadIdx.x & (kWave - 1);
  const int t = blockIdx.x * (kRowThreads / kWave) + threadIdx.x / kWave, h = blockIdx.y, kind = blockIdx.z;
  if (t >= a.n_tokens) return;
  const int s = a.slots[t];
  if ((unsigned)s >= (unsigned)a.n_slots) return;
  const _Float16* x = a.x[kind] + (int64_t)t * a.row_stride + h * HD + lane * E;
  float f[E];
  int8_t q[E];
#pragma unroll
  for (int i = 0; i < E; ++i) f[i] = (float)x[i];
  const float sc = quant_row8_wave<HD, F>(f, q);
  const int64_t at = page_off(a, s, h);
  const int ts = s & ((1 << a.pv.shift) - 1);
#pragma unroll
  for (int i = 0; i < E; ++i) a.pv.kv[kind][at + in_page8(kind, ts, lane * E + i, HD)] = (char)q[i];
  if (lane == 0) a.pv.scale[kind][at / HD + ts] = sc;
}

// A thread per (token, kv head, 8 dimensions) of K and of V.
template <int HD, int F>
__global__ __launch_bounds__(kRowThreads) void load_rows_kernel(RowArgs a) {
  constexpr int P8 = HD / 8;
  const int c = blockIdx.x * kRowThreads + threadIdx.x, p = c % P8, t = c / P8, h = blockIdx.y;
  if (t >= a.n_tokens) return;
  const int s = a.slots[t];
  if ((unsigned)s >= (unsigned)a.n_slots) return;
  const int64_t at = page_off(a, s, h);
  const int ts = s & ((1 << a.pv.shift) - 1);
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    h8_t v;
    if constexpr (F == CQ_KV_FP16) {
      const _Float16* src = (const _Float16*)a.pv.kv[kind] + at;
      if (kind == 0) v = *reinterpret_cast<const h8_t*>(src + in_page(0, ts, 8 * p, HD));
      else
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = src[in_page(1, ts, 8 * p + e, HD)];
    } else {
      const float sc = a.pv.scale[kind][at / HD + ts];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int8_t q = (int8_t)a.pv.kv[kind][at + in_page8(kind, ts, 8 * p + e, HD)];
        v[e] = (_Float16)((F == CQ_KV_FP8 ? e4m3_value((uint8_t)q) : (float)q) * sc);
      }
    }
    *reinterpret_cast<h8_t*>(a.y[kind] + (int64_t)t * a.row_stride + h * HD + 8 * p) = v;
  }
}

int rows_check(const cq_kv_pages* p, int layer, const void* k, const void* v, int64_t row_stride, const int32_t* d_slots, int n) {
  CQ_TRY(pages_check(p));
  if (layer < 0 || layer >= p->n_layers) return fail(CQ_EINVAL, "paged rows: layer outside the pool");
  if (n < 0 || n > (1 << 24)) return fail(CQ_EINVAL, "paged rows: n_tokens outside [0, 2^24]");
  if (n == 0) return CQ_OK;
  if (!k || !v || !d_slots || unaligned16(k) || unaligned16(v)) return fail(CQ_EINVAL, "paged rows: k and v must be set and aligned to 16 bytes");
  if (row_stride < (int64_t)p->n_kv_heads * p->head_dim || row_stride % 8 || row_stride > ((int64_t)1 << 36))
    return fail(CQ_EINVAL, "paged rows: row_stride must be a multiple of 8 that holds a row");
  return CQ_OK;
}

RowArgs row_args(const cq_kv_pages& p, int layer, int64_t row_stride, const int32_t* d_slots, int n) {
  RowArgs a{};
  a.pv = page_view(p);
  a.layer_off = layer * p.layer_stride;
  a.row_stride = row_stride;
  a.slots = d_slots;
  a.n_tokens = n; a.n_kv = p.n_kv_heads;
  a.n_slots = p.n_pages * p.page_tokens;
  return a;
}

// Blocks for `per` threads of each token (n_tokens * per below 2^31).
unsigned blocks_for(int n_tokens, int per) { return (unsigned)(((int64_t)n_tokens * per + kRowThreads - 1) / kRowThreads); }

template <int HD>
void launch_store(const RowArgs& a, int fmt, hipStream_t st) {
  if (fmt == CQ_KV_FP16) {
    hipLaunchKernelGGL(store_rows_kernel<HD>, dim3((a.n_tokens + 31) / 32, a.n_kv, 2), dim3(kRowThreads), 0, st, a);
    return;
  }
  const dim3 grid(blocks_for(a.n_tokens, kWave), a.n_kv, 2);
  if (fmt == CQ_KV_INT8) hipLaunchKernelGGL((store_rows8_kernel<HD, CQ_KV_INT8>), grid, dim3(kRowThreads), 0, st, a);
  else hipLaunchKernelGGL((store_rows8_kernel<HD, CQ_KV_FP8>), grid, dim3(kRowThreads), 0, st, a);
}

template <int HD>
void launch_load(const RowArgs& a, int fmt, hipStream_t st) {
  const dim3 grid(blocks_for(a.n_tokens, HD / 8), a.n_kv);
  if (fmt == CQ_KV_FP16) hipLaunchKernelGGL((load_rows_kernel<HD, CQ_KV_FP16>), grid, dim3(kRowThreads), 0, st, a);
  else if (fmt == CQ_KV_INT8) hipLaunchKernelGGL((load_rows_kernel<HD, CQ_KV_INT8>), grid, dim3(kRowThreads), 0, st, a);
  else hipLaunchKernelGGL((load_rows_kernel<HD, CQ_KV_FP8>), grid, dim3(kRowThreads), 0, st, a);
}

}  // namespace

}  // namespace cq

using namespace cq;

extern "C" int cq_paged_kv_store(const cq_kv_pages* pages, int32_t layer, const void* k, const void* v,
                                 int64_t row_stride, const int32_t* d_slots, int32_t n_tokens, void* stream) {
  CQ_TRY(rows_check(pages, layer, k, v, row_stride, d_slots, n_tokens));
  if (n_tokens == 0) return CQ_OK;
  RowArgs a = row_args(*pages, layer, row_stride, d_slots, n_tokens);
  a.x[0] = (const _Float16*)k; a.x[1] = (const _Float16*)v;
  if (pages->head_dim == 128) launch_store<128>(a, pages->kv_dtype, (hipStream_t)stream);
  else launch_store<64>(a, pages->kv_dtype, (hipStream_t)stream);
  CQ_HIP(hipGetLastError());
  return CQ_OK;
}

extern "C" int cq_paged_kv_load(const cq_kv_pages* pages, int32_t layer, void* k, void* v, int64_t row_stride,
                                const int32_t* d_slots, int32_t n_tokens, void* stream) {
  CQ_TRY(rows_check(pages, layer, k, v, row_stride, d_slots, n_tokens));
  if (n_tokens == 0) return CQ_OK;
  RowArgs a = row_args(*pages, layer, row_stride, d_slots, n_tokens);
  a.y[0] = (_Float16*)k; a.y[1] = (_Float16*)v;
  if (pages->head_dim == 128) launch_load<128>(a, pages->kv_dtype, (hipStream_t)stream);
  else launch_load<64>(a, pages->kv_dtype, (hipStream_t)stream);
  CQ_HIP(hipGetLastError());
  return CQ_OK;
}
