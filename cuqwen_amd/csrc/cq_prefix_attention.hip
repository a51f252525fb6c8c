// Decode attention of a batch whose sequences share a prefix, over paged caches
// (cq_kv_pages): the prefix's K and V are read for all rows of a kv head together,
// each sequence's own pages for its own rows.  No counterpart in the reference.
//
// For row (b, head h of kv head kvh): s_t = q . k_t / sqrt(hd) over the prefix's and
// the sequence's own positions, out = sum exp(s_t - m) v_t / sum exp(s_t - m), formed
// in pieces: each piece of keys leaves (m, l, O) in fp32, and a second launch joins the
// pieces of a row by the log-sum-exp rule.
//
// Work: 32-key tiles of (item, tile), an item being (kv head, 16 query rows) of the
// prefix or (sequence, kv head) of the own part.  All tiles of all items form one
// list that the waves of the grid share evenly (share_of), wherever item borders fall, from the
// lengths found on the device: lengths may be ragged, and a captured launch serves
// other lengths.  Wave w's piece of item i is stored in slot w + i (either w or i grows from one piece to the next, so slots
// differ), and the joining launch finds a row's pieces by the same arithmetic.
#include "cq_attention.h"
#include "cq_pages.h"

#include <algorithm>
#include <cmath>

namespace cq {

namespace {

constexpr int kPxWaves = 8, kPxThreads = kPxWaves * kWave;
constexpr int kPxBlocks = kNumCUs;                    // one block per CU
constexpr int kPxListWaves = kPxBlocks * kPxWaves;    // W of the own list
constexpr int kPxMaxBatch = 1024;
constexpr float kLog2e = 1.4426950408889634f;

struct PxArgs {
  const _Float16* q;
  _Float16* out;
  int64_t q_stride, out_stride;
  PageView pre, own;
  int64_t pre_layer, own_layer;   // element offset of the layer
  const int* pre_table;
  const int* pre_len;
  const int* table;
  const int* start;
  const int* len;
  int pre_pages, max_pages;
  int batch, n_kv, g;
  // workspace
  int64_t* plan;                  // [batch + 1] own tiles before each sequence, then the prefix's tiles
  float* own_o;                   // [slot][16][HD]
  float* own_ml;                  // [slot][16][2]
  float* pre_o;
  float* pre_ml;
};

// Range [first, end) of worker w when F tiles are shared by W workers (the first F
// workers, a tile each, if there are fewer tiles): F w / W, F (w + 1) / W.
__device__ __forceinline__ void share_of(int w, int64_t F, int W, int64_t* first, int64_t* end) {
  *first = F <= W ? min((int64_t)w, F) : F * w / W;
  *end = F <= W ? min((int64_t)w + 1, F) : F * (w + 1) / W;
}
// The worker that has tile x.
__device__ __forceinline__ int worker_of(int64_t x, int64_t F, int W) { return (int)(F <= W ? x : ((x + 1) * W - 1) / F); }

// Positions that a table of n pages holds, and the length cut there.
__device__ __forceinline__ int cut_len(int len, int pages, int shift) {
  return min(max(len, 0), (int)min((int64_t)pages << shift, (int64_t)0x7fffffff));
}

// One kv head of a paged cache as a wave's tiles see it.
struct PxKV {
  PageView pv;
  int64_t off;       // elements: layer and head
  const int* table;  // page of each run of page_tokens positions
};

// The K and V of one 32-key tile in matrix operand order, and where its keys are valid.
template <int HD, int F>
struct PxTile {
  u4_t k[F == CQ_KV_FP16 ? HD / 16 : HD / 32], v[F == CQ_KV_FP16 ? HD / 16 : HD / 32];
  f4_t ks[F == CQ_KV_FP16 ? 1 : 2], vs[F == CQ_KV_FP16 ? 1 : 2];
  int lo, hi;        // valid keys of the tile: [lo, hi)
};

// Requests tile ti (positions [32 ti, 32 ti + 32) cut to [lo, hi)); with `want` false,
// or a page outside the pool, nothing is read and no key is valid.
template <int HD, int F>
__device__ __forceinline__ void px_load(PxTile<HD, F>& t, const PxKV& kv, int ti, int lo, int hi, bool want, int lane) {
  constexpr int ES = F == CQ_KV_FP16 ? 2 : 1, N = F == CQ_KV_FP16 ? HD / 16 : HD / 32;
  const int s5 = kv.pv.shift - 5;
  int page = want ? (int)load_ctl_u32(kv.table + (ti >> s5)) : -1;
  page = __builtin_amdgcn_readfirstlane(page);
  const bool ok = page >= 0 && page < kv.pv.n_pages;
  const int64_t at = kv.off + (int64_t)(ok ? page : 0) * kv.pv.page_stride + (int64_t)(ti & ((1 << s5) - 1)) * (32 * HD);
  const int n = ok ? 32 * HD * ES : 0;
  const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(kv.pv.kv[0] + at * ES, (short)0, n, kBufWord3);
  const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(kv.pv.kv[1] + at * ES, (short)0, n, kBufWord3);
#pragma unroll
  for (int i = 0; i < N; ++i) t.k[i] = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(rk, i * 1024 + lane * 16, 0, 0));
#pragma unroll
  for (int i = 0; i < N; ++i) t.v[i] = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(rv, i * 1024 + lane * 16, 0, 0));
  if constexpr (F != CQ_KV_FP16) {
    const int j = lane >> 4;
    const __amdgpu_buffer_rsrc_t rks = __builtin_amdgcn_make_buffer_rsrc(kv.pv.scale[0] + at / HD, (short)0, ok ? 128 : 0, kBufWord3);
    const __amdgpu_buffer_rsrc_t rvs = __builtin_amdgcn_make_buffer_rsrc(kv.pv.scale[1] + at / HD, (short)0, ok ? 128 : 0, kBufWord3);
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      t.ks[st] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(rks, (st * 16 + 4 * j) * 4, 0, 0));
      t.vs[st] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(rvs, (st * 16 + 4 * j) * 4, 0, 0));
    }
  }
  t.lo = ok ? lo - 32 * ti : 0;
  t.hi = ok ? hi - 32 * ti : 0;
}

// Operand i of a tile's K (or V) as fp16.
template <int F>
__device__ __forceinline__ h8_t px_operand(const u4_t* w, int i, uint32_t magic) {
  if constexpr (F == CQ_KV_FP16) return __builtin_bit_cast(h8_t, w[i]);
  else return codes_to_h8<F>(i & 1 ? u2_t{w[i / 2].z, w[i / 2].w} : u2_t{w[i / 2].x, w[i / 2].y}, magic);
}

// A wave's running softmax over 16 query columns: lane (h, j) holds column h, dims
// dt * 16 + 4 j + i.  One-byte V: P is rounded to fp16 as p * scale / r, r the power of
// two at or below the largest V scale seen (so that small scales do not drive the
// products into fp16's subnormals), and O is kept in units of r.
template <int HD>
struct PxState {
  float m, l, r;
  f4_t o[HD / 16];
};

template <int HD, int F>
__device__ __forceinline__ void px_attend(PxTile<HD, F>& t, const h8_t* qb, PxState<HD>& st, float c2, int lane, uint32_t magic) {
  constexpr int KK = HD / 32, DT = HD / 16;
  const int j = lane >> 4;
  f4_t s[2];
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    s[a] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
      s[a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(px_operand<F>(t.k, a * KK + kk, magic), qb[kk], s[a], 0, 0, 0);
  }
  if constexpr (F != CQ_KV_FP16) {
#pragma unroll
    for (int a = 0; a < 2; ++a) s[a] *= t.ks[a];
  }
  const bool part = t.lo > 0 || t.hi < 32;   // wave-uniform
  if (part) {
    // masked keys may hold anything, in V too: a weight of 0 does not silence a NaN
    uint32_t keep[F == CQ_KV_FP16 ? 4 : 2] = {};   // of an operand's 8 keys
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int key = (e >> 2) * 16 + 4 * j + (e & 3);
      const bool in = key >= t.lo && key < t.hi;
      s[e >> 2][e & 3] = in ? s[e >> 2][e & 3] : -INFINITY;
      if constexpr (F != CQ_KV_FP16) {
        t.vs[e >> 2][e & 3] = in ? t.vs[e >> 2][e & 3] : 0.f;
        keep[e >> 2] |= in ? 0xffu << (8 * (e & 3)) : 0u;
      } else {
        keep[e >> 1] |= in ? 0xffffu << (16 * (e & 1)) : 0u;
      }
    }
    constexpr int N = sizeof(t.v) / sizeof(t.v[0]);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if constexpr (F != CQ_KV_FP16) t.v[n] &= u4_t{keep[0], keep[1], keep[0], keep[1]};
      else t.v[n] &= u4_t{keep[0], keep[1], keep[2], keep[3]};
    }
  }
  float mn = st.m;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int i = 0; i < 4; ++i) mn = fmaxf(mn, s[a][i]);
  mn = fmaxf(mn, __shfl_xor(mn, 16, kWave));
  mn = fmaxf(mn, __shfl_xor(mn, 32, kWave));
  float rn = st.r;
  if constexpr (F != CQ_KV_FP16) {
    float vm = 0.f;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int i = 0; i < 4; ++i) vm = fmaxf(vm, t.vs[a][i]);
    vm = fmaxf(vm, __shfl_xor(vm, 16, kWave));
    vm = fmaxf(vm, __shfl_xor(vm, 32, kWave));
    rn = fmaxf(rn, __uint_as_float(__float_as_uint(vm) & 0x7f800000u));
  }
  if (__any(mn > st.m || rn > st.r)) {
    const float alpha = mn == st.m ? 1.f : __builtin_amdgcn_exp2f((st.m - mn) * c2);
    const float beta = F != CQ_KV_FP16 ? alpha * (st.r / rn) : alpha;
    st.m = mn;
    st.r = rn;
    st.l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) st.o[dt] *= beta;
  }
  const float mm = st.m == -INFINITY ? 0.f : st.m * c2;   // no valid key yet: the masked ones give 0
  const float ri = F != CQ_KV_FP16 ? 1.f / st.r : 1.f;
  h8_t pb;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s[a][i], c2, -mm));
      st.l += p;
      // fp16: half a step of 2^-11 of each weight, while the sum keeps them whole
      pb[a * 4 + i] = (_Float16)(F != CQ_KV_FP16 ? p * (t.vs[a][i] * ri) : p);
    }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) st.o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(px_operand<F>(t.v, dt, magic), pb, st.o[dt], 0, 0, 0);
}

// Tiles [ta, tb) of one cache for the rows q[r0 .. r0 + rows) of a kv head; the
// state goes to (o, ml).
template <int HD, int F>
__device__ __forceinline__ void px_piece(const PxArgs& a, const PxKV& kv, int kvh, int r0, int rows, int lo, int hi, int ta, int tb,
                                         float* o, float* ml, int lane) {
  constexpr int KK = HD / 32, DT = HD / 16;
  const int h = lane & 15, j = lane >> 4;
  const float c2 = kLog2e / sqrtf((float)HD);
  const uint32_t magic = vgpr_const(0x64646464u);
  PxTile<HD, F> A, B;
  px_load<HD, F>(A, kv, ta, lo, hi, true, lane);
  h8_t qb[KK];
  const int r = r0 + min(h, rows - 1), b = r / a.g;
  const _Float16* q = a.q + b * a.q_stride + (kvh * a.g + (r - b * a.g)) * HD;
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) qb[kk] = __builtin_bit_cast(h8_t, load_u4(q + kk * 32 + j * 8));
  PxState<HD> st;
  st.m = -INFINITY;
  st.l = 0.f;
  st.r = 0x1p-100f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) st.o[dt] = f4_t{0.f, 0.f, 0.f, 0.f};
  for (int ti = ta; ti < tb; ti += 2) {
    px_load<HD, F>(B, kv, ti + 1, lo, hi, ti + 1 < tb, lane);
    px_attend<HD, F>(A, qb, st, c2, lane, magic);
    if (ti + 1 >= tb) break;
    px_load<HD, F>(A, kv, ti + 2, lo, hi, ti + 2 < tb, lane);
    px_attend<HD, F>(B, qb, st, c2, lane, magic);
  }
  st.l += __shfl_xor(st.l, 16, kWave);
  st.l += __shfl_xor(st.l, 32, kWave);
  if (h < rows) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f4_t*>(o + h * HD + dt * 16 + 4 * j) = F != CQ_KV_FP16 ? st.o[dt] * st.r : st.o[dt];
    if (j == 0) {
      ml[2 * h] = st.m * c2;   // log2 units from here on
      ml[2 * h + 1] = st.l;
    }
  }
}

template <int HD, int F>
__global__ __launch_bounds__(kPxThreads) void px_stage1(const PxArgs a) {
  __shared__ int64_t cum[kPxMaxBatch + 1];
  __shared__ int64_t part[kPxWaves];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lp = cut_len((int)load_ctl_u32(a.pre_len), a.pre_pages, a.pre.shift);
  const int lo = a.start ? max((int)load_ctl_u32(a.start), 0) : 0;
  // own tiles before each sequence
  int64_t n2[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int b = 2 * threadIdx.x + i, hi = b < a.batch ? cut_len(a.len[b], a.max_pages, a.own.shift) : 0;
    n2[i] = hi > lo ? (int64_t)((hi - 1) >> 5) - (lo >> 5) + 1 : 0;
  }
  int64_t x = n2[0] + n2[1];
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int64_t y = __shfl_up(x, o, kWave);
    if (lane >= o) x += y;
  }
  if (lane == kWave - 1) part[wave] = x;
  __syncthreads();
  for (int w = 0; w < wave; ++w) x += part[w];
  cum[2 * threadIdx.x + 1] = x - n2[1];
  cum[2 * threadIdx.x + 2] = x;
  if (threadIdx.x == 0) cum[0] = 0;
  __syncthreads();
  const int ptiles = (lp + 31) >> 5;
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b <= a.batch; b += kPxThreads) a.plan[b] = cum[b];
    if (threadIdx.x == 0) a.plan[a.batch + 1] = ptiles;
  }
  const int w = blockIdx.x * kPxWaves + wave;
  {
    const int R = a.batch * a.g, n_rg = (R + 15) / 16;
    const int64_t F_ = (int64_t)a.n_kv * n_rg * ptiles;
    int64_t at, end;
    share_of(w, F_, kPxListWaves, &at, &end);
    while (at < end) {
      const int item = (int)(at / ptiles), ta = (int)(at - (int64_t)item * ptiles), kvh = item / n_rg, rg = item % n_rg;
      const int tb = (int)min((int64_t)ptiles, ta + (end - at));
      const PxKV kv{a.pre, a.pre_layer + kvh * a.pre.head_stride, a.pre_table};
      px_piece<HD, F>(a, kv, kvh, rg * 16, min(16, R - rg * 16), 0, lp, ta, tb, a.pre_o + (int64_t)(w + item) * 16 * HD,
                      a.pre_ml + (int64_t)(w + item) * 32, lane);
      at += tb - ta;
    }
  }
  {
    const int64_t F_ = cum[a.batch] * a.n_kv;
    int64_t at, end;
    share_of(w, F_, kPxListWaves, &at, &end);
    while (at < end) {
      int b = 0, top = a.batch;   // last b with n_kv * cum[b] <= at
      while (top - b > 1) {
        const int mid = (b + top) / 2;
        if (cum[mid] * a.n_kv <= at) b = mid; else top = mid;
      }
      b = __builtin_amdgcn_readfirstlane(b);
      const int nt = (int)(cum[b + 1] - cum[b]);
      const int64_t in = at - cum[b] * a.n_kv;
      const int kvh = (int)(in / nt), ta = (int)(in - (int64_t)kvh * nt), item = b * a.n_kv + kvh;
      const int tb = (int)min((int64_t)nt, ta + (end - at));
      const int hi = cut_len((int)load_ctl_u32(a.len + b), a.max_pages, a.own.shift), t0 = lo >> 5;
      const PxKV kv{a.own, a.own_layer + kvh * a.own.head_stride, a.table + (int64_t)b * a.max_pages};
      px_piece<HD, F>(a, kv, kvh, b * a.g, a.g, lo, hi, t0 + ta, t0 + tb, a.own_o + (int64_t)(w + item) * 16 * HD,
                      a.own_ml + (int64_t)(w + item) * 32, lane);
      at += tb - ta;
    }
  }
}

// Joins the pieces of one row (b, head): a block of HD / 4 threads per piece group.
constexpr int kPxMergeThreads = 256;

template <int HD>
__global__ __launch_bounds__(kPxMergeThreads) void px_merge(const PxArgs a) {
  constexpr int TP = HD / 4, G = kPxMergeThreads / TP;   // threads of a piece, pieces at a time
  __shared__ f4_t so[G][TP];
  __shared__ float sm[G], sl[G];
  const int b = blockIdx.x / (a.n_kv * a.g), head = blockIdx.x % (a.n_kv * a.g), kvh = head / a.g, hh = head - kvh * a.g;
  if ((int)load_ctl_u32(a.len + b) < 0) return;
  const int R = a.batch * a.g, n_rg = (R + 15) / 16, row = b * a.g + hh;
  const int64_t ptiles = a.plan[a.batch + 1], c0 = a.plan[b], c1 = a.plan[b + 1], all = a.plan[a.batch] * a.n_kv;
  int n_pre = 0, n_own = 0;
  const float *po = nullptr, *pml = nullptr, *oo = nullptr, *oml = nullptr;
  if (ptiles > 0) {
    const int item = kvh * n_rg + row / 16;
    const int64_t F = a.n_kv * n_rg * ptiles, x0 = item * ptiles;
    const int w0 = worker_of(x0, F, kPxListWaves);
    n_pre = worker_of(x0 + ptiles - 1, F, kPxListWaves) - w0 + 1;
    po = a.pre_o + ((int64_t)(w0 + item) * 16 + row % 16) * HD;
    pml = a.pre_ml + ((int64_t)(w0 + item) * 16 + row % 16) * 2;
  }
  if (c1 > c0) {
    const int item = b * a.n_kv + kvh;
    const int64_t x0 = c0 * a.n_kv + kvh * (c1 - c0);
    const int w0 = worker_of(x0, all, kPxListWaves);
    n_own = worker_of(x0 + (c1 - c0) - 1, all, kPxListWaves) - w0 + 1;
    oo = a.own_o + ((int64_t)(w0 + item) * 16 + hh) * HD;
    oml = a.own_ml + ((int64_t)(w0 + item) * 16 + hh) * 2;
  }
  const int gi = threadIdx.x / TP, d4 = threadIdx.x % TP, n = n_pre + n_own;
  float M = -INFINITY, L = 0.f;
  f4_t O = {0.f, 0.f, 0.f, 0.f};
  for (int p = gi; p < n; p += G) {
    const float* ml = p < n_pre ? pml + (int64_t)p * 32 : oml + (int64_t)(p - n_pre) * 32;
    const float* op = p < n_pre ? po + (int64_t)p * 16 * HD : oo + (int64_t)(p - n_pre) * 16 * HD;
    const float m1 = ml[0], l1 = ml[1];
    const f4_t o1 = *reinterpret_cast<const f4_t*>(op + 4 * d4);
    const float Mn = fmaxf(M, m1);
    const float f0 = M == Mn ? 1.f : __builtin_amdgcn_exp2f(M - Mn), f1 = m1 == Mn ? 1.f : __builtin_amdgcn_exp2f(m1 - Mn);
    M = Mn;
    L = L * f0 + l1 * f1;
    O = O * f0 + o1 * f1;
  }
  if (d4 == 0) { sm[gi] = M; sl[gi] = L; }
  so[gi][d4] = O;
  __syncthreads();
  if (gi != 0) return;
  M = -INFINITY;
#pragma unroll
  for (int k = 0; k < G; ++k) M = fmaxf(M, sm[k]);
  L = 0.f;
  O = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < G; ++k) {
    const float f = sm[k] == M ? 1.f : __builtin_amdgcn_exp2f(sm[k] - M);
    L += sl[k] * f;
    O += so[k][d4] * f;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  h4_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (_Float16)(O[i] * inv);
  *reinterpret_cast<h4_t*>(a.out + b * a.out_stride + head * HD + 4 * d4) = v;
}

// Workspace: plan, then (m, l) and O of the own pieces and of the prefix's.
struct PxSpace { size_t plan, own_ml, own_o, pre_ml, pre_o, bytes; };
PxSpace px_space(int batch, int n_heads, int n_kv, int hd) {
  const size_t g = n_heads / n_kv, n_rg = (batch * g + 15) / 16;
  const size_t own = kPxListWaves + (size_t)batch * n_kv, pre = kPxListWaves + n_kv * n_rg;
  size_t off = 0;
  auto take = [&](size_t n) { const size_t o = off; off += (n + 255) & ~(size_t)255; return o; };
  PxSpace s;
  s.plan = take((batch + 2) * sizeof(int64_t));
  s.own_ml = take(own * 32 * 4);
  s.own_o = take(own * 16 * hd * 4);
  s.pre_ml = take(pre * 32 * 4);
  s.pre_o = take(pre * 16 * hd * 4);
  s.bytes = off;
  return s;
}

bool px_shape_ok(int batch, int n_heads, int n_kv, int hd) {
  return batch >= 0 && batch <= kPxMaxBatch && n_kv >= 1 && n_kv <= 64 && n_heads >= 1 && n_heads % n_kv == 0 &&
         n_heads / n_kv <= 16 && (hd == 64 || hd == 128);
}

template <int HD, int F>
void px_launch(const PxArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((px_stage1<HD, F>), dim3(kPxBlocks), dim3(kPxThreads), 0, st, a);
  hipLaunchKernelGGL((px_merge<HD>), dim3(a.batch * a.n_kv * a.g), dim3(kPxMergeThreads), 0, st, a);
}

template <int HD>
void px_format(const PxArgs& a, int fmt, hipStream_t st) {
  if (fmt == CQ_KV_FP16) px_launch<HD, CQ_KV_FP16>(a, st);
  else if (fmt == CQ_KV_INT8) px_launch<HD, CQ_KV_INT8>(a, st);
  else px_launch<HD, CQ_KV_FP8>(a, st);
}

}  // namespace

}  // namespace cq

using namespace cq;

extern "C" size_t cq_prefix_attention_workspace_bytes(int32_t batch, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim) {
  return px_shape_ok(batch, n_heads, n_kv_heads, head_dim) ? px_space(batch, n_heads, n_kv_heads, head_dim).bytes : 0;
}

extern "C" int cq_prefix_attention_decode(const void* q, int64_t q_stride, void* out, int64_t out_stride,
                                          const cq_kv_pages* prefix, const int32_t* d_prefix_table, int32_t prefix_pages,
                                          const int32_t* d_prefix_len, const cq_kv_pages* own, const int32_t* d_table,
                                          int32_t max_pages, const int32_t* d_start, const int32_t* d_len, int32_t batch,
                                          int32_t layer, int32_t n_heads, void* workspace, void* stream) {
  CQ_TRY(pages_check(prefix));
  CQ_TRY(pages_check(own));
  if (prefix->kv_dtype != own->kv_dtype || prefix->n_kv_heads != own->n_kv_heads || prefix->head_dim != own->head_dim)
    return fail(CQ_EINVAL, "prefix attention: the two caches differ in type or heads");
  if (layer < 0 || layer >= prefix->n_layers || layer >= own->n_layers) return fail(CQ_EINVAL, "prefix attention: layer outside the caches");
  if (!px_shape_ok(batch, n_heads, own->n_kv_heads, own->head_dim))
    return fail(CQ_EINVAL, "prefix attention: need batch in [0, 1024] and up to 16 query heads per kv head");
  if (batch == 0) return CQ_OK;
  if (!q || !out || !d_prefix_table || !d_prefix_len || !d_table || !d_len || !workspace)
    return fail(CQ_EINVAL, "prefix attention: null pointer");
  if (unaligned16(q) || unaligned16(out) || unaligned16(workspace))
    return fail(CQ_EINVAL, "prefix attention: q, out and workspace must be aligned to 16 bytes");
  const int64_t row = (int64_t)n_heads * own->head_dim;
  if (q_stride < row || out_stride < row || q_stride % 8 || out_stride % 8 || q_stride > ((int64_t)1 << 40) || out_stride > ((int64_t)1 << 40))
    return fail(CQ_EINVAL, "prefix attention: row strides must be multiples of 8 that hold a row");
  if (prefix_pages < 1 || max_pages < 1) return fail(CQ_EINVAL, "prefix attention: empty tables");
  const PxSpace s = px_space(batch, n_heads, own->n_kv_heads, own->head_dim);
  char* ws = (char*)workspace;
  PxArgs a{};
  a.q = (const _Float16*)q; a.out = (_Float16*)out; a.q_stride = q_stride; a.out_stride = out_stride;
  a.pre = page_view(*prefix); a.own = page_view(*own);
  a.pre_layer = layer * prefix->layer_stride; a.own_layer = layer * own->layer_stride;
  a.pre_table = d_prefix_table; a.pre_len = d_prefix_len; a.table = d_table; a.start = d_start; a.len = d_len;
  a.pre_pages = prefix_pages; a.max_pages = max_pages;
  a.batch = batch; a.n_kv = own->n_kv_heads; a.g = n_heads / own->n_kv_heads;
  a.plan = (int64_t*)(ws + s.plan);
  a.own_ml = (float*)(ws + s.own_ml); a.own_o = (float*)(ws + s.own_o);
  a.pre_ml = (float*)(ws + s.pre_ml); a.pre_o = (float*)(ws + s.pre_o);
  const hipStream_t st = (hipStream_t)stream;
  if (own->head_dim == 128) px_format<128>(a, own->kv_dtype, st);
  else px_format<64>(a, own->kv_dtype, st);
  CQ_HIP(hipGetLastError());
  return CQ_OK;
}
