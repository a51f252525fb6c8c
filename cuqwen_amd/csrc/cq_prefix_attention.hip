// Decode attention of a batch whose sequences share a prefix, over paged caches
// (cq_kv_pages): the prefix's K and V are read for all rows of a kv head together,
// each sequence's own pages for its own rows.  No counterpart in the reference.
//
// For row (b, head h of kv head kvh): s_t = q . k_t / sqrt(hd) over the prefix's and
// the sequence's own positions, out = sum exp(s_t - m) v_t / sum exp(s_t - m).  Two
// launches:
//   * px_stage1: the prefix, for all rows of a kv head together, in pieces of keys that
//     leave (m, l, O) in fp32; and the own tiles of very long sequences;
//   * px_finish: a block per (sequence, kv head) attends over the sequence's own tiles,
//     joins the pieces of its rows by the log-sum-exp rule and writes the output.
// Where the tables are short px_finish takes the prefix too, once for each sequence, and
// is the only launch; where only the lengths are short (known on the device alone) it
// does so behind a first launch with nothing to do.
//
// What bounds it (per kernel, 7B heads, fp16 unless said otherwise):
//   * two answers to a short question: the launch (0.5B heads, 100 tokens: one of 4.0 us);
//   * up to 16 rows a kv head: HBM (2 sequences: 13.7 us for each further 32640 tokens,
//     4.9 TB/s; a plain copy 4.9), behind about 16 us of two launches, their code, which
//     comes cold from L2 in 64-byte lines, and the joining;
//   * 64 sequences (448 rows): waves that wait for each other (px_shared_piece);
//   * own tokens: HBM (64 sequences with up to 1000: px_finish reads 89 MB, pieces
//     included, in 22.8 us, 3.9 TB/s).
//
// Work of stage 1, whose grid is one block per CU: the steps (a few 32-key tiles) of
// all items of the prefix, an item being (kv head, block of query rows), form one
// list that its blocks share evenly, and the steps of far tiles of all (sequence, kv head) items
// one that the other blocks share evenly (share_of), wherever item borders
// fall, from the lengths found on the device: lengths may be ragged, and a captured
// launch serves other lengths.  Worker w's piece of item i is stored in slot w + i
// (either w or i grows from one piece to the next, so slots differ), and px_finish
// finds a row's pieces by the same arithmetic.
#include "cq_attention.h"
#include "cq_pages.h"

#include <algorithm>
#include <cmath>

namespace cq {

namespace {

constexpr int kPxWaves = 8, kPxThreads = kPxWaves * kWave;
constexpr int kPxBlocks = kNumCUs;                    // one block per CU
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
  int64_t* plan;                  // [batch + 1] far own steps before each sequence
  int* pre_items;                 // first and last worker of each item of the prefix, of each far own item
  int* own_items;
  float* own_o;                   // [slot][16][HD]
  float* own_ml;                  // [slot][16][2]
  float* pre_o;                   // [slot][rows of a block][HD]
  float* pre_ml;
};

// a / b for a >= 0, b > 0; in 32 bits where they do (64-bit divisions are a microsecond of
// code each, and lists of so many tiles are rare).
__device__ __forceinline__ int64_t px_div(int64_t a, int64_t b) {
  if (((uint64_t)(a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}
// Range [first, end) of worker w when F tiles are shared by W workers (the first F
// workers, a tile each, if there are fewer tiles): F w / W, F (w + 1) / W.
__device__ __forceinline__ void share_of(int w, int64_t F, int W, int64_t* first, int64_t* end) {
  *first = F <= W ? min((int64_t)w, F) : px_div(F * w, W);
  *end = F <= W ? min((int64_t)w + 1, F) : px_div(F * (w + 1), W);
}
// The worker that has tile x.
__device__ __forceinline__ int worker_of(int64_t x, int64_t F, int W) { return (int)(F <= W ? x : px_div((x + 1) * W - 1, F)); }

// Of its n own tiles, how many of a sequence's px_finish takes: all or none; stage 1
// takes the others, in pieces.  With few blocks in the second launch the first one's
// are there for sequences of more than a tile per wave (7B heads, 8 sequences over
// 32640, up to 400 of their own, 13 tiles: 30.5 us both ways; one of 8000: 15.0 us in
// pieces, 17.8 with the first 16 here; 16 of up to 100: 33.4 here, 38.6 in pieces; 16 of up
// to 1500: 45.8 with up to 16 here, 40.2 in pieces; 14B heads, E4M3, 8 over 20001, of up to
// 300: 29.4 and 32.3).
__device__ __forceinline__ int px_near(const PxArgs& a, int n) {
  const int most = a.batch * a.n_kv <= 64 ? 8 : 64;
  return n <= most ? n : 0;
}

// Whether px_finish takes the prefix, `ptiles` tiles for each of its `blocks`.  There a
// tile takes 0.16 us while a block has L2 to itself, blocks * 0.8 ns beyond 190 of them
// (20 TB/s; one-byte tiles, bound by their conversion, 1.0 ns); in pieces the prefix
// takes 9 us + 30 ns for each block whose pieces are to be joined.  Measured, here and in
// pieces, 7B heads, fp16: 8 sequences over 1500 tokens 11.8 and 16.8 us, over 2500 22.5
// and 16.9; 64 over 3000 26.5 and 28.3; 256 over 800 27.6 and 41, over 1600 44.8 and 43.9.
__device__ __host__ __forceinline__ bool px_prefix_near(int blocks, int64_t ptiles, bool one_byte) {
  return ptiles * std::max(190, one_byte ? blocks + blocks / 4 : blocks) <= 11000 + (int64_t)36 * blocks;
}

// Positions that a table of n pages holds, and the length cut there.
__device__ __forceinline__ int cut_len(int len, int pages, int shift) {
  return min(max(len, 0), pages << shift);   // at most 2^30 (checked by the host)
}

// Positions [lo, hi) of one kv head of a paged cache.
struct PxKV {
  PageView pv;
  int64_t off;       // elements: layer and head
  const int* table;  // page of each run of page_tokens positions
  int lo, hi;
};

// The K and V of one 32-key tile in matrix operand order, and which of its keys are there.
template <int HD, int F>
struct PxTile {
  u4_t k[F == CQ_KV_FP16 ? HD / 16 : HD / 32], v[F == CQ_KV_FP16 ? HD / 16 : HD / 32];
  f4_t ks[F == CQ_KV_FP16 ? 1 : 2], vs[F == CQ_KV_FP16 ? 1 : 2];
  uint32_t valid;    // a bit per key
};

// Requests tile ti (positions [32 ti, 32 ti + 32) cut to kv's); with `want` false,
// or a page outside the pool, nothing is read and no key is valid.
template <int HD, int F>
__device__ __forceinline__ void px_load(PxTile<HD, F>& t, const PxKV& kv, int ti, bool want, int lane) {
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
  const int lo = max(kv.lo - 32 * ti, 0), hi = min(kv.hi - 32 * ti, 32);
  t.valid = ok && hi > lo ? (0xffffffffu >> (32 - hi)) & (0xffffffffu << lo) : 0u;
}

// Operand i of a tile's K (or V) as fp16.
template <int F>
__device__ __forceinline__ h8_t px_operand(const u4_t* w, int i, uint32_t magic) {
  if constexpr (F == CQ_KV_FP16) return __builtin_bit_cast(h8_t, w[i]);
  else return codes_to_h8<F>(i & 1 ? u2_t{w[i / 2].z, w[i / 2].w} : u2_t{w[i / 2].x, w[i / 2].y}, magic);
}

// The power of two at or below x >= 0, at most 2^126, and 1 / x for such a power: exact,
// where a division would be ten instructions.
__device__ __forceinline__ float px_power(float x) { return fminf(__uint_as_float(__float_as_uint(x) & 0x7f800000u), 0x1p126f); }
__device__ __forceinline__ float px_inverse(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }

// A wave's running softmax over 16 query columns: lane (h, j) holds column h, dims
// dt * 16 + 4 j + i, m in log2 units, and in l its own keys' part of the sum.  One-byte V:
// P is rounded to fp16 as p * scale / r, r the power of two at or below the largest V
// scale seen (so that small scales do not drive the products into fp16's subnormals), and
// O is kept in units of r.
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
  if (t.valid != 0xffffffffu) {   // wave-uniform
    // masked keys may hold anything, in V too: a weight of 0 does not silence a NaN
    const uint32_t mine[2] = {t.valid >> (4 * j), t.valid >> (16 + 4 * j)};   // bits of the lane's keys
    uint32_t in[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      in[e] = (uint32_t)((int32_t)(mine[e >> 2] << (31 - (e & 3))) >> 31);   // all ones: the key is there
      const uint32_t x = __float_as_uint(s[e >> 2][e & 3]);
      s[e >> 2][e & 3] = __uint_as_float((x & in[e]) | (0xff800000u & ~in[e]));
      if constexpr (F != CQ_KV_FP16) t.vs[e >> 2][e & 3] = __uint_as_float(__float_as_uint(t.vs[e >> 2][e & 3]) & in[e]);
    }
    constexpr int N = sizeof(t.v) / sizeof(t.v[0]);
    u4_t keep;   // of an operand's 8 keys, or of two operands'
    if constexpr (F != CQ_KV_FP16) {
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const uint32_t lo = __builtin_amdgcn_perm(in[4 * a + 1], in[4 * a], 0x0c0c0400u), hi = __builtin_amdgcn_perm(in[4 * a + 3], in[4 * a + 2], 0x04000c0cu);
        keep[a] = keep[2 + a] = lo | hi;
      }
    } else {
#pragma unroll
      for (int a = 0; a < 4; ++a) keep[a] = __builtin_amdgcn_perm(in[2 * a + 1], in[2 * a], 0x05040100u);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) t.v[n] &= keep;
  }
  float mn = max3(max3(s[0][0], s[0][1], s[0][2]), s[0][3], s[1][0]);
  mn = fmaxf(st.m, col_max(max3(max3(mn, s[1][1], s[1][2]), s[1][3], -INFINITY)) * c2);
  float rn = st.r;
  if constexpr (F != CQ_KV_FP16) {
    float vm = 0.f;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int i = 0; i < 4; ++i) vm = fmaxf(vm, fabsf(t.vs[a][i]));
    rn = fmaxf(rn, px_power(col_max(vm)));
  }
  if (__any(mn > st.m || rn > st.r)) {
    const float alpha = mn == st.m ? 1.f : __builtin_amdgcn_exp2f(st.m - mn);
    const float beta = F != CQ_KV_FP16 ? alpha * (st.r * px_inverse(rn)) : alpha;
    st.m = mn;
    st.r = rn;
    st.l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) st.o[dt] *= beta;
  }
  const float mm = st.m == -INFINITY ? 0.f : st.m;   // no valid key yet: the masked ones give 0
  const float ri = F != CQ_KV_FP16 ? px_inverse(st.r) : 1.f;
  // each weight in two fp16 parts, 22 bits: the matrix units idle here anyway
  h8_t pb, pc;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s[a][i], c2, -mm));
      st.l += p;
      const float x = F != CQ_KV_FP16 ? p * (t.vs[a][i] * ri) : p;
      pb[a * 4 + i] = (_Float16)x;
      pc[a * 4 + i] = (_Float16)(x - (float)pb[a * 4 + i]);
    }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const h8_t v = px_operand<F>(t.v, dt, magic);
    st.o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pb, st.o[dt], 0, 0, 0);
    st.o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pc, st.o[dt], 0, 0, 0);
  }
}

// Below any V scale that matters (half an fp16 subnormal over 448).
constexpr float kPxSmallest = 0x1p-40f;

// Tiles ta, ta + step, ... < tb for the rows q[r0 .. r0 + rows) of a kv head: the
// wave's state, l complete in every lane and O in the values' own units.  load(tile, k)
// requests tile k; before() runs while the first tile is on its way.
// With LONG two copies of the tile's code take turns on two buffers; without, one copy
// and 64 register moves a tile: code that runs for a tile or two is what an instruction
// cache filled at 100 cycles a line makes it wait for (a tile's is 2-4 KB).
template <int HD, int F, bool LONG, class Load, class Before>
__device__ __forceinline__ void px_run(PxState<HD>& st, const PxArgs& a, int kvh, int r0, int rows, int ta, int tb, int step, int lane,
                                       Load load, Before before) {
  constexpr int KK = HD / 32, DT = HD / 16;
  const int h = lane & 15, j = lane >> 4;
  const float c2 = kLog2e / sqrtf((float)HD);
  const uint32_t magic = vgpr_const(0x64646464u);
  PxTile<HD, F> A, B;
  load(A, ta);
  h8_t qb[KK];
  const int r = r0 + min(h, rows - 1), b = r / a.g;
  const _Float16* q = a.q + b * a.q_stride + (kvh * a.g + (r - b * a.g)) * HD;
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) qb[kk] = __builtin_bit_cast(h8_t, load_u4(q + kk * 32 + j * 8));
  st.m = -INFINITY;
  st.l = 0.f;
  st.r = kPxSmallest;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) st.o[dt] = f4_t{0.f, 0.f, 0.f, 0.f};
  before();
  if constexpr (LONG) {
    for (int ti = ta; ti < tb; ti += 2 * step) {
      load(B, ti + step);
      px_attend<HD, F>(A, qb, st, c2, lane, magic);
      if (ti + step >= tb) break;
      load(A, ti + 2 * step);
      px_attend<HD, F>(B, qb, st, c2, lane, magic);
    }
  } else {
#pragma unroll 1
    for (int ti = ta; ti < tb; ti += step) {
      load(B, ti + step);
      px_attend<HD, F>(A, qb, st, c2, lane, magic);
      A = B;
    }
  }
  st.l += __shfl_xor(st.l, 16, kWave);
  st.l += __shfl_xor(st.l, 32, kWave);
  if constexpr (F != CQ_KV_FP16) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) st.o[dt] *= st.r;
  }
}

// Joins the states of the waves k * RG + rg, k < KH, through LDS (sm: W (2 + DT * 16)
// * 16 floats for W waves): every wave of the block calls it, and gets in O the dim
// tiles kg, kg + KH, ... of its row group, in M and L the joined statistics.
template <int HD, int RG, int KH>
struct PxJoin {
  static constexpr int DT = HD / 16, PER = (DT + KH - 1) / KH;
  float M, L;
  f4_t O[PER];
  __device__ __forceinline__ void run(const PxState<HD>& st, float* sm, int wave, int lane) {
    float* ml = sm + RG * KH * DT * kWave * 4;   // [wave][16][2]
    f4_t* w = reinterpret_cast<f4_t*>(sm) + wave * DT * kWave + lane;
    const int rg = wave % RG, kg = wave / RG, h = lane & 15;
    __syncthreads();   // LDS may be in use
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) w[dt * kWave] = st.o[dt];
    if (lane < 16) {
      ml[(wave * 16 + h) * 2] = st.m;
      ml[(wave * 16 + h) * 2 + 1] = st.l;
    }
    __syncthreads();
    float m1[KH];
    M = -INFINITY;
    L = 0.f;
#pragma unroll
    for (int k = 0; k < KH; ++k) {
      m1[k] = ml[((k * RG + rg) * 16 + h) * 2];
      M = fmaxf(M, m1[k]);
    }
#pragma unroll
    for (int k = 0; k < KH; ++k) {
      m1[k] = m1[k] == M ? 1.f : __builtin_amdgcn_exp2f(m1[k] - M);
      L += ml[((k * RG + rg) * 16 + h) * 2 + 1] * m1[k];
    }
    const f4_t* s = reinterpret_cast<const f4_t*>(sm) + lane;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      O[i] = f4_t{0.f, 0.f, 0.f, 0.f};
      if (kg + i * KH < DT) {
#pragma unroll
        for (int k = 0; k < KH; ++k) O[i] += s[((k * RG + rg) * DT + kg + i * KH) * kWave] * m1[k];
      }
    }
  }
};

// How a block attends over the prefix with ROWS query rows.  Up to 64 rows every wave
// takes 16 of them over tiles of its own in registers (the K / V operands feed one
// instruction each, and HBM is what bounds it); beyond that 32 rows over tiles in LDS,
// which the row groups share.  KH waves share a row group's keys.
template <int HD, int F, int ROWS>
struct PxForm {
  static constexpr bool LDS = ROWS > 64;
  static constexpr int WR = LDS ? 32 : 16;              // rows of a wave
  static constexpr int RG = ROWS / WR, KH = kPxWaves / RG;
  static constexpr int TPW = !LDS ? 1 : KH == 1 ? 2 : KH == 2 ? (HD == 128 && F != CQ_KV_FP16 ? 1 : 2) : (HD == 64 ? 2 : 1);
  static constexpr int TPS = KH * TPW;                  // tiles of a step
  static constexpr int TILE = kTileKeys * HD;           // halves of K (or V) per tile
  static constexpr int STAGE = 2 * TPS * TILE;          // halves: K tiles, then V tiles
  // LDS slots: three (requests two steps ahead) where they fit 96 KB, else two
  static constexpr int NS = F == CQ_KV_FP16 && 3 * STAGE * 2 <= 96 * 1024 ? 3 : 2;
  static constexpr int DT = HD / 16, CG = WR / 16;
  static constexpr int STATE = 4 + 4 * DT * CG;         // floats of one lane's softmax state in LDS (two slices): (m, l) of each, O
  // halves of LDS: the states that PxJoin takes; the stages, over them the states of the other key groups
  static constexpr int SM = std::max({kPxWaves * 16 * (2 + HD) * 2, LDS ? NS * STAGE : 0, LDS ? (KH - 1) * RG * kWave * STATE * 2 : 0});
  static constexpr int SCL = LDS && F != CQ_KV_FP16 ? (NS + 3) * TPS * kTileKeys : 1;   // K scales per slot, V scales three steps
};

// Tiles [tb, te) of a cache for the rows [r0, min(r0 + 16 RG, R)) of a kv head, by the
// waves of a block in registers.  Up to 32 rows HBM bounds it (0.34 us a 32-key E4M3 tile
// and CU, HD 128); 33 to 64 rows over one-byte tiles their conversion, which each of up to
// four row groups does for itself (0.72 us).  Two slices of rows a wave, converted once,
// spill 40 registers and take 44.4 us where this takes 38.4 (8 sequences over 65280, E4M3).
template <int HD, int F, int RG>
__device__ __forceinline__ void px_stream_piece(const PxArgs& a, const PxKV& kv, float* sm, int kvh, int r0, int R, int tb, int te, float* o,
                                                float* ml) {
  constexpr int DT = HD / 16, KH = kPxWaves / RG;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int rg = wave % RG, kg = wave / RG, rw = r0 + rg * 16;
  PxState<HD> st;
  const int end = rw < R ? te : tb;   // a wave without rows takes no tile
  px_run<HD, F, true>(st, a, kvh, min(rw, R - 1), max(min(16, R - rw), 1), tb + kg, end, KH, lane,
                [&](PxTile<HD, F>& t, int k) __attribute__((always_inline)) { px_load<HD, F>(t, kv, k, k < end, lane); },
                []() {});
  PxJoin<HD, RG, KH> jn;
  jn.run(st, sm, wave, lane);
  const int h = lane & 15, j = lane >> 4;
  if (rw + h >= R) return;
#pragma unroll
  for (int i = 0; i < jn.PER; ++i)
    if (kg + i * KH < DT) *reinterpret_cast<f4_t*>(o + (rg * 16 + h) * HD + (kg + i * KH) * 16 + 4 * j) = jn.O[i];
  if (kg == 0 && j == 0) {
    ml[2 * (rg * 16 + h)] = jn.M;
    ml[2 * (rg * 16 + h) + 1] = jn.L;
  }
}

// Asks the compiler for N groups of MF matrix and VA vector instructions with the LDS reads
// of their operands AHEAD groups before them; left to itself it reads each operand where
// it is used.  (7B heads, 64 sequences over 65280, fp16: 105.6 -> 102.6 us; one-byte
// tiles, with their scales to read, 70.0 -> 71.7 over 32640, so not there.)
template <int ID, int AHEAD, int N, int MF, int VA>
__device__ __forceinline__ void px_interleave() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, ID);   // LDS reads
#pragma unroll
  for (int q = 0; q < N; ++q) {
    __builtin_amdgcn_sched_group_barrier(0x8, MF, ID);
    __builtin_amdgcn_sched_group_barrier(0x2, VA, ID);
    if (q < N - AHEAD) __builtin_amdgcn_sched_group_barrier(0x100, 1, ID);
  }
}

// Tiles [tb, te) of the prefix for 128 or 256 rows: the prefill attention's loop
// over pages, without its causal limits.  64 sequences of 7B heads, fp16: 41 us for each
// further 32640 tokens, 730 TFLOP/s.  Over the launch at 32640 tokens the matrix units are
// busy for 21 % of the cycles, LDS for 12 %, and waves wait for 45 %: of the 46 us that the
// loop took before its addresses came from lanes, 14 went with the requests taken out, 9
// with the LDS reads, 8 with most of the PV products, 5 with the exponentials.  Tried and no
// faster: a tile a wave and step with three or four slots (47 us), V requested and awaited
// at the middle of a step (41), a wave priority by key group (41), one copy of the step in
// the code (48), the next operand's reads fully ahead (42).
template <int HD, int F, int ROWS>
__device__ __forceinline__ void px_shared_piece(const PxArgs& a, _Float16* smem, float* scl, int kvh, int r0, int R, int lp, int tb, int te,
                                                float* o_out, float* ml_out) {
  using P = PxForm<HD, F, ROWS>;
  constexpr bool KV8 = F != CQ_KV_FP16;
  constexpr int KK = HD / 32, DT = HD / 16, CG = P::CG, RG = P::RG, KH = P::KH, TPW = P::TPW, TPS = P::TPS, ST = 2 * TPW;
  constexpr int TILE = P::TILE, NS = P::NS, ES = KV8 ? 1 : 2;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int h = lane & 15, j = lane >> 4;
  const int rg = wave % RG, kg = wave / RG, rw = r0 + rg * 32;
  const bool idle = rw >= R;   // no rows: the wave only helps to stage
  const int lim = min(lp, te * kTileKeys), s5 = a.pre.shift - 5;
  const int n_steps = (te - tb + TPS - 1) / TPS;
  const float c2 = kLog2e / sqrtf((float)HD);
  const int64_t head = a.pre_layer + kvh * a.pre.head_stride;

  // Where the tiles lie: lane i holds the byte offset of tile i of the next 64, from a
  // vector's worth of table entries, and a step takes its own with lane reads (as scalar
  // code, two 64-bit products and sums per tile and step, this was a third of the loop's
  // instructions).  Tiles past the range repeat its last one (and are masked).  A page
  // outside the pool is read as page 0 and its keys masked: `bad` holds TPS bits per
  // step, the latest lowest.
  struct Tiles { int64_t off[TPS]; };
  static_assert(kWave % TPS == 0, "whole steps per look-up");
  constexpr uint32_t BITS = (1u << TPS) - 1;
  int64_t lane_off = 0;
  unsigned long long lane_bad = 0;
  uint32_t bad = 0;
  auto tile_at = [&](int ti) __attribute__((always_inline)) { return min(ti, te - 1); };
  auto look_up = [&](int step) __attribute__((always_inline)) {   // called for every step in turn
    constexpr int PER = kWave / TPS;
    const int first = step % PER * TPS;
    if (first == 0) {
      const int ti = tile_at(tb + step * TPS + lane), page = a.pre_table[ti >> s5];
      const bool ok = page >= 0 && page < a.pre.n_pages;
      lane_off = (head + (int64_t)(ok ? page : 0) * a.pre.page_stride + (int64_t)(ti & ((1 << s5) - 1)) * TILE) * ES;
      lane_bad = __ballot(!ok);
    }
    Tiles r;
#pragma unroll
    for (int i = 0; i < TPS; ++i) {
      const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)lane_off, first + i), hi = __builtin_amdgcn_readlane((int)(lane_off >> 32), first + i);
      r.off[i] = (int64_t)((uint64_t)hi << 32 | lo);
    }
    bad = (bad << TPS) | ((uint32_t)(lane_bad >> first) & BITS);
    return r;
  };
  // fp16 cache: straight into LDS, 1 KB per wave instruction, no registers
  constexpr int TB = TILE * 2 / 1024, PW = TPS * TB / kPxWaves;   // KB of a tile's K (or V); instructions per wave and step
  static_assert(KV8 || PW * kPxWaves == TPS * TB, "whole pieces per wave");
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  const uint32_t in_tile = (wave % TB * kWave + lane) * 16;   // of the wave's pieces
  auto dma = [&](const Tiles& tl, int step, int part) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int p = i * kPxWaves + wave;
      // tile of the piece: i (8 KB tiles) or 2 i and 2 i + 1 (4 KB tiles)
      const int64_t off = TB == 8 ? tl.off[i] : wave < 4 ? tl.off[i * 2 % TPS] : tl.off[(i * 2 + 1) % TPS];
      lds_load_1k(lds0 + ((step % NS) * P::STAGE + part * TPS * TILE) * 2 + p * 1024, in_tile, a.pre.kv[part] + off);
    }
  };
  // keys that are not there may hold anything: keep them out of P*V (each wave clears
  // them in the pieces of V that it requested, once they are there)
  auto clear_tail = [&](int step, uint32_t bits) __attribute__((always_inline)) {
    if ((tb + (step + 1) * TPS) * kTileKeys <= lim && bits == 0) return;
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int p = i * kPxWaves + wave, n = p / TB, k0 = tile_at(tb + step * TPS + n) * kTileKeys + 4 * j;
      const int end = bits >> n & 1 ? 0 : lim;
      h8_t* q = reinterpret_cast<h8_t*>(smem + (step % NS) * P::STAGE + TPS * TILE + p * 512 + lane * 8);
      h8_t v = *q;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k0 + (e < 4 ? e : 12 + e) >= end) v[e] = (_Float16)0.f;
      *q = v;
    }
  };
  // one-byte cache: 16-byte pieces through registers, converted to fp16 on the way into
  // LDS, so the codes are expanded once per block
  constexpr int TP = TILE / 16, QL = KV8 ? (TPS * TP + kPxThreads - 1) / kPxThreads : 1;   // pieces of a tile; per thread
  constexpr bool FULL = QL * kPxThreads == TPS * TP;   // else (one piece) the last threads have none
  static_assert(!KV8 || FULL || QL == 1, "whole pieces per thread");
  const uint32_t magic = vgpr_const(0x64646464u);
  struct Pieces { u4_t w[QL]; float s[2]; };
  constexpr int SK = TPS * kTileKeys;
  float *scl_k = scl, *scl_v = scl + NS * SK;   // V scales come with the K of their step, so three slots
  auto load = [&](Pieces& r, const Tiles& tl, int step, int part, uint32_t bits) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < QL; ++i) {
      const int c = FULL ? i * kPxThreads + threadIdx.x : min((int)threadIdx.x, TPS * TP - 1);
      int64_t off = 0;
#pragma unroll
      for (int n = 0; n < TPS; ++n)
        if (c / TP == n) off = tl.off[n];
      r.w[i] = load_u4(a.pre.kv[part] + off + c % TP * 16);
    }
    if (part == 0 && threadIdx.x < SK) {
      const int c = threadIdx.x, n = c / kTileKeys, key = tile_at(tb + step * TPS + n) * kTileKeys + c % kTileKeys;
      int64_t off = 0;
#pragma unroll
      for (int i = 0; i < TPS; ++i)
        if (n == i) off = tl.off[i];
      off = off / HD + c % kTileKeys;
      const bool in = key < lim && !(bits >> n & 1) && tb + step * TPS + n < te;
      r.s[0] = in ? a.pre.scale[0][off] : 0.f;
      r.s[1] = in ? a.pre.scale[1][off] : 0.f;
    }
  };
  auto store = [&](const Pieces& r, int step, int part, uint32_t bits) __attribute__((always_inline)) {
    _Float16* dst = smem + (step % NS) * P::STAGE + part * TPS * TILE;
    const bool whole = F == CQ_KV_INT8 || part == 0 || ((tb + (step + 1) * TPS) * kTileKeys <= lim && bits == 0);
#pragma unroll
    for (int i = 0; i < QL; ++i) {
      const int c = i * kPxThreads + threadIdx.x, q = c % TP;
      if (!FULL && c >= TPS * TP) break;
      // 16 bytes: the operand pieces of two instructions
      _Float16* d = dst + (c / TP) * TILE + ((q / 64) * 128 + q % 64) * 8;
      h8_t v[2] = {codes_to_h8<F>(u2_t{r.w[i].x, r.w[i].y}, magic), codes_to_h8<F>(u2_t{r.w[i].z, r.w[i].w}, magic)};
      if (!whole) {   // an E4M3 code that is not there may be NaN
        const int n = c / TP, k0 = tile_at(tb + step * TPS + n) * kTileKeys + 4 * (q % 64 / 16), end = bits >> n & 1 ? 0 : lim;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k0 + (e < 4 ? e : 12 + e) >= end) v[0][e] = v[1][e] = (_Float16)0.f;
      }
      *reinterpret_cast<h8_t*>(d) = v[0];
      *reinterpret_cast<h8_t*>(d + 512) = v[1];
    }
    if (part == 0 && threadIdx.x < SK) {
      scl_k[step % NS * SK + threadIdx.x] = r.s[0];
      scl_v[step % 3 * SK + threadIdx.x] = r.s[1];
    }
  };
  // Group g = (K of step g + 1, V of step g), requested NS - 1 steps ahead.
  Pieces pk, pv8;
  Tiles tv = look_up(0);   // of the V to be requested next
  auto request = [&](int g) __attribute__((always_inline)) {
    const Tiles tk = look_up(g + 1);
    if constexpr (KV8) {
      load(pk, tk, g + 1, 0, bad & BITS);
      load(pv8, tv, g, 1, 0);
    } else {
      dma(tk, g + 1, 0);
      dma(tv, g, 1);
    }
    tv = tk;
  };
  // Group g in LDS for every wave (its readers' slots free since the last barrier).
  // Step g + NS - 1 has been looked up last by then.
  auto arrive = [&](int g) __attribute__((always_inline)) {
    if constexpr (KV8) {
      store(pk, g + 1, 0, 0);
      store(pv8, g, 1, bad >> (NS - 1) * TPS & BITS);
    } else {
      wait_vm<(NS - 2) * 2 * PW>();
      clear_tail(g, bad >> (NS - 1) * TPS & BITS);
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
    lds_barrier();
  };

  h8_t qb[CG][KK];
#pragma unroll
  for (int cg = 0; cg < CG; ++cg) {
    const int r = min(rw + cg * 16 + h, R - 1), b = r / a.g;
    const _Float16* q = a.q + b * a.q_stride + (kvh * a.g + (r - b * a.g)) * HD;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qb[cg][kk] = __builtin_bit_cast(h8_t, load_u4(q + kk * 32 + j * 8));
  }
  float m[CG], l[CG], r = 0x1p-100f;   // running maximum (raw products, K scale applied), lane's sum, unit of O
  f4_t o[DT][CG];
#pragma unroll
  for (int cg = 0; cg < CG; ++cg) {
    m[cg] = -INFINITY;
    l[cg] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt][cg] = f4_t{0.f, 0.f, 0.f, 0.f};
  }
  typedef f4_t S_t[ST][CG];
  auto qk = [&](S_t& s, int step) __attribute__((always_inline)) {   // S^T of the wave's tiles
    const _Float16* kt = smem + (step % NS) * P::STAGE + kg * TPW * TILE;
#pragma unroll
    for (int st = 0; st < ST; ++st) {
#pragma unroll
      for (int cg = 0; cg < CG; ++cg) s[st][cg] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const h8_t ka = *reinterpret_cast<const h8_t*>(kt + st * 16 * HD + (kk * 64 + lane) * 8);
#pragma unroll
        for (int cg = 0; cg < CG; ++cg) s[st][cg] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qb[cg][kk], s[st][cg], 0, 0, 0);
      }
    }
  };
  auto scale_mask = [&](S_t& s, int step, uint32_t bits) __attribute__((always_inline)) {
    const int t0 = tb + step * TPS + kg * TPW;   // the wave's first tile
    if constexpr (KV8) {
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const f4_t ks = *reinterpret_cast<const f4_t*>(scl_k + step % NS * SK + kg * TPW * kTileKeys + st * 16 + 4 * j);
#pragma unroll
        for (int cg = 0; cg < CG; ++cg) s[st][cg] *= ks;
      }
    }
    if ((t0 + TPW) * kTileKeys > lim || bits) {
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int end = bits >> (kg * TPW + st / 2) & 1 ? 0 : lim;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = t0 * kTileKeys + st * 16 + 4 * j + i;
#pragma unroll
          for (int cg = 0; cg < CG; ++cg) s[st][cg][i] = key >= end ? -INFINITY : s[st][cg][i];
        }
      }
    }
  };
  float mn[CG], rn = r;
  auto row_max = [&](const S_t& s, int step) __attribute__((always_inline)) {   // the running maximum with s
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) {
      float mx = m[cg];
#pragma unroll
      for (int st = 0; st < ST; ++st) mx = max3(max3(mx, s[st][cg][0], s[st][cg][1]), s[st][cg][2], s[st][cg][3]);
      mn[cg] = col_max(mx);
    }
    if constexpr (KV8) {
      float vm = 0.f;
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const f4_t vs = *reinterpret_cast<const f4_t*>(scl_v + step % 3 * SK + kg * TPW * kTileKeys + st * 16 + 4 * j);
        vm = max3(max3(vm, fabsf(vs[0]), fabsf(vs[1])), fabsf(vs[2]), fabsf(vs[3]));
      }
      rn = fmaxf(r, px_power(col_max(vm)));
    }
  };
  auto rescale = [&]() __attribute__((always_inline)) {   // rare once a row has seen some keys
    bool grow = KV8 && rn > r;
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) grow |= mn[cg] > m[cg];
    if (__any(grow)) {
      const float beta = KV8 ? r * px_inverse(rn) : 1.f;
      r = rn;
#pragma unroll
      for (int cg = 0; cg < CG; ++cg) {
        const float alpha = mn[cg] == m[cg] ? 1.f : __builtin_amdgcn_exp2f((m[cg] - mn[cg]) * c2);
        m[cg] = mn[cg];
        l[cg] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt][cg] *= alpha * beta;
      }
    }
  };
  h8_t pb[TPW][CG];
  auto probs = [&](const S_t& s, int step) __attribute__((always_inline)) {   // P^T and the row sums
    const float ri = KV8 ? px_inverse(r) : 1.f;
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) {
      const float mm = m[cg] == -INFINITY ? 0.f : m[cg] * c2;   // no valid key yet: masked scores give exp2(-inf) = 0
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        f4_t vs = {1.f, 1.f, 1.f, 1.f};
        if constexpr (KV8) vs = *reinterpret_cast<const f4_t*>(scl_v + step % 3 * SK + kg * TPW * kTileKeys + st * 16 + 4 * j) * ri;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[st][cg][i], c2, -mm));
          l[cg] += p;
          // fp16 (half a step: 2^-11 of the weight): the matrix units are what many rows wait for
          pb[st / 2][cg][(st & 1) * 4 + i] = (_Float16)(KV8 ? p * vs[i] : p);
        }
      }
    }
  };
  auto pv = [&](int step) __attribute__((always_inline)) {
    const _Float16* vt = smem + (step % NS) * P::STAGE + (TPS + kg * TPW) * TILE;
#pragma unroll
    for (int tw = 0; tw < TPW; ++tw)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const h8_t va = *reinterpret_cast<const h8_t*>(vt + tw * TILE + (dt * 64 + lane) * 8);
#pragma unroll
        for (int cg = 0; cg < CG; ++cg) o[dt][cg] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[tw][cg], o[dt][cg], 0, 0, 0);
      }
  };

  // Software pipeline: step n forms P(n) from S(n) while the matrix cores take
  // S(n + 1), then takes P(n) V(n) while the maximum of S(n + 1) is formed; it reads
  // group n (K(n + 1), V(n)) from LDS.
  S_t sa, sb;
  __syncthreads();   // the piece before has left LDS
  const uint32_t bad0 = bad & BITS;
  if constexpr (KV8) {
    load(pk, tv, 0, 0, bad0);
    store(pk, 0, 0, 0);
    request(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);
  } else {
    dma(tv, 0, 0);
#pragma unroll
    for (int g = 0; g < NS - 1; ++g) request(g);
    wait_vm<(NS - 1) * 2 * PW>();
  }
  lds_barrier();
  auto first = [&]() __attribute__((always_inline)) {
    qk(sa, 0);
    scale_mask(sa, 0, bad0);
    row_max(sa, 0);
    rescale();
    arrive(0);
  };
  auto step = [&](S_t& cur, S_t& nxt, int n) __attribute__((always_inline)) {
    request(n + NS - 1);
    __builtin_amdgcn_sched_barrier(0);
    qk(nxt, n + 1);
    probs(cur, n);
    if constexpr (!KV8) px_interleave<0, 4, ST * KK, CG, 8>();
    // P(n) is formed here, among the matrix instructions of S(n + 1), not moved down to its use
#pragma unroll
    for (int tw = 0; tw < TPW; ++tw)
#pragma unroll
      for (int cg = 0; cg < CG; ++cg) asm volatile("" : "+v"(pb[tw][cg]));
    __builtin_amdgcn_sched_barrier(0);
    scale_mask(nxt, n + 1, bad >> (NS - 1) * TPS & BITS);   // looked up: up to step n + NS
    pv(n);
    row_max(nxt, n + 1);
    if constexpr (!KV8) px_interleave<1, 8, TPW * DT, CG, 4>();
    rescale();
    arrive(n + 1);
  };
  if (idle) {   // the same requests and barriers
    arrive(0);
    for (int n = 0; n + 1 < n_steps; ++n) {
      request(n + NS - 1);
      arrive(n + 1);
    }
  } else {
    first();
    int n = 0;
    for (; n + 2 < n_steps; n += 2) {
      step(sa, sb, n);
      step(sb, sa, n + 1);
    }
    if (n + 1 < n_steps) {
      step(sa, sb, n);
      probs(sb, n + 1);
      pv(n + 1);
    } else {
      probs(sa, n);
      pv(n);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): the requests past the range land before the slots are reused
  __syncthreads();
#pragma unroll
  for (int cg = 0; cg < CG; ++cg) {
    m[cg] *= c2;   // log2 units from here on
    l[cg] += __shfl_xor(l[cg], 16, kWave);
    l[cg] += __shfl_xor(l[cg], 32, kWave);
    if constexpr (KV8) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt][cg] *= r;
    }
  }
  if constexpr (KH > 1) {
    // the other key groups' states into group 0's
    f4_t* mg = reinterpret_cast<f4_t*>(smem);
    if (kg > 0 && !idle) {
      f4_t* w = mg + ((kg - 1) * RG + rg) * kWave * (P::STATE / 4) + lane;
      *w = f4_t{m[0], l[0], m[1], l[1]};
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int cg = 0; cg < CG; ++cg) *(w += kWave) = o[dt][cg];
    }
    __syncthreads();
    if (kg == 0 && !idle) {
#pragma unroll
      for (int k = 1; k < KH; ++k) {
        const f4_t* w = mg + ((k - 1) * RG + rg) * kWave * (P::STATE / 4) + lane;
        const f4_t ml = *w;
        float f0[CG], f1[CG];
#pragma unroll
        for (int cg = 0; cg < CG; ++cg) {
          const float m1 = ml[2 * cg], M = fmaxf(m[cg], m1);
          f0[cg] = m[cg] == M ? 1.f : __builtin_amdgcn_exp2f(m[cg] - M);
          f1[cg] = m1 == M ? 1.f : __builtin_amdgcn_exp2f(m1 - M);
          m[cg] = M;
          l[cg] = l[cg] * f0[cg] + ml[2 * cg + 1] * f1[cg];
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int cg = 0; cg < CG; ++cg) {
            const f4_t p = *(w += kWave);
            o[dt][cg] = o[dt][cg] * f0[cg] + p * f1[cg];
          }
      }
    }
  }
  if (kg == 0) {
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) {
      const int row = rg * 32 + cg * 16 + h;
      if (r0 + row >= R) continue;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f4_t*>(o_out + (int64_t)row * HD + dt * 16 + 4 * j) = o[dt][cg];
      if (j == 0) {
        ml_out[2 * row] = m[cg];
        ml_out[2 * row + 1] = l[cg];
      }
    }
  }
}

// Blocks that take the prefix, of kPxBlocks; the others take the far own tiles.  Costs
// in block time, microseconds: a step of the prefix and the chain of a piece of it, an
// own step.
template <int HD, int F, int ROWS>
__device__ __forceinline__ int px_pre_blocks(int64_t pre_steps, int64_t pre_items, int64_t own_steps) {
  using P = PxForm<HD, F, ROWS>;
  if (own_steps == 0) return kPxBlocks;
  if (pre_steps == 0) return 0;
  constexpr float tile = HD == 128 ? 0.8f : 0.4f;
  const float pre = (float)pre_steps * (P::TPS * tile * (ROWS <= 64 ? 1.f : ROWS == 128 ? 0.9f : 1.7f)) +
                    (float)min(pre_items, pre_steps) * (P::LDS ? 7.f : 3.f);
  const float own = (float)own_steps * (kPxWaves * tile);
  int n = (int)((float)kPxBlocks * pre / (pre + own) + 0.5f);
  n = max(n, kPxBlocks - (int)min(own_steps, (int64_t)kPxBlocks));   // no more blocks than steps
  n = min(n, (int)min(pre_steps, (int64_t)kPxBlocks));
  return min(max(n, 1), kPxBlocks - 1);
}

template <int HD, int F, int ROWS>
__global__ __launch_bounds__(kPxThreads, 2) void px_stage1(const PxArgs a) {
  using P = PxForm<HD, F, ROWS>;
  __shared__ __align__(16) _Float16 smem[P::SM];
  __shared__ __align__(16) float scl[P::SCL];
  __shared__ int64_t cum[kPxMaxBatch + 1];
  __shared__ int64_t part[kPxWaves];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lp = cut_len((int)load_ctl_u32(a.pre_len), a.pre_pages, a.pre.shift);
  const int lo = a.start ? max((int)load_ctl_u32(a.start), 0) : 0;
  // steps (8 tiles) of far own tiles before each sequence
  int64_t n2[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int b = 2 * threadIdx.x + i, hi = b < a.batch ? cut_len(a.len[b], a.max_pages, a.own.shift) : 0;
    const int tiles = hi > lo ? ((hi - 1) >> 5) - (lo >> 5) + 1 : 0;
    n2[i] = (tiles - px_near(a, tiles) + kPxWaves - 1) / kPxWaves;
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
  const int R = a.batch * a.g, n_rb = (R + ROWS - 1) / ROWS, ptiles = (lp + 31) >> 5, steps = px_prefix_near(a.batch * a.n_kv, ptiles, F != CQ_KV_FP16) ? 0 : (ptiles + P::TPS - 1) / P::TPS;
  const int64_t pre_steps = (int64_t)a.n_kv * n_rb * steps, own_steps = cum[a.batch] * a.n_kv;
  const int n_pre = px_pre_blocks<HD, F, ROWS>(pre_steps, a.n_kv * n_rb, own_steps);
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b <= a.batch; b += kPxThreads) a.plan[b] = cum[b];
  int64_t at, end;
  if ((int)blockIdx.x < n_pre) {
    const int w = blockIdx.x;
    share_of(w, pre_steps, n_pre, &at, &end);
    while (at < end) {
      const int item = (int)px_div(at, steps), sa = (int)(at - (int64_t)item * steps), kvh = item / n_rb, rb = item % n_rb;
      const int sb = (int)min((int64_t)steps, sa + (end - at));
      float *o = a.pre_o + (int64_t)(w + item) * ROWS * HD, *ml = a.pre_ml + (int64_t)(w + item) * ROWS * 2;
      const int tb = sa * P::TPS, te = min(sb * P::TPS, ptiles);
      if (threadIdx.x == 0 && sa == 0) a.pre_items[2 * item] = w;
      if (threadIdx.x == 0 && sb == steps) a.pre_items[2 * item + 1] = w;
      if constexpr (P::LDS) px_shared_piece<HD, F, ROWS>(a, smem, scl, kvh, rb * ROWS, R, lp, tb, te, o, ml);
      else {
        const PxKV kv{a.pre, a.pre_layer + kvh * a.pre.head_stride, a.pre_table, 0, lp};
        px_stream_piece<HD, F, P::RG>(a, kv, reinterpret_cast<float*>(smem), kvh, rb * ROWS, R, tb, te, o, ml);
      }
      at += sb - sa;
    }
    return;
  }
  const int w = blockIdx.x - n_pre;
  share_of(w, own_steps, kPxBlocks - n_pre, &at, &end);
  while (at < end) {
    int b = 0, top = a.batch;   // last b with n_kv * cum[b] <= at
    while (top - b > 1) {
      const int mid = (b + top) / 2;
      if (cum[mid] * a.n_kv <= at) b = mid; else top = mid;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    const int ns = (int)(cum[b + 1] - cum[b]);
    const int64_t in = at - cum[b] * a.n_kv;
    const int kvh = (int)px_div(in, ns), sa = (int)(in - (int64_t)kvh * ns), item = b * a.n_kv + kvh;
    const int sb = (int)min((int64_t)ns, sa + (end - at));
    if (threadIdx.x == 0 && sa == 0) a.own_items[2 * item] = w;
    if (threadIdx.x == 0 && sb == ns) a.own_items[2 * item + 1] = w;
    const int hi = cut_len((int)load_ctl_u32(a.len + b), a.max_pages, a.own.shift), t0 = lo >> 5;
    const PxKV kv{a.own, a.own_layer + kvh * a.own.head_stride, a.table + (int64_t)b * a.max_pages, lo, hi};
    px_stream_piece<HD, F, 1>(a, kv, reinterpret_cast<float*>(smem), kvh, b * a.g, (b + 1) * a.g, t0 + sa * kPxWaves,
                              min(t0 + sb * kPxWaves, ((hi - 1) >> 5) + 1), a.own_o + (int64_t)(w + item) * 16 * HD,
                              a.own_ml + (int64_t)(w + item) * 32);
    at += sb - sa;
  }
}

// The pieces of one row: row `at` of o and ml is its first, the next lies `stride` rows on.
struct PxPieces {
  uint32_t at, stride;
  int n;
};

// Running sum of one row's pieces for 4 dims: m, l as in a wave's state.
struct PxSum {
  float m, l;
  f4_t o;
};

// Pieces p0, p0 + step, ... of a row into s, U requested at a time.
template <int HD>
__device__ __forceinline__ void px_add_pieces(PxSum& s, const float* o, const float* ml, const PxPieces& pc, int p0, int step, int d4) {
  constexpr int U = 8;
#pragma unroll 1
  for (int p = p0; p < pc.n; p += U * step) {
    float m1[U], l1[U];
    f4_t v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {   // the workspace is smaller than 2^31 bytes
      const uint32_t at = pc.at + (uint32_t)min(p + u * step, pc.n - 1) * pc.stride;
      m1[u] = ml[at * 2];
      l1[u] = ml[at * 2 + 1];
      v[u] = *reinterpret_cast<const f4_t*>(o + (at * HD + 4 * d4));
    }
    float M = s.m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p + u * step >= pc.n) m1[u] = -INFINITY;
      M = fmaxf(M, m1[u]);
    }
    const float mm = M == -INFINITY ? 0.f : M;   // nothing seen yet: weights of 0
    const float f0 = __builtin_amdgcn_exp2f(s.m - mm);
    s.m = M;
    s.l *= f0;
    s.o *= f0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float f = __builtin_amdgcn_exp2f(m1[u] - mm);
      s.l += l1[u] * f;
      s.o += v[u] * f;
    }
  }
}

// Block (sequence b, kv head; rows [per * y, per * (y + 1)) of its group): with PIECES those that stage 1 left, HD / 4 threads to a
// row and several of its pieces at a time (while the first tiles are on their way);
// the near own tiles (and a near prefix's), W waves taking every W-th.  All join in LDS.
template <int HD, int F, int W, bool PIECES>
__global__ __launch_bounds__(W * kWave, 2) void px_finish(const PxArgs a, int rows, int per) {
  constexpr int DT = HD / 16;
  constexpr int TP = HD / 4, G = W * kWave / TP;   // threads of a row; rows (or parts of one row's pieces) at a time
  __shared__ __align__(16) float sm[W * 16 * HD];
  __shared__ __align__(8) float sml[W * 16 * 2];
  __shared__ __align__(16) f4_t po_[PIECES ? G : 1][TP];
  __shared__ float pm_[PIECES ? G : 1], pl_[PIECES ? G : 1];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int h = lane & 15;
  const int rs = blockIdx.y, b = blockIdx.x / a.n_kv, kvh = blockIdx.x - b * a.n_kv;
  const int len = (int)load_ctl_u32(a.len + b);
  const int lp = cut_len((int)load_ctl_u32(a.pre_len), a.pre_pages, a.pre.shift);
  const int lo = a.start ? max((int)load_ctl_u32(a.start), 0) : 0;
  if (len < 0) return;
  const int hi = cut_len(len, a.max_pages, a.own.shift), t0 = lo >> 5;
  const int ptiles = (lp + 31) >> 5, mine = hi > lo ? ((hi - 1) >> 5) - t0 + 1 : 0;
  const bool pre_near = !PIECES || px_prefix_near(a.batch * a.n_kv, ptiles, F != CQ_KV_FP16);
  const int n0 = pre_near ? ptiles : 0, n = n0 + (PIECES ? px_near(a, mine) : mine);
  const PxKV pre{a.pre, a.pre_layer + kvh * a.pre.head_stride, a.pre_table, 0, lp};
  const PxKV own{a.own, a.own_layer + kvh * a.own.head_stride, a.table + (int64_t)b * a.max_pages, lo, hi};
  // rows side by side: a power of two that holds the group's; the other threads share a row's pieces
  const int row0 = rs * per, own_rows = min(per, a.g - row0);
  const int rp = per <= 1 ? 1 : 1 << (32 - __builtin_clz(per - 1)), gi = threadIdx.x / TP, d4 = threadIdx.x % TP;
  const int my = gi & (rp - 1), part = gi / rp, parts = G / rp;
  PxSum sum{-INFINITY, 0.f, f4_t{0.f, 0.f, 0.f, 0.f}};
  PxPieces pc[2] = {};
  if constexpr (PIECES) {
    // (the lists of pieces are read whether or not there are any: nothing waits for the plan)
    const int row = b * a.g + row0 + min(my, own_rows - 1), pi = kvh * ((a.batch * a.g + rows - 1) / rows) + row / rows, oi = b * a.n_kv + kvh;
    const int64_t c0 = a.plan[b], c1 = a.plan[b + 1];
    const int pw = a.pre_items[2 * pi], pe = a.pre_items[2 * pi + 1], ow = a.own_items[2 * oi], oe = a.own_items[2 * oi + 1];
    if (!pre_near && my < own_rows) pc[0] = PxPieces{(uint32_t)((pw + pi) * rows + row % rows), (uint32_t)rows, pe - pw + 1};
    if (c1 > c0 && my < own_rows) pc[1] = PxPieces{(uint32_t)((ow + oi) * 16 + row - b * a.g), 16u, oe - ow + 1};
  }
  PxState<HD> st;
  px_run<HD, F, false>(
      st, a, kvh, b * a.g, a.g, wave, n, W, lane,
      [&](PxTile<HD, F>& t, int k) __attribute__((always_inline)) {
        const bool first = k < n0;
        px_load<HD, F>(t, first ? pre : own, first ? k : t0 + k - n0, k < n, lane);
      },
      [&]() __attribute__((always_inline)) {
        if constexpr (PIECES) {
#pragma unroll 1
          for (int s = 0; s < 2; ++s)
            px_add_pieces<HD>(sum, s ? a.own_o : a.pre_o, s ? a.own_ml : a.pre_ml, s ? pc[1] : pc[0], part, parts, d4);
        }
      });
  const int n_w = min(W, n);   // waves that had a tile
  if (wave < n_w) {
    f4_t* w = reinterpret_cast<f4_t*>(sm) + wave * DT * kWave + lane;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) w[dt * kWave] = st.o[dt];
    if (lane < 16) {
      sml[(wave * 16 + h) * 2] = st.m;
      sml[(wave * 16 + h) * 2 + 1] = st.l;
    }
  }
  if constexpr (PIECES) {
    po_[gi][d4] = sum.o;
    if (d4 == 0) pm_[gi] = sum.m, pl_[gi] = sum.l;
  }
  __syncthreads();
  // a thread per (row, 4 dims); loops short in code, for the sake of the instruction cache
  for (int r = gi; r < own_rows; r += G) {
    const int row = row0 + r, n_sum = PIECES ? parts : 0;
    float M = -INFINITY, L = 0.f;
#pragma unroll 4
    for (int k = 0; k < n_w; ++k) M = fmaxf(M, sml[(k * 16 + row) * 2]);
#pragma unroll 4
    for (int k = 0; k < n_sum; ++k) M = fmaxf(M, pm_[k * rp + r]);
    const float mm = M == -INFINITY ? 0.f : M;
    f4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = 0; k < n_w; ++k) {
      const float f = __builtin_amdgcn_exp2f(sml[(k * 16 + row) * 2] - mm);
      L += sml[(k * 16 + row) * 2 + 1] * f;
      O += reinterpret_cast<const f4_t*>(sm)[(k * DT + d4 / 4) * kWave + d4 % 4 * 16 + row] * f;
    }
#pragma unroll 4
    for (int k = 0; k < n_sum; ++k) {
      const float f = __builtin_amdgcn_exp2f(pm_[k * rp + r] - mm);
      L += pl_[k * rp + r] * f;
      O += po_[k * rp + r][d4] * f;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    h4_t v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (_Float16)(O[e] * inv);
    *reinterpret_cast<h4_t*>(a.out + b * a.out_stride + (kvh * a.g + row) * HD + 4 * d4) = v;
  }
}

// Query rows of a stage 1 block for R rows per kv head.  Many rows: 128 where a tile is
// 16 KB (half the pieces' bytes, which is what the end of the launch waits for), else 256
// (7B heads, 64 sequences over 8160, fp16: 30.0 us with 128, 32.5 with 256; E4M3 over 16000:
// 54.8 and 48.7; 0.5B heads, 128 over 4000: 25.0 and 20.0).
int px_rows(int64_t R, int hd, bool one_byte) {
  return R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : R <= 128 || (hd == 128 && !one_byte) ? 128 : 256;
}

// Workspace: plan, then (m, l) and O of the own pieces and of the prefix's.
struct PxSpace { size_t plan, pre_items, own_items, own_ml, own_o, pre_ml, pre_o, bytes; };
PxSpace px_space(int batch, int n_heads, int n_kv, int hd, bool one_byte) {
  const size_t R = (size_t)batch * (n_heads / n_kv), rows = px_rows(R, hd, one_byte);
  const size_t own = kPxBlocks + (size_t)batch * n_kv, pre = (kPxBlocks + n_kv * ((R + rows - 1) / rows)) * rows;
  size_t off = 0;
  auto take = [&](size_t n) { const size_t o = off; off += (n + 255) & ~(size_t)255; return o; };
  PxSpace s;
  s.plan = take((batch + 1) * sizeof(int64_t));
  s.pre_items = take(n_kv * ((R + rows - 1) / rows) * 2 * sizeof(int));
  s.own_items = take((size_t)batch * n_kv * 2 * sizeof(int));
  s.own_ml = take(own * 32 * 4);
  s.own_o = take(own * 16 * hd * 4);
  s.pre_ml = take(pre * 2 * 4);
  s.pre_o = take(pre * hd * 4);
  s.bytes = off;
  return s;
}

bool px_shape_ok(int batch, int n_heads, int n_kv, int hd) {
  return batch >= 0 && batch <= kPxMaxBatch && n_kv >= 1 && n_kv <= 64 && n_heads >= 1 && n_heads % n_kv == 0 &&
         n_heads / n_kv <= 16 && (hd == 64 || hd == 128);
}

template <int HD, int F, int ROWS>
void px_launch_rows(const PxArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((px_stage1<HD, F, ROWS>), dim3(kPxBlocks), dim3(kPxThreads), 0, st, a);
}

// 8 waves a block while every block has a CU of its own (two sequences of 7B heads over
// 1000 tokens: 9.4 us, with 4 waves 10.7), then 4, two blocks to a CU (256 over 200: 14.3
// us, with 8 waves 22.3) unless the group has more rows than 4 waves hold side by side.
// Where blocks leave CUs idle several take the rows of one group, each with the pieces
// of its rows (and all of the own tiles).
template <int HD, int F, bool PIECES>
void px_launch_finish(const PxArgs& a, int rows, hipStream_t st) {
  const int blocks = a.batch * a.n_kv;
  const int split = PIECES ? std::max(1, std::min(a.g, kPxBlocks / blocks)) : 1, per = (a.g + split - 1) / split;
  const dim3 grid(blocks, (a.g + per - 1) / per);
  if (blocks <= kPxBlocks || a.g > 4 * kWave / (HD / 4)) hipLaunchKernelGGL((px_finish<HD, F, 8, PIECES>), grid, dim3(8 * kWave), 0, st, a, rows, per);
  else hipLaunchKernelGGL((px_finish<HD, F, 4, PIECES>), grid, dim3(4 * kWave), 0, st, a, rows, per);
}

template <int HD, int F>
void px_launch(const PxArgs& a, hipStream_t st) {
  // the most that the tables hold: short ones need no first launch
  const int64_t pre_tiles = (int64_t)a.pre_pages << (a.pre.shift - 5), own_tiles = (int64_t)a.max_pages << (a.own.shift - 5);
  constexpr bool ONE = F != CQ_KV_FP16;
  const int rows = px_rows((int64_t)a.batch * a.g, HD, ONE);
  if (own_tiles <= 64 && px_prefix_near(a.batch * a.n_kv, pre_tiles, ONE)) {
    px_launch_finish<HD, F, false>(a, rows, st);
    return;
  }
  switch (rows) {
    case 16: px_launch_rows<HD, F, 16>(a, st); break;
    case 32: px_launch_rows<HD, F, 32>(a, st); break;
    case 64: px_launch_rows<HD, F, 64>(a, st); break;
    case 128: px_launch_rows<HD, F, 128>(a, st); break;
    default:
      if constexpr (HD != 128 || ONE) px_launch_rows<HD, F, 256>(a, st);
  }
  px_launch_finish<HD, F, true>(a, rows, st);
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
  if (!px_shape_ok(batch, n_heads, n_kv_heads, head_dim)) return 0;
  // of either kind of cache
  return std::max(px_space(batch, n_heads, n_kv_heads, head_dim, false).bytes, px_space(batch, n_heads, n_kv_heads, head_dim, true).bytes);
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
  constexpr int64_t most = (int64_t)1 << 30;   // tile numbers and their positions stay far below 2^31
  if (prefix_pages < 1 || max_pages < 1 || (int64_t)prefix_pages * prefix->page_tokens > most || (int64_t)max_pages * own->page_tokens > most)
    return fail(CQ_EINVAL, "prefix attention: a table holds 1 to 2^30 positions");
  const PxSpace s = px_space(batch, n_heads, own->n_kv_heads, own->head_dim, own->kv_dtype != CQ_KV_FP16);
  char* ws = (char*)workspace;
  PxArgs a{};
  a.q = (const _Float16*)q; a.out = (_Float16*)out; a.q_stride = q_stride; a.out_stride = out_stride;
  a.pre = page_view(*prefix); a.own = page_view(*own);
  a.pre_layer = layer * prefix->layer_stride; a.own_layer = layer * own->layer_stride;
  a.pre_table = d_prefix_table; a.pre_len = d_prefix_len; a.table = d_table; a.start = d_start; a.len = d_len;
  a.pre_pages = prefix_pages; a.max_pages = max_pages;
  a.batch = batch; a.n_kv = own->n_kv_heads; a.g = n_heads / own->n_kv_heads;
  a.plan = (int64_t*)(ws + s.plan);
  a.pre_items = (int*)(ws + s.pre_items);
  a.own_items = (int*)(ws + s.own_items);
  a.own_ml = (float*)(ws + s.own_ml); a.own_o = (float*)(ws + s.own_o);
  a.pre_ml = (float*)(ws + s.pre_ml); a.pre_o = (float*)(ws + s.pre_o);
  const hipStream_t st = (hipStream_t)stream;
  if (own->head_dim == 128) px_format<128>(a, own->kv_dtype, st);
  else px_format<64>(a, own->kv_dtype, st);
  CQ_HIP(hipGetLastError());
  return CQ_OK;
}
