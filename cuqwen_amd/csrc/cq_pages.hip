// Pages of a KV cache shared by several sequences: fork, append (with copy on
// write), trim, compact and copy.  No counterpart in the reference.
//
// The page map (counts, tables, lengths) lives on the device and is changed by
// kernels alone, so a decode loop over a batch needs no host round trip and can
// be captured.  Which pages a call takes or moves is decided by one block
// (every sequence a thread, the counts read once in page order), a second launch
// moves the bytes: allocation in order is what makes the outcome independent of
// timing, and a few hundred to a few thousand words are one block's work.
#include "cq_pages.h"

#include <algorithm>

namespace cq {

namespace {

// ------------------------------------------------------------- page copies
// What bounds it: HBM, at 2 bytes moved per byte copied.  A wave takes one run (a
// page's K or V of one head in one layer, 2-32 KB and contiguous in every layout)
// at a time, four 1 KB requests in flight, as many waves as the chip holds.  int8 pages of
// 32768 tokens, 6 layers of 7B heads: 415 MB moved in 88 us, 4.7 TB/s (a plain copy of 2 GiB:
// 4.9); 48 of 96 sequences' pages moved together, 923 MB: 182 us, 5.1 TB/s.
constexpr int kCopyThreads = 256, kCopyBlocks = 2048;

struct CopyGeo {
  int n_layers, n_kv, run16;   // 16-byte pieces of a whole run
  int tokens, srow16;          // page tokens; a page's scales of one head in 16-byte pieces (0: fp16)
  int64_t hd;                  // elements per scale
  int es;                      // bytes per element
};

__device__ __forceinline__ void copy_run(const u4_t* s, u4_t* d, int n, int lane) {
  int i = lane;
  for (; i + 3 * kWave < n; i += 4 * kWave) {
    const u4_t a = load_u4_stream(s + i), b = load_u4_stream(s + i + kWave);
    const u4_t c = load_u4_stream(s + i + 2 * kWave), e = load_u4_stream(s + i + 3 * kWave);
    d[i] = a; d[i + kWave] = b; d[i + 2 * kWave] = c; d[i + 3 * kWave] = e;
  }
  for (; i < n; i += kWave) d[i] = load_u4_stream(s + i);
}

// Run `part` of a page: K or V, kv head, layer (part = (layer * 2 + kind) * n_kv + head).
__device__ __forceinline__ void copy_part(const PageView& from, const PageView& to, const CopyGeo& g, int src, int dst, int part,
                                          int tokens, int lane) {
  const int head = part % g.n_kv, kind = part / g.n_kv % 2, layer = part / (2 * g.n_kv);
  const int64_t s = layer * from.layer_stride + src * from.page_stride + head * from.head_stride;
  const int64_t d = layer * to.layer_stride + dst * to.page_stride + head * to.head_stride;
  const int shift = __builtin_ctz(g.tokens);
  copy_run((const u4_t*)(from.kv[kind] + s * g.es), (u4_t*)(to.kv[kind] + d * g.es), (int)((int64_t)g.run16 * tokens >> shift), lane);
  if (g.srow16)
    copy_run((const u4_t*)(from.scale[kind] + s / g.hd), (u4_t*)(to.scale[kind] + d / g.hd), (int)((int64_t)g.srow16 * tokens >> shift), lane);
}

// Pairs (src[i], dst[i]), i < *d_n, of one pool, the first tokens[i] tokens of each
// (nullptr: whole pages); the lists come from the planning launch before.
__device__ __forceinline__ void copy_pairs(const PageView& pv, const CopyGeo& g, int n, const int* src, const int* dst,
                                           const int* tokens, int wave, int n_waves, int lane) {
  const int parts = g.n_layers * 2 * g.n_kv;
  const int64_t units = (int64_t)n * parts;
  for (int64_t u = wave; u < units; u += n_waves) {
    const int i = (int)(u / parts);
    copy_part(pv, pv, g, src[i], dst[i], (int)(u - (int64_t)i * parts), tokens ? tokens[i] : g.tokens, lane);
  }
}

// cq_pages_copy.  A wave takes consecutive units, so it meets few pairs, and looks
// through the lists for another use of its pair's target each time the pair changes:
// a check in front of the copy would be a launch of its own.
__global__ __launch_bounds__(kCopyThreads) void copy_pages_kernel(PageView from, PageView to, CopyGeo g, const int* src,
                                                                  const int* dst, int n, bool same, int* status) {
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * (kCopyThreads / kWave) + threadIdx.x / kWave);
  const int n_waves = gridDim.x * (kCopyThreads / kWave);
  const int parts = g.n_layers * 2 * g.n_kv;
  const int64_t units = (int64_t)n * parts;
  int64_t u = units * wave / n_waves;
  const int64_t end = units * (wave + 1) / n_waves;
  int pair = -1, code = CQ_OK, a = 0, b = 0;
  for (; u < end; ++u) {
    const int i = (int)(u / parts), part = (int)(u - (int64_t)i * parts);
    if (i != pair) {
      pair = i;
      a = __builtin_amdgcn_readfirstlane(src[i]);
      b = __builtin_amdgcn_readfirstlane(dst[i]);
      bool clash = false;
      for (int k = lane; k < n; k += kWave) clash |= k != i && (dst[k] == b || (same && src[k] == b));
      code = a < 0 || a >= from.n_pages || b < 0 || b >= to.n_pages ? CQ_ERANGE : __any(clash) ? CQ_EINVAL : CQ_OK;
    }
    if (part == 0 && lane == 0) status[i] = code;
    if (code == CQ_OK && !(same && a == b)) copy_part(from, to, g, a, b, part, g.tokens, lane);
  }
}

// -------------------------------------------------------------- fork, trim
// A block takes kSeqGroup entries, thread (column, entry) with the entry in the lowest
// lane bits: siblings name the same page in the same column, so the first lane of a run
// of equal pages counts for the whole run (64 forks of a prompt of 313 pages: 2504 atomics
// instead of 20032).  Integer sums: the order of the atomics does not show.
// What bounds them: the launch, three memory round trips (the lists; the lengths; the
// table) and the fetch of their code, which is why a thread looks after one entry only
// (a thread following a column through eight entries: fork 7.6 us for 64 x 313, trim 8.8;
// so 5.4 and 4.8).
// Lengths are written once every thread of the block has read them; no entry that
// another block carries out has the same sequence.
constexpr int kSeqGroup = 8, kMapThreads = 1024, kMapCols = kMapThreads / kSeqGroup;

__device__ __forceinline__ int pages_of(int tokens, int page_tokens) { return (int)(((int64_t)tokens + page_tokens - 1) / page_tokens); }

// Whether some k in [0, n) is bad(k) for this thread's entry.  `flags`: a word of LDS.
template <class Bad>
__device__ __forceinline__ bool entry_clashes(int n, int q, int* flags, Bad bad) {
  if (threadIdx.x == 0) *flags = 0;
  bool mine = false;
#pragma unroll 1
  for (int k = threadIdx.x / kSeqGroup; k < n; k += kMapCols) mine |= bad(k);
  __syncthreads();
  if (mine) atomicOr(flags, 1 << q);
  __syncthreads();
  return *flags >> q & 1;
}

// Adds `sign` to the count of page id (-1: none) for each lane, a run of equal ids among
// the lanes of one column at once.
__device__ __forceinline__ void count_pages(int* ref, int n_pages, int id, int q, int sign) {
  const int left = __shfl_up(id, 1, kWave);   // by every lane, those of entry 0 too
  const bool same = q > 0 && left == id;
  const unsigned long long follows = __ballot(same);
  if (same || id < 0 || id >= n_pages) return;
  const int lane = threadIdx.x & (kWave - 1);
  const int run = 1 + __builtin_ctzll(~(follows >> lane >> 1));
  atomicAdd(ref + id, sign * run);
}

__global__ __launch_bounds__(kMapThreads) void fork_kernel(cq_page_map m, const int* parent, const int* child, int n,
                                                           int* status) {
  __shared__ int flags;
  const int q = threadIdx.x % kSeqGroup, i = blockIdx.x * kSeqGroup + q;
  const int p = i < n ? parent[i] : -1, c = i < n ? child[i] : -1;
  const bool ok = p >= 0 && p < m.n_seqs && c >= 0 && c < m.n_seqs;
  const int len = ok ? m.len[p] : 0, old = ok ? m.len[c] : 0;
  const bool clash = entry_clashes(n, q, &flags, [&](int k) {
    const int x = child[k];
    return x == p || (k < i && x == c);
  });
  const int code = !ok ? CQ_ERANGE : clash || old != 0 ? CQ_EINVAL
                 : len < 0 || (int64_t)len > (int64_t)m.max_pages * m.page_tokens ? CQ_ERANGE : CQ_OK;
  const int held = code == CQ_OK ? pages_of(len, m.page_tokens) : 0;
  if (threadIdx.x < kSeqGroup && i < n) {
    status[i] = code;
    if (code == CQ_OK) m.len[c] = len;
  }
  for (int col = threadIdx.x / kSeqGroup; __any(col < held); col += kMapCols) {
    int id = -1;
    if (col < held) {
      id = m.table[(int64_t)p * m.max_pages + col];
      m.table[(int64_t)c * m.max_pages + col] = id;
    }
    count_pages(m.ref, m.n_pages, id, q, 1);
  }
}

__global__ __launch_bounds__(kMapThreads) void trim_kernel(cq_page_map m, const int* seq, const int* keep, int n, int* status) {
  __shared__ int flags;
  const int q = threadIdx.x % kSeqGroup, i = blockIdx.x * kSeqGroup + q;
  const int s = i < n ? seq[i] : -1, want = i < n && keep ? keep[i] : 0;
  const bool ok = s >= 0 && s < m.n_seqs && want >= 0;
  const int len = ok ? m.len[s] : 0;
  const bool clash = entry_clashes(n, q, &flags, [&](int k) { return k < i && seq[k] == s; });
  const int code = !ok ? CQ_ERANGE : clash ? CQ_EINVAL : len < 0 || (int64_t)len > (int64_t)m.max_pages * m.page_tokens ? CQ_ERANGE : CQ_OK;
  const bool go = code == CQ_OK && want < len;
  const int kept = go ? pages_of(want, m.page_tokens) : 0, held = go ? pages_of(len, m.page_tokens) : 0;
  if (threadIdx.x < kSeqGroup && i < n) {
    status[i] = code;
    if (go) m.len[s] = want;
  }
  for (int col = threadIdx.x / kSeqGroup; __any(col < held); col += kMapCols) {
    int id = -1;
    if (col >= kept && col < held) {
      int* at = m.table + (int64_t)s * m.max_pages + col;
      id = *at;
      *at = -1;
    }
    count_pages(m.ref, m.n_pages, id, q, -1);
  }
}

// ------------------------------------------------------------------ append
// The plan is one block's chain of round trips (lengths, last pages and their counts, the
// free pages in order, the new table entries): 4 to 6 us.  The second launch writes the
// slots and makes the copies on write (64 answers branching off a page of 43 tokens, 8
// layers of 7B heads: 134 MB in 23 us, part of it from the Infinity Cache).
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / kWave;
static_assert(kPlanThreads == kMaxSeqs, "a thread per sequence");

// Workspace of append and compact, in ints.  Append: [copies, tokens (-1: refused)]
// [first token of each sequence, n_seqs][length before, n_seqs][copy source, target,
// tokens: n_seqs each][pages taken, in order].  Compact: [moves][targets][sources].
constexpr int kHead = 16;
inline size_t map_workspace_ints(int n_seqs, int n_pages) {
  return kHead + std::max<size_t>((size_t)5 * n_seqs + n_pages, (size_t)2 * n_pages);
}

// Inclusive sum over the wave on DPP lane moves (rows of 16, then across rows).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int wave_scan(int v) {
  v = dpp_add<0x111, 0xf>(v);   // row_shr 1, 2, 4, 8
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);   // row_bcast 15 into rows 1 and 3
  return dpp_add<0x143, 0xc>(v);   // row_bcast 31 into rows 2 and 3
}

// Exclusive sums of four values over the block at once, and the whole sums.
struct Four { int v[4]; };
__device__ __forceinline__ Four block_scan(Four x, Four (*part), Four* total) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  Four s;
#pragma unroll
  for (int i = 0; i < 4; ++i) s.v[i] = wave_scan(x.v[i]);
  if (lane == kWave - 1) part[wave] = s;
  __syncthreads();
  Four all = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) s.v[i] -= x.v[i];
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    const Four p = part[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (w < wave) s.v[i] += p.v[i];
      all.v[i] += p.v[i];
    }
  }
  *total = all;
  return s;
}

// Pages [begin, n_pages) in order, kPlanThreads * 4 at a time: calls take(page, rank)
// for those that satisfy `pick`, rank counting them from 0; ends once `enough` have
// been found.  Returns how many were found.
template <class Pick, class Take>
__device__ __forceinline__ int in_page_order(const int* ref, int begin, int n_pages, int enough, int* part, Pick pick,
                                             Take take) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  int found = 0;
  for (int base = begin; base < n_pages && found < enough; base += 4 * kPlanThreads) {
    const int p0 = base + wave * 4 * kWave + lane;
    int r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = p0 + i * kWave < n_pages ? ref[p0 + i * kWave] : 0;
    unsigned long long hit[4];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hit[i] = __ballot(p0 + i * kWave < n_pages && pick(p0 + i * kWave, r[i]));
      mine += __popcll(hit[i]);
    }
    __syncthreads();
    if (lane == 0) part[wave] = mine;
    __syncthreads();
    int rank = found, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
      if (w < wave) rank += part[w];
      all += part[w];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (hit[i] >> lane & 1) take(p0 + i * kWave, rank + __popcll(hit[i] & ((1ull << lane) - 1)));
      rank += __popcll(hit[i]);
    }
    found += all;
  }
  return found;
}

// Last i in [0, n) with v[i] <= x (v ascending, v[0] <= x).
__device__ __forceinline__ int last_at_most(const int* v, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (v[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kPlanThreads) void append_plan_kernel(cq_page_map m, const int* add, int n_slots, int* status,
                                                                   int* ws) {
  __shared__ __align__(16) int last_of[kMaxSeqs];
  __shared__ int part[kPlanWaves], first_of[kMaxSeqs], flag, near[kMaxSeqs];
  __shared__ int before_of[kMaxSeqs], copy_of[kMaxSeqs];   // pages before; index of the copy, -1: none
  __shared__ Four part4[kPlanWaves];
  const int s = threadIdx.x, n = m.n_seqs, pt = m.page_tokens;
  int* tok0 = ws + kHead;
  int *len0 = tok0 + n, *csrc = len0 + n, *cdst = csrc + n, *ctok = cdst + n, *list = ctok + n;
  if (s == 0) flag = 0;
  const int most = m.max_pages * pt;   // below 2^31 (checked by the host)
  int a = s < n ? add[s] : 0, len = s < n ? m.len[s] : 0;
  bool bad = a < 0 || len < 0 || len > most || a > most - len;
  if (bad) a = len = 0;
  const int before = pages_of(len, pt), after = pages_of(len + a, pt);
  int last = -1, holders = 0;
  if (a > 0 && len % pt != 0) {   // it writes into the last page it holds
    last = m.table[(int64_t)s * m.max_pages + before - 1];
    if (last < 0 || last >= m.n_pages) bad = true, last = -1;
    else holders = m.ref[last];
  }
  last_of[s] = last;
  __syncthreads();
  if (bad) flag = 1;
  // writers of this page in earlier sequences: those that leave it for a copy count no longer
  bool copy = false;
  if (holders > 1) {
    int earlier = 0;
    for (int q = 0; q < s; q += 4) {
      const int4 v = *reinterpret_cast<const int4*>(last_of + q);
      earlier += (v.x == last) + (q + 1 < s && v.y == last) + (q + 2 < s && v.z == last) + (q + 3 < s && v.w == last);
    }
    copy = holders - earlier > 1;
  }
  // tokens in two halves of 16 bits (their sum may pass 32), pages, copies
  Four sum;
  const Four base = block_scan(Four{{a & 0xffff, a >> 16, after - before + copy, copy}}, part4, &sum);
  const long long tokens = ((long long)sum.v[1] << 16) + sum.v[0];
  const bool refused = flag != 0 || tokens > n_slots;   // the scan's barrier lies between
  const int pages = refused ? 0 : sum.v[2], copies = refused ? 0 : sum.v[3];   // pages: at most n_slots / 32 + 2 n_seqs
  const int t0 = (base.v[1] << 16) + base.v[0], p0 = base.v[2], c0 = base.v[3];
  first_of[s] = p0;
  before_of[s] = before;
  copy_of[s] = copy ? c0 : -1;
  int code = refused ? CQ_ERANGE : CQ_OK;
  if (pages > 0) {
    const int found = in_page_order(m.ref, 0, m.n_pages, pages, part, [](int, int r) { return r <= 0; }, [&](int p, int rank) {
      if (rank < kMaxSeqs) near[rank] = p;
      else if (rank < pages) list[rank] = p;
    });
    if (found < pages) code = CQ_ENOMEM;
  }
  if (s == 0) {
    status[0] = code;
    status[1] = pages;
    status[2] = copies;
    status[3] = refused ? 0 : (int)tokens;
    ws[0] = code == CQ_OK ? copies : 0;
    ws[1] = code == CQ_OK ? (int)tokens : -1;
  }
  if (code != CQ_OK) return;
  if (s < n) {
    tok0[s] = t0;
    len0[s] = len;
    if (copy) {
      csrc[c0] = last;
      ctok[c0] = (len % pt + 31) & ~31;
      atomicSub(m.ref + last, 1);
    }
    if (a > 0) m.len[s] = len + a;
  }
  if (pages == 0) return;
  __syncthreads();   // the list is written
  for (int r = s; r < pages; r += kPlanThreads) {
    const int p = r < kMaxSeqs ? near[r] : list[r], q = last_at_most(first_of, n, r);
    int col = before_of[q] + r - first_of[q];
    if (copy_of[q] >= 0) {
      --col;   // its own copy of the last page first
      if (r == first_of[q]) cdst[copy_of[q]] = p;
    }
    m.table[(int64_t)q * m.max_pages + col] = p;
    m.ref[p] = 1;
  }
}

// Slots of the new tokens (the first slot_blocks blocks) and the copies on write.
__global__ __launch_bounds__(kCopyThreads) void append_apply_kernel(PageView pv, CopyGeo g, cq_page_map m, int* slots,
                                                                    int n_slots, int slot_blocks, const int* ws) {
  __shared__ int tok0[kMaxSeqs];
  const int n = m.n_seqs;
  const int* w_tok0 = ws + kHead;
  const int *len0 = w_tok0 + n, *csrc = len0 + n, *cdst = csrc + n, *ctok = cdst + n;
  if ((int)blockIdx.x < slot_blocks) {
    const int tokens = ws[1], stride = slot_blocks * kCopyThreads, mask = (1 << pv.shift) - 1;
    if (tokens > 0)
      for (int i = threadIdx.x; i < n; i += kCopyThreads) tok0[i] = w_tok0[i];
    __syncthreads();
    for (int64_t t = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; t < n_slots; t += stride) {
      int slot = -1;
      if (t < tokens) {
        const int q = last_at_most(tok0, n, (int)t), pos = len0[q] + (int)t - tok0[q];
        slot = (m.table[(int64_t)q * m.max_pages + (pos >> pv.shift)] << pv.shift) | (pos & mask);
      }
      slots[t] = slot;
    }
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane((blockIdx.x - slot_blocks) * (kCopyThreads / kWave) + threadIdx.x / kWave);
  copy_pairs(pv, g, ws[0], csrc, cdst, ctok, wave, (gridDim.x - slot_blocks) * (kCopyThreads / kWave), threadIdx.x & (kWave - 1));
}

// ----------------------------------------------------------------- compact
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(cq_page_map m, int* remap, int* status, int* ws) {
  __shared__ int part[kPlanWaves];
  int *to = ws + kHead, *from = to + m.n_pages;
  const int all = 0x7fffffff;
  const int used = in_page_order(m.ref, 0, m.n_pages, all, part, [](int, int r) { return r > 0; }, [](int, int) {});
  const int holes = in_page_order(m.ref, 0, used, all, part, [&](int p, int r) { remap[p] = r > 0 ? p : -1; return r <= 0; },
                                  [&](int p, int rank) { to[rank] = p; });
  const int moves = in_page_order(m.ref, used, m.n_pages, all, part, [&](int p, int r) { remap[p] = -1; return r > 0; },
                                  [&](int p, int rank) { from[rank] = p; });
  __syncthreads();
  for (int i = threadIdx.x; i < moves; i += kPlanThreads) {
    remap[from[i]] = to[i];
    m.ref[to[i]] = m.ref[from[i]];
    m.ref[from[i]] = 0;
  }
  if (threadIdx.x == 0) {
    ws[0] = moves;   // == holes
    status[0] = CQ_OK;
    status[1] = used;
    status[2] = holes;
    status[3] = 0;
  }
}

// Tables (the first table_blocks blocks) and the moves.
__global__ __launch_bounds__(kCopyThreads) void compact_apply_kernel(PageView pv, CopyGeo g, cq_page_map m, const int* remap,
                                                                     int table_blocks, const int* ws) {
  const int moves = ws[0];
  if (moves == 0) return;
  if ((int)blockIdx.x < table_blocks) {
    for (int s = blockIdx.x; s < m.n_seqs; s += table_blocks) {
      const int len = m.len[s];
      if (len <= 0) continue;
      const int held = min((int)(((int64_t)len + m.page_tokens - 1) / m.page_tokens), m.max_pages);
      int* row = m.table + (int64_t)s * m.max_pages;
      for (int c = threadIdx.x; c < held; c += kCopyThreads) {
        const int p = row[c];
        if (p < 0 || p >= m.n_pages) continue;
        const int q = remap[p];
        if (q >= 0 && q != p) row[c] = q;
      }
    }
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane((blockIdx.x - table_blocks) * (kCopyThreads / kWave) + threadIdx.x / kWave);
  copy_pairs(pv, g, moves, ws + kHead + m.n_pages, ws + kHead, nullptr, wave, (gridDim.x - table_blocks) * (kCopyThreads / kWave),
             threadIdx.x & (kWave - 1));
}

// ------------------------------------------------------------------- host
CopyGeo copy_geo(const cq_kv_pages& p) {
  CopyGeo g;
  g.n_layers = p.n_layers; g.n_kv = p.n_kv_heads; g.tokens = p.page_tokens; g.hd = p.head_dim;
  g.es = p.kv_dtype == CQ_KV_FP16 ? 2 : 1;
  g.run16 = p.page_tokens * p.head_dim * g.es / 16;
  g.srow16 = p.kv_dtype == CQ_KV_FP16 ? 0 : p.page_tokens * 4 / 16;
  return g;
}

int map_check(const cq_page_map* m) {
  if (!m || !m->ref || !m->table || !m->len) return fail(CQ_EINVAL, "page map: null pointer");
  if (m->n_seqs < 1 || m->n_seqs > kMaxSeqs) return fail(CQ_EINVAL, "page map: n_seqs outside [1, 1024]");
  if (m->page_tokens < 32 || m->page_tokens > kMaxPageTokens || (m->page_tokens & (m->page_tokens - 1)))
    return fail(CQ_EINVAL, "page map: page_tokens must be a power of two in [32, 32768]");
  if (m->n_pages < 1 || m->n_pages > kMaxPages || (int64_t)m->n_pages * m->page_tokens >= ((int64_t)1 << 31))
    return fail(CQ_EINVAL, "page map: n_pages outside [1, 2^20], or 2^31 slots or more");
  if (m->max_pages < 1 || (int64_t)m->max_pages * m->page_tokens >= ((int64_t)1 << 31))
    return fail(CQ_EINVAL, "page map: max_pages * page_tokens outside [1, 2^31)");
  return CQ_OK;
}

int pool_and_map_check(const cq_kv_pages* p, const cq_page_map* m) {
  CQ_TRY(pages_check(p));
  CQ_TRY(map_check(m));
  if (p->n_pages != m->n_pages || p->page_tokens != m->page_tokens) return fail(CQ_EINVAL, "pages: the pool and the map differ");
  return CQ_OK;
}

// Blocks for `units` runs, a wave each, at most what keeps every CU's waves busy; of
// more runs than that every wave takes the same number.
int copy_blocks(int64_t units) {
  const int64_t per = kCopyThreads / kWave, rounds = std::max<int64_t>(1, (units + kCopyBlocks * per - 1) / (kCopyBlocks * per));
  return (int)std::max<int64_t>(1, (units + rounds * per - 1) / (rounds * per));
}

hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }

}  // namespace

}  // namespace cq

using namespace cq;

extern "C" int cq_kv_pages_layout(int32_t kv_dtype, int32_t n_layers, int32_t n_pages, int32_t page_tokens,
                                  int32_t n_kv_heads, int32_t head_dim, cq_kv_pages* out, size_t* kv_bytes,
                                  size_t* scale_bytes) {
  if (!out) return fail(CQ_EINVAL, "pages: null description");
  CQ_TRY(pages_geometry_check(kv_dtype, n_layers, n_pages, page_tokens, n_kv_heads, head_dim));
  const int64_t run = (int64_t)page_tokens * head_dim;
  cq_kv_pages p{};
  p.head_stride = run;
  p.page_stride = run * n_kv_heads;
  p.layer_stride = p.page_stride * n_pages;
  p.kv_dtype = kv_dtype; p.n_layers = n_layers; p.n_pages = n_pages; p.page_tokens = page_tokens;
  p.n_kv_heads = n_kv_heads; p.head_dim = head_dim;
  *out = p;
  const size_t elems = (size_t)p.layer_stride * n_layers;
  if (kv_bytes) *kv_bytes = elems * (kv_dtype == CQ_KV_FP16 ? 2 : 1);
  if (scale_bytes) *scale_bytes = kv_dtype == CQ_KV_FP16 ? 0 : elems / head_dim * sizeof(float);
  return CQ_OK;
}

extern "C" size_t cq_pages_workspace_bytes(const cq_page_map* m) {
  if (!m || m->n_seqs <= 0 || m->n_pages <= 0) return 0;
  return map_workspace_ints(m->n_seqs, m->n_pages) * sizeof(int);
}

extern "C" int cq_pages_fork(const cq_page_map* m, const int32_t* d_parent, const int32_t* d_child, int32_t n,
                             int32_t* d_status, void* stream) {
  CQ_TRY(map_check(m));
  if (n < 0 || n > kMaxSeqs) return fail(CQ_EINVAL, "pages_fork: n outside [0, 1024]");
  if (n == 0) return CQ_OK;
  if (!d_parent || !d_child || !d_status) return fail(CQ_EINVAL, "pages_fork: null pointer");
  hipLaunchKernelGGL(fork_kernel, dim3((n + kSeqGroup - 1) / kSeqGroup), dim3(kMapThreads), 0, as_stream(stream), *m, d_parent,
                     d_child, n, d_status);
  CQ_HIP(hipGetLastError());
  return CQ_OK;
}

extern "C" int cq_pages_trim(const cq_page_map* m, const int32_t* d_seq, const int32_t* d_keep, int32_t n,
                             int32_t* d_status, void* stream) {
  CQ_TRY(map_check(m));
  if (n < 0 || n > kMaxSeqs) return fail(CQ_EINVAL, "pages_trim: n outside [0, 1024]");
  if (n == 0) return CQ_OK;
  if (!d_seq || !d_status) return fail(CQ_EINVAL, "pages_trim: null pointer");
  hipLaunchKernelGGL(trim_kernel, dim3((n + kSeqGroup - 1) / kSeqGroup), dim3(kMapThreads), 0, as_stream(stream), *m, d_seq,
                     d_keep, n, d_status);
  CQ_HIP(hipGetLastError());
  return CQ_OK;
}

extern "C" int cq_pages_append(const cq_kv_pages* pages, const cq_page_map* m, const int32_t* d_add, int32_t* d_slots,
                               int32_t n_slots, int32_t* d_status, void* workspace, void* stream) {
  CQ_TRY(pool_and_map_check(pages, m));
  if (!d_add || !d_status || !workspace || unaligned16(workspace) || n_slots < 0 || (n_slots > 0 && !d_slots))
    return fail(CQ_EINVAL, "pages_append: bad arguments");
  const hipStream_t st = as_stream(stream);
  hipLaunchKernelGGL(append_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, *m, d_add, n_slots, d_status, (int*)workspace);
  CQ_HIP(hipGetLastError());
  const int slot_blocks = (int)std::min<int64_t>(256, ((int64_t)n_slots + kCopyThreads - 1) / kCopyThreads);
  const int most = copy_blocks((int64_t)m->n_seqs * pages->n_layers * 2 * pages->n_kv_heads);
  hipLaunchKernelGGL(append_apply_kernel, dim3(slot_blocks + most), dim3(kCopyThreads), 0, st, page_view(*pages),
                     copy_geo(*pages), *m, d_slots, n_slots, slot_blocks, (const int*)workspace);
  CQ_HIP(hipGetLastError());
  return CQ_OK;
}

extern "C" int cq_pages_compact(const cq_kv_pages* pages, const cq_page_map* m, int32_t* d_remap, int32_t* d_status,
                                void* workspace, void* stream) {
  CQ_TRY(pool_and_map_check(pages, m));
  if (!d_remap || !d_status || !workspace || unaligned16(workspace)) return fail(CQ_EINVAL, "pages_compact: bad arguments");
  const hipStream_t st = as_stream(stream);
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, *m, d_remap, d_status, (int*)workspace);
  CQ_HIP(hipGetLastError());
  const int table_blocks = std::min(m->n_seqs, 128);
  const int most = copy_blocks((int64_t)(m->n_pages / 2 + 1) * pages->n_layers * 2 * pages->n_kv_heads);
  hipLaunchKernelGGL(compact_apply_kernel, dim3(table_blocks + most), dim3(kCopyThreads), 0, st, page_view(*pages),
                     copy_geo(*pages), *m, d_remap, table_blocks, (const int*)workspace);
  CQ_HIP(hipGetLastError());
  return CQ_OK;
}

extern "C" int cq_pages_copy(const cq_kv_pages* src, const cq_kv_pages* dst, const int32_t* d_src, const int32_t* d_dst,
                             int32_t n, int32_t* d_status, void* stream) {
  CQ_TRY(pages_check(src));
  CQ_TRY(pages_check(dst));
  if (src->kv_dtype != dst->kv_dtype || src->n_layers != dst->n_layers || src->page_tokens != dst->page_tokens ||
      src->n_kv_heads != dst->n_kv_heads || src->head_dim != dst->head_dim)
    return fail(CQ_EINVAL, "pages_copy: the pools differ in type or shape");
  if (n < 0 || n > 4096) return fail(CQ_EINVAL, "pages_copy: n outside [0, 4096]");
  if (n == 0) return CQ_OK;
  if (!d_src || !d_dst || !d_status) return fail(CQ_EINVAL, "pages_copy: null pointer");
  const CopyGeo g = copy_geo(*src);
  hipLaunchKernelGGL(copy_pages_kernel, dim3(copy_blocks((int64_t)n * g.n_layers * 2 * g.n_kv)), dim3(kCopyThreads), 0,
                     as_stream(stream), page_view(*src), page_view(*dst), g, d_src, d_dst, n, src->k == dst->k, d_status);
  CQ_HIP(hipGetLastError());
  return CQ_OK;
}
