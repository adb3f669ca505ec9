// The page pool of a paged key / value cache (include/paged_cache.h) for gfx950: sharing, cutting, growing with
// copy on write, freeing and compaction decided on the device, so that a decode loop never waits for the host.
//
// Everything that decides is integer work whose result does not depend on the order it runs in: reference
// counts by integer atomics, ranks by prefix sums over fixed blocks.  The header's rules are a chain of dependences
// over the whole pool: small pools (up to 8,192 pages) are decided by every workgroup for itself in its LDS, in one
// launch with the copies (update_small); for larger ones each link is a launch:
//   update_start   counts' = refs, marks cleared
//   update_refs    the pages that a row had and does not keep, or keeps and had not, subtracted / added
//                  (beams mostly continue rows that share their pages: nothing to do); growing rows marked
//   update_count   free pages counted a block; the rows' requests numbered
//   update_commit  the new table (a row finds its own free pages: block by the counts, then by rank), the new
//                  reference counts, and the copies of the used tokens in every plane
// and for the compaction compact_small, or compact_count, compact_rank and compact_commit.
//
// Measured on one MI355X: a beam step of 112 rows (28 groups of 4, 300 pages, six layers, 1.6 MB copied) 9.8 us in
// update_small, against 18 us in four launches; 256 rows of up to 16,000 tokens in a pool of 158,000 pages 18 us
// in four (2.7 + 3.5 + 3.4 + 8.5), bound by their dependence on each other; the same with one workgroup per
// pool would read its 640 KB of counts alone, twice.  The compaction of 8,192 pages of 128 KB, of which
// 1,966 move: 10 us of ranks and 61 us of copies, 5.0 TB/s read and written — the rate of a large copy.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged_cache.h"
#include "paged_error.h"

namespace {

constexpr int kT = 256;          // threads a workgroup
constexpr int kBlock = 1024;     // pages whose free (live) count is one block sum
constexpr int kCopyWgs = 2048;   // workgroups that share the copies (8 a CU)
constexpr int kSmallT = 1024;    // update_small: threads, and rows at most
// compact_small saves two launches (4,000 pages of 24 KB: 20 -> 15 us), but its copies begin late and reach less of
// the memory's rate (8,192 pages of 128 KB: 71 -> 78 us)
constexpr int64_t kSmallBytes = 256ll << 20;
// update_small's counts take 12 bytes of LDS a page, and each of its workgroups reads the whole table
constexpr int kSmallPages = 8192, kSmallEntries = 16384, kSmallWgs = 256;

struct Row {
  int keep, total, kept, page;  // tokens kept, new length, pages kept, partial last page of a growing row (or -1)
};

struct Upd {
  const int *table, *lens, *refs, *parents, *new_lens;
  int n, width, pages, ps, sh, blocks;
  int *table_out, *lens_out, *refs_out, *short_out;
  int *held, *growing, *highest, *counts, *first, *cow;  // workspace (first: n + 1, the last the total)
  unsigned char* data;
  int planes, heads, rb;
};

__device__ __forceinline__ int pages_of(int tokens, int sh) { return (int)(((unsigned)tokens + (1u << sh) - 1u) >> sh); }

__device__ __forceinline__ int clamp_len(const Upd& a, int v) { return max(0, min(v, a.width * a.ps)); }

__device__ __forceinline__ int parent_of(const Upd& a, int s) {
  const int p = a.parents ? a.parents[s] : s;
  return (unsigned)p < (unsigned)a.n ? p : -1;
}

// what row s keeps of its parent and grows to
__device__ __forceinline__ Row row_of(const Upd& a, int s, int p) {
  Row r;
  const int base = p >= 0 ? clamp_len(a, a.lens[p]) : 0;
  r.total = a.new_lens ? clamp_len(a, a.new_lens[s]) : base;
  r.keep = min(base, r.total);
  r.kept = pages_of(r.keep, a.sh);
  r.page = -1;
  if (r.total > r.keep && (r.keep & (a.ps - 1))) {
    const int x = a.table[(long long)p * a.width + r.kept - 1];
    if ((unsigned)x < (unsigned)a.pages) r.page = x;
  }
  return r;
}

// how many of page x's growing rows take a copy (its references: held)
__device__ __forceinline__ int copies_of(int held, int growing) {
  return held > 1 ? (growing == held ? growing - 1 : growing) : 0;
}
__device__ __forceinline__ bool takes_copy(int held, int growing, int highest, int s) {
  return held > 1 && !(growing == held && highest == s);
}

__device__ __forceinline__ void copy16(unsigned char* dst, const unsigned char* src) {
  *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
}

// the used tokens of page src to page dst in planes pl0 .. pl0 + planes - 1
__device__ __forceinline__ void copy_used(const Upd& a, int pl0, int planes, int src, int dst, int keep, int tid,
                                          int threads) {
  const long long head_bytes = (long long)a.ps * a.rb, page = head_bytes * a.heads;
  const int used = (keep & (a.ps - 1)) * a.rb / 16;  // 16-byte chunks a head
  for (long long i = tid; i < (long long)planes * a.heads * used; i += threads) {
    const long long hd = i / used;
    const int pl = pl0 + (int)(hd / a.heads);
    unsigned char* base = a.data + pl * (page * a.pages);
    const long long off = hd % a.heads * head_bytes + i % used * 16;
    copy16(base + dst * page + off, base + src * page + off);
  }
}

// sum over the workgroup
template <int THREADS>
__device__ __forceinline__ int block_sum(int v) {
  __shared__ int part[THREADS / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) t += part[i];
  return t;
}

// exclusive prefix over the workgroup's threads; total: the sum
template <int THREADS, class I>
__device__ __forceinline__ I block_scan(I v, I& total) {
  __shared__ I part[THREADS / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  I inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const I u = __shfl_up(inc, o);
    if (lane >= o) inc += u;
  }
  __syncthreads();
  if (lane == 63) part[w] = inc;
  __syncthreads();
  I before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) {
    if (i < w) before += part[i];
    total += part[i];
  }
  return before + inc - v;
}

// sums that may pass 2^31 (requests of all rows) are kept there: only "more than the pool" matters
__device__ __forceinline__ int clamp_sum(long long v) { return (int)min(v, (long long)INT32_MAX); }

// the state as it was
__device__ __forceinline__ void keep_state(const Upd& a, int wg, int wgs, int threads) {
  const long long tid = (long long)wg * threads + threadIdx.x, all = (long long)wgs * threads;
  for (long long e = tid; e < (long long)a.n * a.width; e += all) a.table_out[e] = a.table[e];
  for (long long e = tid; e < a.pages; e += all) a.refs_out[e] = a.refs[e];
  for (long long e = tid; e < a.n; e += all) a.lens_out[e] = a.lens[e];
}

// n <= kSmallT, pages <= kSmallPages, n * width <= kSmallEntries.  Every workgroup decides all, writes its share of
// the outputs and does its share of the copies
__global__ __launch_bounds__(kSmallT) void update_small(Upd a) {
  extern __shared__ int lds[];
  int *held = lds, *growing = held + a.pages, *highest = growing + a.pages;  // highest: later the pages asked for
  __shared__ int s_keep[kSmallT], s_total[kSmallT], s_parent[kSmallT], s_first[kSmallT], s_cow[kSmallT];
  const int tid = threadIdx.x, wg = blockIdx.x, wgs = gridDim.x;
  for (int x = tid; x < a.pages; x += kSmallT) {
    held[x] = a.refs[x];
    growing[x] = 0;
    highest[x] = -1;
  }
  Row r{0, 0, 0, -1};
  int p = -1, old_len = 0;
  if (tid < a.n) {
    p = parent_of(a, tid);
    r = row_of(a, tid, p);
    old_len = clamp_len(a, a.lens[tid]);
    s_keep[tid] = r.keep;
    s_total[tid] = r.total;
    s_parent[tid] = p;
    s_first[tid] = old_len;  // (until the requests are numbered)
  }
  __syncthreads();
  for (int e = tid; e < a.n * a.width; e += kSmallT) {
    const int s = e / a.width, c = e - s * a.width;
    const int q = s_parent[s];
    const int had = c < pages_of(s_first[s], a.sh) ? a.table[e] : -1;
    const int has = c < pages_of(s_keep[s], a.sh) ? a.table[q * a.width + c] : -1;
    if (had == has) continue;
    if ((unsigned)had < (unsigned)a.pages) atomicSub(held + had, 1);
    if ((unsigned)has < (unsigned)a.pages) atomicAdd(held + has, 1);
  }
  if (r.page >= 0) {
    atomicAdd(growing + r.page, 1);
    atomicMax(highest + r.page, tid);
  }
  __syncthreads();
  int cow = 0, need = 0;
  if (tid < a.n) {
    cow = r.page >= 0 && takes_copy(held[r.page], growing[r.page], highest[r.page], tid);
    need = pages_of(r.total, a.sh) - r.kept + cow;
  }
  // (need <= kSmallEntries + 1 over kSmallT rows: the sum fits)
  int asked;
  const int first = block_scan<kSmallT>(need, asked);
  // the free pages: each thread ranks a run of them
  const int run = (a.pages + kSmallT - 1) / kSmallT, x0 = min(a.pages, tid * run), x1 = min(a.pages, x0 + run);
  int mine = 0;
  for (int x = x0; x < x1; ++x) mine += held[x] == 0;
  int free;
  int rank = block_scan<kSmallT>(mine, free);  // (its barriers: every row has read `highest`)
  const bool ok = asked <= free;
  if (wg == 0 && tid == 0) a.short_out[0] = ok ? 0 : asked - free;
  if (!ok) {
    keep_state(a, wg, wgs, kSmallT);
    return;
  }
  int* pool = highest;
  for (int x = x0; x < x1; ++x) {
    if (held[x] != 0) continue;
    if (rank < asked) {
      pool[rank] = x;
      growing[x] = -1;  // (asked for; no row grows in a free page)
    }
    ++rank;
  }
  if (tid < a.n) {
    s_first[tid] = first;
    s_cow[tid] = cow ? r.page : -1;
    if (wg == 0) a.lens_out[tid] = r.total;
  }
  __syncthreads();
  for (int x = wg * kSmallT + tid; x < a.pages; x += wgs * kSmallT)
    a.refs_out[x] = growing[x] < 0 ? 1 : held[x] - copies_of(held[x], growing[x]);
  for (int e = wg * kSmallT + tid; e < a.n * a.width; e += wgs * kSmallT) {
    const int s = e / a.width, c = e - s * a.width;
    const int kept = pages_of(s_keep[s], a.sh), own = s_cow[s] >= 0;
    int x = -1;
    if (own && c == kept - 1) {
      x = pool[s_first[s]];
    } else if (c < kept) {
      x = a.table[s_parent[s] * a.width + c];
      if ((unsigned)x >= (unsigned)a.pages) x = -1;
    } else if (c < pages_of(s_total[s], a.sh)) {
      x = pool[s_first[s] + own + c - kept];
    }
    a.table_out[e] = x;
  }
  if (!a.data) return;
  // a quarter of the workgroup takes a row's copy in one plane
  const int part = tid >> 8, lane = tid & 255;
  for (int e = wg * 4 + part; e < a.n * a.planes; e += wgs * 4) {
    const int s = e / a.planes, pl = e - s * a.planes;
    if (s_cow[s] >= 0) copy_used(a, pl, 1, s_cow[s], pool[s_first[s]], s_keep[s], lane, 256);
  }
}

__global__ __launch_bounds__(kT) void update_start(Upd a) {
  const int x = blockIdx.x * kT + threadIdx.x;
  if (x >= a.pages) return;
  a.held[x] = a.refs[x];
  a.growing[x] = 0;
  a.highest[x] = -1;
}

// grid: x over the columns of the table, y over rows
__global__ __launch_bounds__(kT) void update_refs(Upd a) {
  const int c = blockIdx.x * kT + threadIdx.x;
  for (int s = blockIdx.y; s < a.n; s += gridDim.y) {
    const int p = parent_of(a, s);
    const Row r = row_of(a, s, p);
    const int len = pages_of(clamp_len(a, a.lens[s]), a.sh);
    if (c == 0 && r.page >= 0) {
      atomicAdd(a.growing + r.page, 1);
      atomicMax(a.highest + r.page, s);
    }
    const int had = c < len ? a.table[(long long)s * a.width + c] : -1;
    const int has = c < r.kept ? a.table[(long long)p * a.width + c] : -1;
    if (had == has) continue;
    if ((unsigned)had < (unsigned)a.pages) atomicSub(a.held + had, 1);
    if ((unsigned)has < (unsigned)a.pages) atomicAdd(a.held + has, 1);
  }
}

// workgroups 0 .. blocks-1 count the free pages of their block, the last one numbers the rows' requests
__global__ __launch_bounds__(kT) void update_count(Upd a) {
  if ((int)blockIdx.x < a.blocks) {
    int v = 0;
    for (int i = threadIdx.x; i < kBlock; i += kT) {
      const int x = blockIdx.x * kBlock + i;
      if (x < a.pages && a.held[x] == 0) ++v;
    }
    v = block_sum<kT>(v);
    if (threadIdx.x == 0) a.counts[blockIdx.x] = v;
    return;
  }
  long long asked = 0;
  for (int s0 = 0; s0 < a.n; s0 += kT) {
    const int s = s0 + threadIdx.x;
    int need = 0, cow = 0;
    if (s < a.n) {
      const Row r = row_of(a, s, parent_of(a, s));
      cow = r.page >= 0 && takes_copy(a.held[r.page], a.growing[r.page], a.highest[r.page], s);
      need = pages_of(r.total, a.sh) - r.kept + cow;
      a.cow[s] = cow;
    }
    long long total;
    const long long k = block_scan<kT>((long long)need, total);
    if (s < a.n) a.first[s] = clamp_sum(asked + k);
    asked += total;
  }
  if (threadIdx.x == 0) a.first[a.n] = clamp_sum(asked);
}

// workgroups 0 .. blocks-1: the reference counts of their pages; the others: rows, then shares of the copies
__global__ __launch_bounds__(kT) void update_commit(Upd a) {
  __shared__ int s_block, s_before;
  const int tid = threadIdx.x;
  int v = 0, below = 0;
  for (int i = tid; i < a.blocks; i += kT) {
    v += a.counts[i];
    if (i < (int)blockIdx.x) below += a.counts[i];
  }
  const int free = block_sum<kT>(v);
  const int asked = a.first[a.n];
  const bool ok = asked <= free;
  if (blockIdx.x == 0 && tid == 0) a.short_out[0] = ok ? 0 : asked - free;
  if (!ok) {
    keep_state(a, blockIdx.x, gridDim.x, kT);
    return;
  }
  if ((int)blockIdx.x < a.blocks) {
    int before = block_sum<kT>(below);  // free pages of the blocks before
    for (int i = 0; i < kBlock; i += kT) {
      const int x = blockIdx.x * kBlock + i + tid;
      const int held = x < a.pages ? a.held[x] : 1;
      int total;
      const int k = before + block_scan<kT>((int)(held == 0), total);
      before += total;
      if (x >= a.pages) continue;
      a.refs_out[x] = held == 0 ? (k < asked ? 1 : 0) : held - copies_of(held, a.growing[x]);
    }
    return;
  }
  const int wg = blockIdx.x - a.blocks, wgs = gridDim.x - a.blocks;
  for (int s = wg; s < a.n; s += wgs) {
    const int p = parent_of(a, s);
    const Row r = row_of(a, s, p);
    const int cow = a.cow[s], first = a.first[s], need = a.first[s + 1] - first;
    const int total = pages_of(r.total, a.sh);
    int* out = a.table_out + (long long)s * a.width;
    if (tid == 0) a.lens_out[s] = r.total;
    for (int c = tid; c < a.width; c += kT) {
      if (c < r.kept - cow) {
        const int x = a.table[(long long)p * a.width + c];
        out[c] = (unsigned)x < (unsigned)a.pages ? x : -1;
      } else if (c >= total) {
        out[c] = -1;
      }
    }
    if (need == 0) continue;
    // the row's free pages, first .. first + need - 1 in rank, to the columns from kept - cow on: the block that
    // holds the first by the blocks' counts, then block by block
    int before = 0;
    for (int b0 = 0; b0 < a.blocks; b0 += kT) {
      const int here = b0 + tid < a.blocks ? a.counts[b0 + tid] : 0;
      int sum;
      const int k = before + block_scan<kT>(here, sum);
      if (k <= first && first < k + here) s_block = b0 + tid, s_before = k;  // (one thread: first < free)
      if (first < before + sum) break;
      before += sum;
    }
    __syncthreads();
    before = s_before;
    for (int b = s_block; b < a.blocks && before < first + need; ++b) {
      for (int i = 0; i < kBlock; i += kT) {
        const int x = b * kBlock + i + tid;
        const bool f = x < a.pages && a.held[x] == 0;
        int sum;
        const int k = before + block_scan<kT>((int)f, sum) - first;
        before += sum;
        if (f && k >= 0 && k < need) out[r.kept - cow + k] = x;
      }
    }
    if (!cow || !a.data) continue;
    __syncthreads();  // (the row's own writes)
    const int dst = out[r.kept - 1];
    copy_used(a, 0, a.planes, r.page, dst, r.keep, tid, kT);
  }
}

struct Cmp {
  const int *table, *refs;
  long long entries;
  int pages, blocks, planes;
  long long page_bytes;
  unsigned char* data;
  int *table_out, *refs_out, *remap_out, *live_out;
  int *counts, *rank, *src, *dst, *moved;  // workspace
};

// sum of counts[0 .. n)
__device__ __forceinline__ int sum_counts(const int* counts, int n) {
  int v = 0;
  for (int i = threadIdx.x; i < n; i += kT) v += counts[i];
  return block_sum<kT>(v);
}

__global__ __launch_bounds__(kT) void compact_count(Cmp a) {
  int v = 0;
  for (int i = threadIdx.x; i < kBlock; i += kT) {
    const int x = blockIdx.x * kBlock + i;
    if (x < a.pages && a.refs[x] > 0) ++v;
  }
  v = block_sum<kT>(v);
  if (threadIdx.x == 0) a.counts[blockIdx.x] = v;
}

__global__ __launch_bounds__(kT) void compact_rank(Cmp a) {
  const int live = sum_counts(a.counts, a.blocks);
  // live pages below `live`: whole blocks, then the rest of the block it ends in
  const int lb = live / kBlock;
  int v = 0;
  for (int i = threadIdx.x; i < live - lb * kBlock; i += kT) v += a.refs[lb * kBlock + i] > 0;
  const int below = sum_counts(a.counts, lb) + block_sum<kT>(v);
  int before = sum_counts(a.counts, blockIdx.x);
  for (int i = 0; i < kBlock; i += kT) {
    const int x = blockIdx.x * kBlock + i + threadIdx.x;
    const bool on = x < a.pages && a.refs[x] > 0;
    int total;
    const int k = before + block_scan<kT>((int)on, total);  // live pages before x
    before += total;
    if (x >= a.pages) continue;
    if (on && x >= live) {
      a.src[k - below] = x;
      a.rank[x] = k - below;
    } else if (!on && x < live) {
      a.dst[x - k] = x;
      a.rank[x] = x - k;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.live_out[0] = live;
    a.moved[0] = live - below;
  }
}

__device__ __forceinline__ void copy_page(unsigned char* base, long long page_bytes, int src, int dst, int tid,
                                          int threads) {
  const unsigned char* f = base + src * page_bytes;
  unsigned char* t = base + dst * page_bytes;
  for (long long i = tid * 16; i < page_bytes; i += threads * 16) copy16(t + i, f + i);
}

// pages <= kSmallPages: every workgroup ranks all pages in its LDS, writes its share of the outputs and does its
// share of the copies
__global__ __launch_bounds__(kSmallT) void compact_small(Cmp a) {
  extern __shared__ short lds16[];  // (16 bits: two workgroups a CU, which the copies need)
  short *to = lds16, *src = to + a.pages, *dst = src + a.pages;  // to[x]: where page x goes (-1: free)
  const int tid = threadIdx.x, wg = blockIdx.x, wgs = gridDim.x;
  const int run = (a.pages + kSmallT - 1) / kSmallT, x0 = min(a.pages, tid * run), x1 = min(a.pages, x0 + run);
  uint32_t on = 0;  // bit i: page x0 + i lives (run <= 8)
  for (int x = x0; x < x1; ++x) on |= (uint32_t)(a.refs[x] > 0) << (x - x0);
  int live;
  int before = block_scan<kSmallT>((int)__popc(on), live);
  int v = 0;
  for (int x = x0; x < x1; ++x) v += ((on >> (x - x0)) & 1u) && x < live;
  const int below = block_sum<kSmallT>(v), moved = live - below;
  for (int x = x0; x < x1; ++x) {
    const bool o = (on >> (x - x0)) & 1u;
    if (o && x >= live) src[before - below] = (short)x;
    if (!o && x < live) dst[x - before] = (short)x;
    to[x] = (short)(o ? (x < live ? x : -2 - (before - below)) : -1);
    before += o;
  }
  __syncthreads();
  if (wg == 0 && tid == 0) a.live_out[0] = live;
  for (int x = wg * kSmallT + tid; x < a.pages; x += wgs * kSmallT) {
    const int t = to[x];
    a.remap_out[x] = t < -1 ? dst[-2 - t] : t;
    if (x >= live)
      a.refs_out[x] = 0;
    else if (t >= 0)
      a.refs_out[x] = a.refs[x];
  }
  for (int k = wg * kSmallT + tid; k < moved; k += wgs * kSmallT) a.refs_out[dst[k]] = a.refs[src[k]];
  for (long long e = (long long)wg * kSmallT + tid; e < a.entries; e += (long long)wgs * kSmallT) {
    const int x = a.table[e];
    const int t = (unsigned)x < (unsigned)a.pages ? to[x] : -1;
    a.table_out[e] = t < -1 ? dst[-2 - t] : t;
  }
  if (!a.data) return;
  const long long plane = a.page_bytes * a.pages;
  const int part = tid >> 8, lane = tid & 255;  // a quarter of the workgroup takes a page of one plane
  for (long long e = (long long)wg * 4 + part; e < (long long)moved * a.planes; e += (long long)wgs * 4) {
    const int k = (int)(e / a.planes), pl = (int)(e % a.planes);
    copy_page(a.data + pl * plane, a.page_bytes, src[k], dst[k], lane, 256);
  }
}

__global__ __launch_bounds__(kT) void compact_commit(Cmp a) {
  const int live = a.live_out[0], moved = a.moved[0];
  const long long tid = (long long)blockIdx.x * kT + threadIdx.x, all = (long long)gridDim.x * kT;
  for (long long x = tid; x < a.pages; x += all) {
    const bool on = a.refs[x] > 0;
    a.remap_out[x] = !on ? -1 : x < live ? (int)x : a.dst[a.rank[x]];
    a.refs_out[x] = x >= live ? 0 : on ? a.refs[x] : a.refs[a.src[a.rank[x]]];
  }
  for (long long e = tid; e < a.entries; e += all) {
    int x = a.table[e];
    if ((unsigned)x >= (unsigned)a.pages || a.refs[x] <= 0)
      x = -1;
    else if (x >= live)
      x = a.dst[a.rank[x]];
    a.table_out[e] = x;
  }
  if (!a.data) return;
  const long long plane = a.page_bytes * a.pages;
  for (long long e = blockIdx.x; e < (long long)moved * a.planes; e += gridDim.x) {
    const int k = (int)(e / a.planes), pl = (int)(e % a.planes);
    copy_page(a.data + pl * plane, a.page_bytes, a.src[k], a.dst[k], threadIdx.x, kT);
  }
}

__global__ __launch_bounds__(kT) void pages_copy(const int* src, const int* dst, long long count, unsigned char* data,
                                                 int planes, int pages, long long page_bytes) {
  const long long plane = page_bytes * pages;
  for (long long e = blockIdx.x; e < count * planes; e += gridDim.x) {
    const int f = src[e / planes], t = dst[e / planes];
    if ((unsigned)f >= (unsigned)pages || (unsigned)t >= (unsigned)pages) continue;
    copy_page(data + (e % planes) * plane, page_bytes, f, t, threadIdx.x, kT);
  }
}

int64_t pad16(int64_t ints) { return (ints * 4 + 15) / 16 * 16; }

bool launched(const char* who) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return mfl_paged_error("%s: launch failed: %s", who, hipGetErrorString(e));
  return true;
}

bool pool_ok(const char* who, int64_t pages, int64_t planes, int64_t page_bytes, const void* data) {
  if (pages < 0 || pages > (1ll << 30)) return mfl_paged_error("%s: %lld pages", who, (long long)pages);
  if (data && (planes < 1 || planes > (1 << 20) || page_bytes < 16 || page_bytes % 16 || page_bytes > (1ll << 30)))
    return mfl_paged_error("%s: planes %lld, page of %lld bytes (a multiple of 16)", who, (long long)planes,
                           (long long)page_bytes);
  if (reinterpret_cast<uintptr_t>(data) & 15u) return mfl_paged_error("%s: data is not 16-byte aligned", who);
  return true;
}

}  // namespace

extern "C" {

int64_t mfl_pages_update_workspace_bytes(int64_t n, int64_t pages) {
  if (n < 0 || pages < 0) return -1;
  return 3 * pad16(pages) + pad16((pages + kBlock - 1) / kBlock) + pad16(n + 1) + pad16(n);
}

int mfl_pages_update(const int32_t* table, const int32_t* lens, const int32_t* refs, const int32_t* parents,
                     const int32_t* new_lens, int64_t n, int64_t width, int64_t pages, int64_t page_size, void* data,
                     int64_t planes, int64_t heads, int64_t row_bytes, int32_t* table_out, int32_t* lens_out,
                     int32_t* refs_out, int32_t* short_out, void* workspace, void* stream) {
  const char* who = "mfl_pages_update";
  mfl_paged_error("%s", "");
  if (n < 0 || n > (1 << 20) || width < 0) {
    mfl_paged_error("%s: n %lld (at most 2^20), width %lld", who, (long long)n, (long long)width);
    return 1;
  }
  if (page_size < 1 || page_size > 1024 || (page_size & (page_size - 1)) || width * page_size > (1ll << 30)) {
    mfl_paged_error("%s: page_size %lld is no power of two up to 1024, or a row of more than 2^30 tokens", who,
                    (long long)page_size);
    return 1;
  }
  if (data && (heads < 1 || heads > 4096 || row_bytes < 16 || row_bytes % 16 || row_bytes > 65536)) {
    mfl_paged_error("%s: heads %lld, rows of %lld bytes (a multiple of 16)", who, (long long)heads,
                    (long long)row_bytes);
    return 1;
  }
  if (!pool_ok(who, pages, planes, heads * page_size * row_bytes, data)) return 1;
  if (!short_out || !workspace || (n > 0 && (!lens || !lens_out)) || (n * width > 0 && (!table || !table_out)) ||
      (pages > 0 && (!refs || !refs_out))) {
    mfl_paged_error("%s: NULL pointer", who);
    return 1;
  }
  Upd a{};
  a.table = table, a.lens = lens, a.refs = refs, a.parents = parents, a.new_lens = new_lens;
  a.n = (int)n, a.width = (int)width, a.pages = (int)pages, a.ps = (int)page_size;
  a.sh = __builtin_ctzll((unsigned long long)page_size);
  a.blocks = (int)((pages + kBlock - 1) / kBlock);
  a.table_out = table_out, a.lens_out = lens_out, a.refs_out = refs_out, a.short_out = short_out;
  char* ws = static_cast<char*>(workspace);
  a.held = reinterpret_cast<int*>(ws), ws += pad16(pages);
  a.growing = reinterpret_cast<int*>(ws), ws += pad16(pages);
  a.highest = reinterpret_cast<int*>(ws), ws += pad16(pages);
  a.counts = reinterpret_cast<int*>(ws), ws += pad16(a.blocks);
  a.first = reinterpret_cast<int*>(ws), ws += pad16(n + 1);
  a.cow = reinterpret_cast<int*>(ws);
  a.data = static_cast<unsigned char*>(data);
  a.planes = (int)planes, a.heads = (int)heads, a.rb = (int)row_bytes;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (n <= kSmallT && pages <= kSmallPages && n * width <= kSmallEntries) {
    // enough workgroups for the copies (4 a workgroup at a time)
    const int64_t want = data ? (n * planes + 3) / 4 : 1;
    const unsigned wgs = (unsigned)(want < 1 ? 1 : want > kSmallWgs ? kSmallWgs : want);
    hipLaunchKernelGGL(update_small, dim3(wgs), dim3(kSmallT), (size_t)(pages > 0 ? pages : 1) * 12, st, a);
    return launched(who) ? 0 : 1;
  }
  const unsigned cols = (unsigned)((width + kT - 1) / kT > 0 ? (width + kT - 1) / kT : 1);
  const unsigned rows = (unsigned)(n < 1 ? 1 : n > 32768 ? 32768 : n);
  if (pages > 0) hipLaunchKernelGGL(update_start, dim3((unsigned)((pages + kT - 1) / kT)), dim3(kT), 0, st, a);
  if (n > 0) hipLaunchKernelGGL(update_refs, dim3(cols, rows), dim3(kT), 0, st, a);
  hipLaunchKernelGGL(update_count, dim3((unsigned)a.blocks + 1), dim3(kT), 0, st, a);
  hipLaunchKernelGGL(update_commit, dim3((unsigned)a.blocks + rows), dim3(kT), 0, st, a);
  return launched(who) ? 0 : 1;
}

int64_t mfl_pages_compact_workspace_bytes(int64_t pages) {
  if (pages < 0) return -1;
  return 3 * pad16(pages) + pad16((pages + kBlock - 1) / kBlock) + 16;
}

int mfl_pages_compact(const int32_t* table, int64_t entries, const int32_t* refs, int64_t pages, void* data,
                      int64_t planes, int64_t page_bytes, int32_t* table_out, int32_t* refs_out, int32_t* remap_out,
                      int32_t* live_out, void* workspace, void* stream) {
  const char* who = "mfl_pages_compact";
  mfl_paged_error("%s", "");
  if (!pool_ok(who, pages, planes, page_bytes, data)) return 1;
  if (entries < 0 || entries > (1ll << 40)) {
    mfl_paged_error("%s: %lld table entries", who, (long long)entries);
    return 1;
  }
  if (!live_out || !workspace || (entries > 0 && (!table || !table_out)) ||
      (pages > 0 && (!refs || !refs_out || !remap_out))) {
    mfl_paged_error("%s: NULL pointer", who);
    return 1;
  }
  Cmp a{};
  a.table = table, a.refs = refs, a.entries = entries, a.pages = (int)pages;
  a.blocks = (int)((pages + kBlock - 1) / kBlock);
  a.planes = (int)planes, a.page_bytes = page_bytes;
  a.data = static_cast<unsigned char*>(data);
  a.table_out = table_out, a.refs_out = refs_out, a.remap_out = remap_out, a.live_out = live_out;
  char* ws = static_cast<char*>(workspace);
  a.rank = reinterpret_cast<int*>(ws), ws += pad16(pages);
  a.src = reinterpret_cast<int*>(ws), ws += pad16(pages);
  a.dst = reinterpret_cast<int*>(ws), ws += pad16(pages);
  a.counts = reinterpret_cast<int*>(ws), ws += pad16(a.blocks);
  a.moved = reinterpret_cast<int*>(ws);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (pages <= kSmallPages && (!data || pages * planes * page_bytes <= kSmallBytes)) {
    const unsigned wgs = data ? 2 * kSmallWgs : 8;  // (how many pages move is known on the device alone)
    hipLaunchKernelGGL(compact_small, dim3(wgs), dim3(kSmallT), (size_t)(pages > 0 ? pages : 1) * 6, st, a);
    return launched(who) ? 0 : 1;
  }
  if (a.blocks > 0) hipLaunchKernelGGL(compact_count, dim3((unsigned)a.blocks), dim3(kT), 0, st, a);
  hipLaunchKernelGGL(compact_rank, dim3((unsigned)(a.blocks > 0 ? a.blocks : 1)), dim3(kT), 0, st, a);
  hipLaunchKernelGGL(compact_commit, dim3(kCopyWgs), dim3(kT), 0, st, a);
  return launched(who) ? 0 : 1;
}

int mfl_pages_copy(const int32_t* src, const int32_t* dst, int64_t count, void* data, int64_t planes, int64_t pages,
                   int64_t page_bytes, void* stream) {
  const char* who = "mfl_pages_copy";
  mfl_paged_error("%s", "");
  if (count < 0 || count > (1ll << 30)) {
    mfl_paged_error("%s: count %lld", who, (long long)count);
    return 1;
  }
  if (!pool_ok(who, pages, planes, page_bytes, data)) return 1;
  if (count == 0 || pages == 0) return 0;
  if (!src || !dst || !data) {
    mfl_paged_error("%s: NULL pointer", who);
    return 1;
  }
  const long long items = count * planes;
  hipLaunchKernelGGL(pages_copy, dim3((unsigned)(items < kCopyWgs ? items : kCopyWgs)), dim3(kT), 0,
                     static_cast<hipStream_t>(stream), src, dst, (long long)count, static_cast<unsigned char*>(data),
                     (int)planes, (int)pages, (long long)page_bytes);
  return launched(who) ? 0 : 1;
}

}  // extern "C"
