// The page pool of a paged key / value cache (include/paged_cache.h) for gfx950: sharing, cutting, growing with
// copy on write, freeing and compaction decided on the device, so that a decode loop never waits for the host.
//
// Everything that decides is integer work whose result does not depend on the order it runs in: reference
// counts by integer atomics, ranks by prefix sums over fixed blocks.  The order of the rules in the header is a
// chain of dependences over the whole pool, so each link is a launch:
//   update_start   refs' = refs, marks cleared             update_refs    rows' pages subtracted / added
//   update_marks   growing rows marked on shared pages;    update_rank    free pages listed in ascending order;
//                  free pages counted a block                             the rows' requests numbered
//   update_commit  the new table and counts; the copies of the used tokens in every plane
// and for the compaction: compact_count, compact_rank, compact_commit.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged_cache.h"
#include "paged_error.h"

namespace {

constexpr int kT = 256;          // threads a workgroup
constexpr int kBlock = 1024;     // pages whose free (live) count is one block sum
constexpr int kCopyWgs = 2048;   // workgroups that share the copies (8 a CU)

struct Row {
  int keep, total, kept, page;  // tokens kept, new length, pages kept, shared partial last page (-1: none)
};

struct Upd {
  const int *table, *lens, *refs, *parents, *new_lens;
  int n, width, pages, ps, sh, blocks;
  int *table_out, *lens_out, *refs_out, *short_out;
  int *growing, *highest, *counts, *pool, *first, *cow;  // workspace (first: n + 1, the last the total)
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

__global__ __launch_bounds__(kT) void update_start(Upd a) {
  const int x = blockIdx.x * kT + threadIdx.x;
  if (x >= a.pages) return;
  a.refs_out[x] = a.refs[x];
  a.growing[x] = 0;
  a.highest[x] = -1;
}

// grid: x over the columns of the table, y over rows
__global__ __launch_bounds__(kT) void update_refs(Upd a) {
  const int c = blockIdx.x * kT + threadIdx.x;
  for (int s = blockIdx.y; s < a.n; s += gridDim.y) {
    const int p = parent_of(a, s);
    const Row r = row_of(a, s, p);
    const int held = pages_of(clamp_len(a, a.lens[s]), a.sh);
    const int same = p == s ? min(held, r.kept) : 0;  // pages the row had and keeps
    if (c < held && c >= same) {
      const int x = a.table[(long long)s * a.width + c];
      if ((unsigned)x < (unsigned)a.pages) atomicSub(a.refs_out + x, 1);
    }
    if (c < r.kept && c >= same) {
      const int x = a.table[(long long)p * a.width + c];
      if ((unsigned)x < (unsigned)a.pages) atomicAdd(a.refs_out + x, 1);
    }
  }
}

__device__ __forceinline__ int block_sum(int v) {
  __shared__ int part[kT / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int i = 0; i < kT / 64; ++i) t += part[i];
  __syncthreads();
  return t;
}

// exclusive prefix over the workgroup's threads; total: the sum
__device__ __forceinline__ int block_scan(int v, int& total) {
  __shared__ int part[kT / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 63) part[w] = inc;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kT / 64; ++i) {
    if (i < w) before += part[i];
    total += part[i];
  }
  __syncthreads();
  return before + inc - v;
}

// workgroups 0 .. blocks-1 count the free pages of their block, the others mark rows
__global__ __launch_bounds__(kT) void update_marks(Upd a) {
  if ((int)blockIdx.x < a.blocks) {
    int v = 0;
    for (int i = threadIdx.x; i < kBlock; i += kT) {
      const int x = blockIdx.x * kBlock + i;
      if (x < a.pages && a.refs_out[x] == 0) ++v;
    }
    v = block_sum(v);
    if (threadIdx.x == 0) a.counts[blockIdx.x] = v;
    return;
  }
  const int s = ((int)blockIdx.x - a.blocks) * kT + threadIdx.x;
  if (s >= a.n) return;
  const Row r = row_of(a, s, parent_of(a, s));
  if (r.page >= 0 && a.refs_out[r.page] > 1) {
    atomicAdd(a.growing + r.page, 1);
    atomicMax(a.highest + r.page, s);
  }
}

// sum of counts[0 .. n)
__device__ __forceinline__ int sum_counts(const int* counts, int n) {
  int v = 0;
  for (int i = threadIdx.x; i < n; i += kT) v += counts[i];
  return block_sum(v);
}

// workgroup `blocks` numbers the rows' requests, the others list their block's free pages
__global__ __launch_bounds__(kT) void update_rank(Upd a) {
  if ((int)blockIdx.x < a.blocks) {
    int before = sum_counts(a.counts, blockIdx.x);
    for (int i = 0; i < kBlock; i += kT) {
      const int x = blockIdx.x * kBlock + i + threadIdx.x;
      const bool free = x < a.pages && a.refs_out[x] == 0;
      int total;
      const int k = block_scan(free, total);
      if (free) a.pool[before + k] = x;
      before += total;
    }
    return;
  }
  long long asked = 0;  // (n * width < 2^31 is not given: more than `pages` is all that matters)
  for (int s0 = 0; s0 < a.n; s0 += kT) {
    const int s = s0 + threadIdx.x;
    int need = 0, cow = 0;
    if (s < a.n) {
      const Row r = row_of(a, s, parent_of(a, s));
      if (r.page >= 0) {
        const int refs = a.refs_out[r.page];
        cow = refs > 1 && !(a.growing[r.page] == refs && a.highest[r.page] == s);
      }
      need = pages_of(r.total, a.sh) - r.kept + cow;
      a.cow[s] = cow;
    }
    int total;
    const int k = block_scan(need, total);
    if (s < a.n) a.first[s] = (int)min(asked + k, (long long)INT32_MAX);
    asked += total;
  }
  if (threadIdx.x == 0) a.first[a.n] = (int)min(asked, (long long)INT32_MAX);
}

__device__ __forceinline__ void copy16(unsigned char* dst, const unsigned char* src) {
  *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
}

// grid: x = column blocks, y = rows: the table; then every workgroup takes its share of the copies
__global__ __launch_bounds__(kT) void update_commit(Upd a) {
  const int free = sum_counts(a.counts, a.blocks);
  const int asked = a.first[a.n];
  const bool ok = asked <= free;
  const int wg = blockIdx.y * gridDim.x + blockIdx.x, wgs = gridDim.x * gridDim.y;
  if (wg == 0 && threadIdx.x == 0) a.short_out[0] = ok ? 0 : asked - free;
  if (!ok) {
    // the state as it was
    for (long long e = (long long)wg * kT + threadIdx.x; e < (long long)a.n * a.width; e += (long long)wgs * kT)
      a.table_out[e] = a.table[e];
    for (int e = wg * kT + threadIdx.x; e < a.pages; e += wgs * kT) a.refs_out[e] = a.refs[e];
    for (int e = wg * kT + threadIdx.x; e < a.n; e += wgs * kT) a.lens_out[e] = a.lens[e];
    return;
  }
  const int c = blockIdx.x * kT + threadIdx.x;
  for (int s = blockIdx.y; s < a.n; s += gridDim.y) {
    const int p = parent_of(a, s);
    const Row r = row_of(a, s, p);
    const int cow = a.cow[s], first = a.first[s];
    if (c == 0) {
      a.lens_out[s] = r.total;
      if (cow) atomicSub(a.refs_out + r.page, 1);
    }
    if (c >= a.width) continue;
    int x = -1;
    if (c < r.kept) {
      x = a.table[(long long)p * a.width + c];
      if ((unsigned)x >= (unsigned)a.pages) x = -1;
      if (cow && c == r.kept - 1) x = -2;
    } else if (c < pages_of(r.total, a.sh)) {
      x = -3;
    }
    if (x < -1) {
      x = a.pool[first + (x == -2 ? 0 : cow + c - r.kept)];
      a.refs_out[x] = 1;  // (asked for once, held by nothing else)
    }
    a.table_out[(long long)s * a.width + c] = x;
  }
  if (!a.data) return;
  const long long head_bytes = (long long)a.ps * a.rb, plane = head_bytes * a.heads * a.pages;
  for (long long e = wg; e < (long long)a.n * a.planes; e += wgs) {
    const int s = (int)(e / a.planes), pl = (int)(e % a.planes);
    if (!a.cow[s]) continue;
    const Row r = row_of(a, s, parent_of(a, s));
    const int dst = a.pool[a.first[s]];
    const int used = (r.keep & (a.ps - 1)) * a.rb / 16;  // 16-byte chunks a head
    unsigned char* base = a.data + pl * plane;
    for (int i = threadIdx.x; i < a.heads * used; i += kT) {
      const long long off = (long long)(i / used) * head_bytes + (long long)(i % used) * 16;
      copy16(base + dst * head_bytes * a.heads + off, base + r.page * head_bytes * a.heads + off);
    }
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

__global__ __launch_bounds__(kT) void compact_count(Cmp a) {
  int v = 0;
  for (int i = threadIdx.x; i < kBlock; i += kT) {
    const int x = blockIdx.x * kBlock + i;
    if (x < a.pages && a.refs[x] > 0) ++v;
  }
  v = block_sum(v);
  if (threadIdx.x == 0) a.counts[blockIdx.x] = v;
}

__global__ __launch_bounds__(kT) void compact_rank(Cmp a) {
  const int live = sum_counts(a.counts, a.blocks);
  // live pages below `live`: whole blocks, then the rest of the block it ends in
  const int lb = live / kBlock;
  int v = 0;
  for (int i = threadIdx.x; i < live - lb * kBlock; i += kT) v += a.refs[lb * kBlock + i] > 0;
  const int below = sum_counts(a.counts, lb) + block_sum(v);
  int before = sum_counts(a.counts, blockIdx.x);
  for (int i = 0; i < kBlock; i += kT) {
    const int x = blockIdx.x * kBlock + i + threadIdx.x;
    const bool on = x < a.pages && a.refs[x] > 0;
    int total;
    const int k = before + block_scan(on, total);  // live pages before x
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

__device__ __forceinline__ void copy_page(unsigned char* base, long long page_bytes, int src, int dst) {
  const unsigned char* f = base + src * page_bytes;
  unsigned char* t = base + dst * page_bytes;
  for (long long i = threadIdx.x * 16; i < page_bytes; i += kT * 16) copy16(t + i, f + i);
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
    copy_page(a.data + pl * plane, a.page_bytes, a.src[k], a.dst[k]);
  }
}

__global__ __launch_bounds__(kT) void pages_copy(const int* src, const int* dst, long long count, unsigned char* data,
                                                 int planes, int pages, long long page_bytes) {
  const long long plane = page_bytes * pages;
  for (long long e = blockIdx.x; e < count * planes; e += gridDim.x) {
    const int f = src[e / planes], t = dst[e / planes];
    if ((unsigned)f >= (unsigned)pages || (unsigned)t >= (unsigned)pages) continue;
    copy_page(data + (e % planes) * plane, page_bytes, f, t);
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
  a.growing = reinterpret_cast<int*>(ws), ws += pad16(pages);
  a.highest = reinterpret_cast<int*>(ws), ws += pad16(pages);
  a.pool = reinterpret_cast<int*>(ws), ws += pad16(pages);
  a.counts = reinterpret_cast<int*>(ws), ws += pad16(a.blocks);
  a.first = reinterpret_cast<int*>(ws), ws += pad16(n + 1);
  a.cow = reinterpret_cast<int*>(ws);
  a.data = static_cast<unsigned char*>(data);
  a.planes = (int)planes, a.heads = (int)heads, a.rb = (int)row_bytes;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned cols = (unsigned)((width + kT - 1) / kT > 0 ? (width + kT - 1) / kT : 1);
  const unsigned rows = (unsigned)(n < 1 ? 1 : n > 32768 ? 32768 : n);
  if (pages > 0) hipLaunchKernelGGL(update_start, dim3((unsigned)((pages + kT - 1) / kT)), dim3(kT), 0, st, a);
  if (n > 0) hipLaunchKernelGGL(update_refs, dim3(cols, rows), dim3(kT), 0, st, a);
  if (a.blocks + n > 0)
    hipLaunchKernelGGL(update_marks, dim3((unsigned)(a.blocks + (n + kT - 1) / kT)), dim3(kT), 0, st, a);
  hipLaunchKernelGGL(update_rank, dim3((unsigned)a.blocks + 1), dim3(kT), 0, st, a);
  // enough workgroups for the copies as well
  unsigned gy = rows;
  if (data && cols * gy < (unsigned)kCopyWgs) gy = (kCopyWgs + cols - 1) / cols;
  hipLaunchKernelGGL(update_commit, dim3(cols, gy), dim3(kT), 0, st, a);
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
