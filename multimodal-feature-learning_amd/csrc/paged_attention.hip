// Attention of a chunk of new tokens over a paged key / value cache (include/paged_cache.h) for gfx950.
//
// The `G = heads / kv_heads` query heads of one key head and the chunk's rows are one list of rows
// m = i * G + g of a (sequence, key head): all of them read the same keys, so they share tiles.  A wave
// holds 32 such rows as the COLUMNS of 32 x 32 MFMA tiles: S^T = K Q^T (keys down, rows across), so a
// row's scores sit in one lane and its partner lane + 32, the running maximum and sum are two registers
// (one exchange a tile), the rescale of O^T is a per-lane factor, and the score registers, rounded to the
// values' type, are the B operand of O^T += V^T P^T with no movement.  One pass over the keys:
//   m' = max(m, max_j s_j),  l' = l 2^(c (m - m')) + sum_j 2^(c (s_j - m')),  O' = O 2^(c (m - m')) + P V
// with c = scale * log2(e); m, l and O stay in fp32 and are rounded once at the end.  P is rounded to the
// values' 16-bit type, the only one that the matrix product takes beside them: at most 2^-8 (bf16) or 2^-11 (fp16)
// of each weight, as much as the output's own rounding.  l sums the unrounded weights.  fp16 has no such relative
// bound below its smallest normal number, 2^-14, and nothing below 2^-25: its weights are computed 2^7 times
// as large (kShift), so that the steps of its subnormal numbers are at most 2^-32 of the largest weight off.  At the weights'
// true size, 2^17 keys of 2^-25.2 beside one of 1 lose all they add, 7 times the output's rounding.
//
// The reference value m follows the maximum only when that has grown by more than 2^8 (any m gives the same
// quotient): most steps then need no rescale of O and no exchange between lanes.
//
//   paged_att_split  few rows a (sequence, key head): a wave takes 32 rows and a range of the keys through its own
//                    ring of tiles in LDS; where the keys make two ranges, two waves of a workgroup take one each and meet in LDS
//   paged_att_rows   more rows: 4 waves of 32 rows share double-buffered tiles of 64 keys
//   paged_att_join   key ranges of either: (m, l, O) of a row out of the workspace
//
// Keys and values go to LDS by global_load_lds (16 bytes a lane): no registers are held while the loads fly,
// so a wave keeps 16 to 32 KB in flight, and the rows of up to four loads that lie in one page have one
// scalar address.  Two classes of calls have less: fp32 wider than 64, whose tile of 32 KB is the whole ring (its loads
// fly between the steps, not beside them), and pages of fewer than 16 tokens (8 in fp32 wider than 64) or widths
// other than 32, 64 and 128, whose loads have an address a lane (load_tile).
//
// Measured on one MI355X (a 1 GB copy moves 5.0 TB/s, an 8192^3 product runs at 1.19 PFLOP/s in bf16, 154 TFLOP/s
// in fp32), us a call:
//   24 single tokens over 1 .. 16,384 keys, 32 / 8 heads of 128, bf16: 178, 5.1 TB/s — the memory's rate.  fp32 467
//   (3.9 TB/s); bf16 in pages of 8 tokens 209, at width 96 204 (3.4 TB/s of what it needs), fp32 at width 96 629
//   one single token over 131,071 keys, 16 / 2 heads of 128, fp16: 35 (3.9 TB/s); the kernels take 26 + 5
//   2 x 4,096 rows over 6,001 / 12,288 keys, 32 / 8 heads of 128, bf16: 965, 0.99 PFLOP/s.  A wave's step of 64
//   keys takes the matrix unit 1,024 cycles and the vector unit some 1,000 (214 instructions, 32 of them matrix products
//   and 32 exponentials at a quarter of the rate); with two waves a SIMD they overlap in part.  Not the loads' bandwidth
//   (the same tile loaded again and again takes as long; 96 % come from the L2), but issuing them was 9 % until runs
//   shared an address.  Priorities for the matrix products, 8 waves a tile, rings of 3 and 4, steps of 32 and 128 keys,
//   and a pipeline over steps (Q K of the next and P V of the last beside this one's exponentials) measured
//   the same or slower: what they gain in overlap they lose in registers, and with them in waves.
//
// MFMA 32x32x16 (16-bit): A lane (h, r): row r = lane & 31, k 8h..8h+7 (h = lane >> 5); B the same with
// columns; D register e: row 8 (e >> 2) + 4 h + (e & 3), column lane & 31.  The reduction of the second
// product runs over keys, and any order of them serves when both operands use it: B's slots are the lane's
// own score registers 8s .. 8s+7, so A's lane reads the keys 16 s + 4 h + {0..3, 8..11} of its value
// column, transposed out of LDS by ds_read_b64_tr_b16.  fp32: 32x32x2 steps in the same layout.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "paged_cache.h"
#include "paged_error.h"

namespace {

constexpr int kRowsW = 32;    // rows a wave holds
constexpr int kKeys = 32;     // keys of one score tile
constexpr float kLog2e = 1.4426950408889634f;

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

struct Args {
  const unsigned char *q, *kn, *vn;
  unsigned char *kp, *vp, *out;
  float* ws;
  const int *table, *kv_lens, *starts, *offsets;
  int n, rows, heads, kvh, G, D, pages, ps, sh, width, causal, splits, tiles, zero_tail;
  int range;              // keys a split takes at least
  long long total, slots; // packed rows; rows of the whole call (of a partial in the workspace)
  long long q_seq, q_row, q_head, k_seq, k_row, k_head, v_seq, v_row, v_head;  // bytes
  float c;  // scale * log2(e)
};

// 16 zero bytes a chunk: the source of key rows that are not there (their weight is zero, but 0 times
// whatever lies in an unwritten page row may be NaN)
__device__ const uint4 g_zero[32] = {};

template <class T>
struct Elem;
template <>
struct Elem<__bf16> {
  typedef bf16x8 frag;
  static __device__ __forceinline__ f32x16 mfma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Elem<_Float16> {
  typedef f16x8 frag;
  static __device__ __forceinline__ f32x16 mfma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// LDS image of key rows: DP elements a row in 16-byte chunks, no padding, chunk c of row r stored at
// c ^ k_swz(r) (keys: 16 lanes read one chunk column of 16 rows) or c ^ v_swz(r) (values: the transposed
// read takes 4 chunks of 4 neighbouring rows) so that either read touches every bank once
template <class T, int DP>
struct Geo {
  static constexpr int EB = sizeof(T);
  static constexpr int RB = DP * EB;   // bytes a row
  static constexpr int NC = RB / 16;   // chunks a row
  static constexpr int QF = EB == 2 ? DP / 16 : DP / 8;  // query fragments of 16 bytes
  static constexpr int OB = DP / 32;   // 32-column blocks of the output
  static __device__ __forceinline__ int k_swz(int r) { return (NC >= 16 ? r : r / (16 / NC)) & (NC - 1); }
  static __device__ __forceinline__ int v_swz(int r) {
    if (EB == 4) return 0;
    return NC == 16 ? 4 * (r & 3) : NC == 8 ? 4 * ((r >> 1) & 1) : 0;
  }
};

struct Seq {
  int st, kv, rows;      // first position, visible length, rows of this call
  long long q0, q1;      // packed: first row and the one behind the last; else 0 (the strides are in the pointers)
};

__device__ __forceinline__ Seq seq_of(const Args& a, int s) {
  Seq q;
  q.kv = max(0, min(a.kv_lens[s], a.width * a.ps));  // (width * page_size < 2^31: checked on the host)
  q.q0 = q.q1 = 0;
  q.rows = a.rows;
  int len = a.rows;
  if (a.offsets) {
    const long long o0 = max(0ll, min((long long)a.offsets[s], a.total));
    const long long o1 = max(o0, min((long long)a.offsets[s + 1], a.total));
    q.q0 = o0;
    q.q1 = o1;
    len = (int)(o1 - o0);
    q.rows = min(len, a.rows);
  }
  const long long st = a.starts ? (long long)a.starts[s] : (long long)a.kv_lens[s] - len;
  // a start beyond +-2^30 sees everything or nothing: clamped so that positions stay in 32 bits
  q.st = (int)max(-(1ll << 30), min(st, (1ll << 30)));
  return q;
}

// the key / value row j of the chunk or of the cache; false: not there
struct RowSrc {
  const unsigned char *k, *v;
};
__device__ __forceinline__ bool row_src(const Args& a, const Seq& q, const unsigned char* kn, const unsigned char* vn,
                                        int kh, int j, int page, int rb, RowSrc& r) {
  r.k = r.v = reinterpret_cast<const unsigned char*>(g_zero);
  if (j >= q.kv) return false;
  if ((unsigned)page >= (unsigned)a.pages) return false;
  if (a.kn && (unsigned)(j - q.st) < (unsigned)q.rows) {
    r.k = kn + (long long)(j - q.st) * a.k_row;
    r.v = vn + (long long)(j - q.st) * a.v_row;
    return true;
  }
  const long long off = (((long long)page * a.kvh + kh) * a.ps + (j & (a.ps - 1))) * rb;
  r.k = a.kp + off;
  r.v = a.vp + off;
  return true;
}

// (m0, which holds the LDS address, is a reserved register to the compiler and warned about in clobber lists; nothing
// else in this file uses it)
#pragma clang diagnostic ignored "-Winline-asm"

// 16 bytes a lane from global memory to LDS at byte `dst` + 16 * lane (dst: wave-uniform, below 64 KB).
// The loads count in vmcnt; nothing but wait_loads() waits for them
__device__ __forceinline__ void load_lds(const unsigned char* src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(dst)
               : "memory", "m0");
}
// N of them, load i from base + off[i] + 1024 i to dst + 1024 i (the offset in the instruction counts on both sides)
template <int N>
__device__ __forceinline__ void load_lds_run(const unsigned char* base, const uint32_t (&off)[N], uint32_t dst) {
  static_assert(N == 1 || N == 2 || N == 4, "");
  if constexpr (N == 4)
    asm volatile(
        "s_mov_b32 m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %4\n\t"
        "global_load_lds_dwordx4 %1, %4 offset:%6\n\tglobal_load_lds_dwordx4 %2, %4 offset:%7\n\t"
        "global_load_lds_dwordx4 %3, %4 offset:%8" ::"v"(off[0]),
        "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base), "s"(dst), "i"(1024), "i"(2 * 1024), "i"(3 * 1024)
        : "memory", "m0");
  else if constexpr (N == 2)
    asm volatile(
        "s_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %2\n\t"
        "global_load_lds_dwordx4 %1, %2 offset:1024" ::"v"(off[0]),
        "v"(off[1]), "s"(base), "s"(dst)
        : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off[0]), "s"(base), "s"(dst)
                 : "memory", "m0");
}
// all but the last N vector memory operations of the wave are done
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "vmcnt has six bits");
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// a barrier that does not wait for loads to LDS, and that no LDS access crosses
__device__ __forceinline__ void wave_barrier() { asm volatile("s_barrier" ::: "memory"); }

__device__ __forceinline__ uint32_t lds_at(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// 64 entries of a sequence's table a time, one a lane, and the next 64 on their way
struct Pages {
  int base, cur, nxt;
  unsigned long long bad;  // entries of `cur` outside the pool

  __device__ __forceinline__ int entry(const Args& a, const int* tab, int i) const { return i < a.width ? tab[i] : -1; }
  __device__ __forceinline__ void start(const Args& a, const int* tab, int first, int lane) {
    base = first;
    cur = entry(a, tab, base + lane);
    nxt = entry(a, tab, base + 64 + lane);
    bad = __ballot((unsigned)cur >= (unsigned)a.pages);
  }
  // entries first .. last (uniform, ascending from call to call, fewer than 64 of them from a multiple) are in `cur`
  __device__ __forceinline__ void need(const Args& a, const int* tab, int first, int last, int lane) {
    if (last - base < 64) return;
    if (first - base == 64) {
      base += 64;
      cur = nxt;
      nxt = entry(a, tab, base + 64 + lane);
      bad = __ballot((unsigned)cur >= (unsigned)a.pages);
    } else {
      start(a, tab, first, lane);
    }
  }
  __device__ __forceinline__ bool any_bad(int first, int last) const {
    if (bad == 0ull) return false;
    const int w = last - first + 1;
    return ((bad >> (first - base)) & (w >= 64 ? ~0ull : (1ull << w) - 1ull)) != 0ull;
  }
};

// loads of 1 KB (64 lanes) for image rows r0 .. of keys j0 + r0 ..: IT of them for keys and values each, LDS images
// at kd and vd.  `safe`: keys below it come from the pages and are there.  Where up to 16 rows lie in one page
// (and a row has all DP columns) the run of their loads has one scalar address: what this loop issues
// beside the loads is a third of a step's instructions otherwise.  The other branch takes every tile that holds one of the
// chunk's own keys, and all tiles of smaller pages and other widths
template <class T, int DP, int IT>
__device__ __forceinline__ void load_tile(const Args& a, const Seq& q, const Pages& pg, const unsigned char* kn,
                                          const unsigned char* vn, int kh, int j0, int r0, int safe, uint32_t kd,
                                          uint32_t vd, int lane) {
  typedef Geo<T, DP> Ge;
  constexpr int RP = 64 / Ge::NC;  // rows a load
  constexpr int RN0 = RP >= 16 ? 1 : 16 / RP, RN1 = RN0 > 4 ? 4 : RN0, RN = RN1 > IT ? IT : RN1;  // loads a run
  static_assert(IT % RN == 0, "");
  const int lr = lane / Ge::NC, cp = lane % Ge::NC;
  const int jb = j0 + r0;
  const uint32_t d0 = r0 / RP * 1024;
  if (jb + IT * RP <= safe && a.ps >= RN * RP && a.D == DP && !pg.any_bad(jb >> a.sh, (jb + IT * RP - 1) >> a.sh)) {
    const uint32_t head = (uint32_t)a.ps * Ge::RB;  // bytes of one head's rows of a page
#pragma unroll
    for (int g = 0; g < IT / RN; ++g) {
      const int j = jb + g * RN * RP;
      const uint32_t page = __builtin_amdgcn_readlane(pg.cur, (j >> a.sh) - pg.base);
      const unsigned long long off = (unsigned long long)(page * (uint32_t)a.kvh + (uint32_t)kh) * head +
                                     (uint32_t)(j & (a.ps - 1)) * Ge::RB;
      uint32_t ok[RN], ov[RN];
#pragma unroll
      for (int t = 0; t < RN; ++t) {
        const int row = r0 + (g * RN + t) * RP + lr;
        ok[t] = lr * Ge::RB + ((cp ^ Ge::k_swz(row)) << 4);
        ov[t] = lr * Ge::RB + ((cp ^ Ge::v_swz(row)) << 4);
      }
      load_lds_run<RN>(a.kp + off, ok, kd + d0 + g * RN * 1024);
      load_lds_run<RN>(a.vp + off, ov, vd + d0 + g * RN * 1024);
    }
  } else {
    const int rb = a.D * Ge::EB, nch = rb / 16;
#pragma unroll 1
    for (int t = 0; t < IT; ++t) {
      const int row = r0 + t * RP + lr;
      const int j = j0 + row;
      const int page = __shfl(pg.cur, (j >> a.sh) - pg.base);
      RowSrc r;
      row_src(a, q, kn, vn, kh, j, page, rb, r);
      const int ck = cp ^ Ge::k_swz(row), cv = cp ^ Ge::v_swz(row);
      if (ck < nch) load_lds(r.k + ck * 16, kd + d0 + t * 1024);
      if (cv < nch) load_lds(r.v + cv * 16, vd + d0 + t * 1024);
    }
  }
}

// chunks behind a row's D elements: zero once, the loads leave them alone
__device__ __forceinline__ void clear_lds(unsigned char* lds, int bytes, int tid, int threads) {
  for (int i = tid * 16; i < bytes; i += threads * 16) *reinterpret_cast<uint4*>(lds + i) = uint4{0, 0, 0, 0};
}

// the rows of a wave, as MFMA columns
template <class T, int DP>
struct Cols {
  uint4 qf[Geo<T, DP>::QF];
  f32x16 o[Geo<T, DP>::OB];
  float m, l;  // reference value; sum of the weights (of the lane's own scores until cols_sum)
  int lim;  // keys this lane's row sees
};

template <class T, int DP>
__device__ __forceinline__ void cols_init(Cols<T, DP>& w, const Args& a, const Seq& q, const unsigned char* qb, int kh,
                                          int m0, int lane) {
  const int row = m0 + (lane & 31), h = lane >> 5;
  const int i = row / a.G, g = row - i * a.G;
  const bool ok = i < q.rows;
  // (a lane behind the last row takes the last row's limit: nothing reads what it computes, and the tiles
  // that every row sees need no masking)
  w.lim = m0 >= q.rows * a.G ? 0 : a.causal ? max(0, min(q.kv, q.st + min(i, q.rows - 1) + 1)) : q.kv;
  const unsigned char* src = qb + (long long)i * a.q_row + (long long)(kh * a.G + g) * a.q_head;
  const int nch = a.D * (int)sizeof(T) / 16;
#pragma unroll
  for (int t = 0; t < Geo<T, DP>::QF; ++t) {
    const int ch = 2 * t + h;
    w.qf[t] = ok && ch < nch ? *reinterpret_cast<const uint4*>(src + ch * 16) : uint4{0, 0, 0, 0};
  }
#pragma unroll
  for (int d = 0; d < Geo<T, DP>::OB; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) w.o[d][e] = 0.f;
  w.m = -INFINITY;
  w.l = 0.f;
}

// S^T of 32 keys (LDS image kt) against the wave's rows
template <class T, int DP>
__device__ __forceinline__ f32x16 scores(const Cols<T, DP>& w, const unsigned char* kt, int lane) {
  typedef Geo<T, DP> Ge;
  const int r = lane & 31, h = lane >> 5;
  const int swz = Ge::k_swz(r);
  f32x16 s;
#pragma unroll
  for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
  for (int t = 0; t < Ge::QF; ++t) {
    const uint4 kv = *reinterpret_cast<const uint4*>(kt + r * Ge::RB + ((2 * t + h) ^ swz) * 16);
    if constexpr (Ge::EB == 2) {
      typedef typename Elem<T>::frag frag;
      s = Elem<T>::mfma(__builtin_bit_cast(frag, kv), __builtin_bit_cast(frag, w.qf[t]), s);
    } else {
      const f32x4 x = __builtin_bit_cast(f32x4, kv), y = __builtin_bit_cast(f32x4, w.qf[t]);
#pragma unroll
      for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], s, 0, 0, 0);
    }
  }
  return s;
}

// 16-bit: the A operand of 16 keys (s) and 32 value columns (d) of the image vt
template <class T, int DP>
__device__ __forceinline__ typename Elem<T>::frag value_frag(const unsigned char* vt, int s, int d, int lane) {
  typedef Geo<T, DP> Ge;
  const int h = lane >> 5, li = lane & 15, half = (lane >> 4) & 1;
  const int r0 = 16 * s + 4 * h + (li >> 2), r1 = r0 + 8;
  const int ch = d * 4 + half * 2 + ((li & 3) >> 1), by = (li & 1) * 8;
  const s16x4 x0 =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vt + r0 * Ge::RB + (ch ^ Ge::v_swz(r0)) * 16 + by));
  const s16x4 x1 =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vt + r1 * Ge::RB + (ch ^ Ge::v_swz(r1)) * 16 + by));
  return __builtin_bit_cast(typename Elem<T>::frag, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
}

// fp32: the value of the lane's column at register e's key
template <int DP>
__device__ __forceinline__ float value_at(const unsigned char* vt, int e, int d, int lane) {
  const int r = 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
  return *reinterpret_cast<const float*>(vt + r * Geo<float, DP>::RB + (d * 32 + (lane & 31)) * 4);
}

// O^T += V^T P^T of 32 keys (LDS image vt), p the weights in score layout
template <class T, int DP>
__device__ __forceinline__ void weigh(Cols<T, DP>& w, const f32x16& p, const unsigned char* vt, int lane) {
  typedef Geo<T, DP> Ge;
  if constexpr (Ge::EB == 2) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      typename Elem<T>::frag b;
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = (T)p[8 * s + e];
#pragma unroll
      for (int d = 0; d < Ge::OB; ++d) w.o[d] = Elem<T>::mfma(value_frag<T, DP>(vt, s, d, lane), b, w.o[d]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e)
#pragma unroll
      for (int d = 0; d < Ge::OB; ++d)
        w.o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(value_at<DP>(vt, e, d, lane), p[e], w.o[d], 0, 0, 0);
  }
}

template <class T>
__device__ __forceinline__ bool non_finite(T x) {
  if constexpr (sizeof(T) == 4) {
    return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
  } else {
    constexpr uint16_t ex = __is_same(T, __bf16) ? 0x7f80 : 0x7c00;
    return (__builtin_bit_cast(uint16_t, x) & ex) == ex;
  }
}

// the 16 bytes with values that are not finite replaced by 0; true: there were some
template <class T>
__device__ __forceinline__ bool scrub(uint4& v) {
  constexpr int N = 16 / (int)sizeof(T);
  T x[N];
  __builtin_memcpy(x, &v, 16);
  bool any = false;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const bool nf = non_finite<T>(x[e]);
    any |= nf;
    if (nf) x[e] = (T)0.f;
  }
  __builtin_memcpy(&v, x, 16);
  return any;
}

// the same over an LDS image (its loads have been waited for); the wave's later reads see the result
template <class T>
__device__ __forceinline__ bool scrub_image(unsigned char* p, int bytes, int lane, int lanes) {
  bool any = false;
#pragma unroll 1
  for (int i = lane * 16; i < bytes; i += lanes * 16) {
    uint4 v = *reinterpret_cast<const uint4*>(p + i);
    if (scrub<T>(v)) {
      *reinterpret_cast<uint4*>(p + i) = v;
      any = true;
    }
  }
  wait_lds();
  return any;
}

// bit kk: key j0 + kk lies in a page of the pool (asked only where a tile has one that does not)
__device__ __forceinline__ uint32_t keys_there(const Args& a, const int* tab, int j0, int kv, int lane) {
  const int j = j0 + (lane & 31);
  const int page = j < kv ? tab[j >> a.sh] : -1;
  return (uint32_t)__ballot((unsigned)page < (unsigned)a.pages);
}

// scores of keys j0 .. j0+31 that the lane's row does not see become -inf; `there` bit kk: key j0+kk exists
__device__ __forceinline__ void mask_scores(f32x16& s, int j0, int lim, uint32_t there, int lane) {
  const int h = lane >> 5;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int kk = 8 * (e >> 2) + 4 * h + (e & 3);
    if (j0 + kk >= lim || !((there >> kk) & 1u)) s[e] = -INFINITY;
  }
}

// the online softmax's step for NT score tiles: s replaced by the weights against m; m, l and O rescaled when
// some row's maximum outgrows m by 2^kLazy.  w.l: the sum of the lane's own scores only
constexpr float kLazy = 8.f;
// the weights are 2^kShift times their size, in O and l alike and in every range, so that it drops out of the quotient.
// fp16: at most 2^(kLazy + kShift) = 2^15, which it holds
template <class T>
constexpr float kShift = __is_same(T, _Float16) ? 7.f : 0.f;
template <class T, int DP, int NT>
__device__ __forceinline__ void soft_step(Cols<T, DP>& w, f32x16 (&s)[NT], float c) {
  float mx = s[0][0];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[t][e]);
  if (__any((mx - w.m) * c > kLazy)) {  // (-inf - -inf: false, nothing seen yet)
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float mn = fmaxf(w.m, mx);
    const float al = __builtin_amdgcn_exp2f(w.m == mn ? 0.f : (w.m - mn) * c);
    w.m = mn;
    w.l *= al;
#pragma unroll
    for (int d = 0; d < Geo<T, DP>::OB; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) w.o[d][e] *= al;
  }
  const float base = w.m == -INFINITY ? 0.f : w.m * c - kShift<T>;  // (nothing seen yet: every weight is 2^-inf = 0)
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[t][e] = __builtin_amdgcn_exp2f(fmaf(s[t][e], c, -base));
      sum[e & 3] += s[t][e];
    }
  w.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

template <class T>
__device__ __forceinline__ void store4(unsigned char* dst, const float* v) {
  if constexpr (sizeof(T) == 2) {
    typedef __attribute__((ext_vector_type(4))) T t4;
    t4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (T)v[e];
    *reinterpret_cast<uint2*>(dst) = __builtin_bit_cast(uint2, x);
  } else {
    *reinterpret_cast<f32x4*>(dst) = f32x4{v[0], v[1], v[2], v[3]};
  }
}

// Keys that some rows of a tile see and others do not (the chunk's own, under the causal mask) must not reach the
// latter: the matrix product would make NaN of 0 times an infinite or NaN value.  Tiles with such keys are
// staged with these values scrubbed to 0, and where there were any they are added here, after the loop, to the
// rows that see them (a finite positive weight leaves them what they are).  Keys j0 .. j1 of the sequence
template <class T, int DP>
__device__ __forceinline__ void add_non_finite(Cols<T, DP>& w, const Args& a, const Seq& q, const unsigned char* kn,
                                               const unsigned char* vn, const int* tab, int kh, int j0, int j1,
                                               int lane) {
  const int h = lane >> 5;
#pragma unroll 1
  for (int j = j0; j < j1; ++j) {
    RowSrc r;
    if (!row_src(a, q, kn, vn, kh, j, tab[j >> a.sh], a.D * (int)sizeof(T), r)) continue;
    const bool see = j < w.lim;
#pragma unroll
    for (int d = 0; d < Geo<T, DP>::OB; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int col = d * 32 + 8 * b + 4 * h;
        if (col >= a.D || !see) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const T x = reinterpret_cast<const T*>(r.v)[col + e];
          if (non_finite<T>(x)) w.o[d][4 * b + e] += (float)x;
        }
      }
  }
}

// the wave's rows to `out`: a lane holds 4 neighbouring columns a register quad
template <class T, int DP>
__device__ __forceinline__ void cols_store(const Cols<T, DP>& w, const Args& a, const Seq& q, int s, int kh, int m0,
                                           int lane) {
  const int row = m0 + (lane & 31), h = lane >> 5;
  const int i = row / a.G, g = row - i * a.G;
  if (i >= q.rows) return;
  const float inv = w.l > 0.f ? 1.f / w.l : (w.l == 0.f ? 0.f : w.l);  // (NaN stays NaN)
  const long long r = (a.offsets ? q.q0 : (long long)s * a.rows) + i;
  unsigned char* dst = a.out + (r * a.heads + kh * a.G + g) * (long long)a.D * (long long)sizeof(T);
#pragma unroll
  for (int d = 0; d < Geo<T, DP>::OB; ++d)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int col = d * 32 + 8 * b + 4 * h;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = w.o[d][4 * b + e] * inv;
      if (col < a.D) store4<T>(dst + col * (int)sizeof(T), v);
    }
}

// the chunk's own keys and values of rows i0 .. i1 into the pages
template <class T>
__device__ __forceinline__ void write_chunk(const Args& a, const Seq& q, int s, const unsigned char* kn,
                                            const unsigned char* vn, int kh, int i0, int i1, int tid, int threads) {
  const int rb = a.D * (int)sizeof(T), nch = rb / 16;
  for (int e = i0 * nch + tid; e < i1 * nch; e += threads) {
    const int i = e / nch, ch = e - i * nch;
    const int p = q.st + i;
    if (p < 0 || p >= q.kv) continue;
    const int page = a.table[(long long)s * a.width + (p >> a.sh)];
    if ((unsigned)page >= (unsigned)a.pages) continue;
    const long long dst = (((long long)page * a.kvh + kh) * a.ps + (p & (a.ps - 1))) * rb + ch * 16;
    *reinterpret_cast<uint4*>(a.kp + dst) = *reinterpret_cast<const uint4*>(kn + (long long)i * a.k_row + ch * 16);
    *reinterpret_cast<uint4*>(a.vp + dst) = *reinterpret_cast<const uint4*>(vn + (long long)i * a.v_row + ch * 16);
  }
}

// packed rows first .. last - 1 of `out`
__device__ __forceinline__ void zero_rows(const Args& a, long long first, long long last, int part, int parts, int eb) {
  const long long per = (long long)a.heads * a.D * eb / 16;
  uint4* dst = reinterpret_cast<uint4*>(a.out);
  for (long long e = first * per + (long long)part * blockDim.x + threadIdx.x; e < last * per;
       e += (long long)parts * blockDim.x)
    dst[e] = uint4{0, 0, 0, 0};
}

template <class T, int DP>
__device__ __forceinline__ void cols_sum(Cols<T, DP>& w) {
  w.l += __shfl_xor(w.l, 32);
}

// What the ranges of a row leave in the workspace: `used` (slots * heads int32: how many ranges, 0 or 1: nothing to
// join), then per range (m, l) pairs and O rows of DP floats, slots * heads of each
struct Part {
  int* used;
  float *ml, *o;
};
__device__ __forceinline__ Part part_of(const Args& a, int split, int DP) {
  const long long sh = a.slots * a.heads;
  Part p;
  p.used = reinterpret_cast<int*>(a.ws);
  float* f = a.ws + (sh + 3) / 4 * 4;
  p.ml = f + split * sh * 2;
  p.o = f + (a.splits * sh * 2 + 3) / 4 * 4 + split * sh * DP;
  return p;
}

template <class T, int DP>
__device__ __forceinline__ void cols_part(const Cols<T, DP>& w, const Args& a, const Seq& q, int s, int kh, int m0,
                                          int split, int used, int lane) {
  const int row = m0 + (lane & 31), h = lane >> 5;
  const int i = row / a.G, g = row - i * a.G;
  if (i >= q.rows) return;
  const Part p = part_of(a, split, DP);
  const long long id = ((a.offsets ? q.q0 : (long long)s * a.rows) + i) * a.heads + kh * a.G + g;
  if (h == 0) {
    if (split == 0) p.used[id] = used;
    p.ml[id * 2] = w.m;
    p.ml[id * 2 + 1] = w.l;
  }
#pragma unroll
  for (int d = 0; d < Geo<T, DP>::OB; ++d)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int col = d * 32 + 8 * b + 4 * h;
      if (col < a.D)
        *reinterpret_cast<f32x4*>(p.o + id * DP + col) =
            f32x4{w.o[d][4 * b], w.o[d][4 * b + 1], w.o[d][4 * b + 2], w.o[d][4 * b + 3]};
    }
}

// a row written whole: nothing for the join to do
__device__ __forceinline__ void mark_whole(const Args& a, const Seq& q, int s, int kh, int m0, int lane) {
  const int row = m0 + (lane & 31);
  const int i = row / a.G, g = row - i * a.G;
  if (i >= q.rows || lane >= 32) return;
  reinterpret_cast<int*>(a.ws)[((a.offsets ? q.q0 : (long long)s * a.rows) + i) * a.heads + kh * a.G + g] = 1;
}

// packed rows first .. last - 1 are not this call's to write
__device__ __forceinline__ void mark_rows(const Args& a, long long first, long long last, int part, int parts) {
  for (long long e = first * a.heads + (long long)part * blockDim.x + threadIdx.x; e < last * a.heads;
       e += (long long)parts * blockDim.x)
    reinterpret_cast<int*>(a.ws)[e] = 0;
}

// what a workgroup has to do, the same in both kernels.  Work items are numbered (tile * splits + split) * kvh +
// kh: the workgroups that read one key head's pages are kvh apart and, with 8 XCDs taking workgroups in
// turn, share an L2 when kvh is a multiple of 8 (and a half or a quarter of them when it is 4 or 2).  Tiles: a.tiles
// of each sequence, or (packed) those that the sequences have, counted here, and one or more behind the last (s == n)
struct Job {
  int s, tile, split, kh;
  int part, parts;  // of the workgroups of sequence s (or behind the last)
};
template <int ROWS>
__device__ __forceinline__ Job job_of(const Args& a, int lane) {
  Job j;
  unsigned x = blockIdx.x;
  j.kh = x % (unsigned)a.kvh;
  x /= (unsigned)a.kvh;
  j.split = x % (unsigned)a.splits;
  const int e = x / (unsigned)a.splits;
  int mine = a.tiles, at;
  if (!a.offsets) {
    at = e % a.tiles;
    j.s = e / a.tiles;
  } else {
    int before = 0;
    j.s = a.n;
    for (int c = 0; c < a.n; c += 64) {
      const int i = min(a.n - 1, c + lane);
      const long long o0 = max(0ll, min((long long)a.offsets[i], a.total));
      const long long o1 = max(o0, min((long long)a.offsets[i + 1], a.total));
      const int t = c + lane < a.n ? (min((int)(o1 - o0), a.rows) * a.G + ROWS - 1) / ROWS : 0;
      int inc = t;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(inc, o);
        if (lane >= o) inc += u;
      }
      const unsigned long long hit = __ballot(before + inc > e);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        j.s = c + l;
        mine = __builtin_amdgcn_readlane(t, l);
        at = e - before - (__builtin_amdgcn_readlane(inc, l) - mine);
        break;
      }
      before += __builtin_amdgcn_readlane(inc, 63);
    }
    if (j.s == a.n) {
      at = e - before;
      mine = a.tiles - before;  // (a.tiles: one more than the sequences can have)
    }
  }
  j.tile = j.s < a.n ? mine - 1 - at : 0;  // (a sequence's last rows see the most keys: they begin first)
  j.part = (at * a.splits + j.split) * a.kvh + j.kh;
  j.parts = mine * a.splits * a.kvh;
  return j;
}

// packed calls (s == n): the rows before the first sequence and behind the last
__device__ __forceinline__ void rest_of_rows(const Args& a, const Job& j, int eb) {
  const long long r0 = max(0ll, min((long long)a.offsets[0], a.total));
  const long long r1 = max(r0, min((long long)a.offsets[a.n], a.total));
  if (a.zero_tail) {
    zero_rows(a, 0, r0, j.part, j.parts, eb);
    zero_rows(a, r1, a.total, j.part, j.parts, eb);
  }
  if (a.splits > 1) {
    mark_rows(a, 0, r0, j.part, j.parts);
    mark_rows(a, r1, a.total, j.part, j.parts);
  }
}
// ... and a sequence's rows behind its first a.rows
__device__ __forceinline__ void rows_behind(const Args& a, const Job& j, const Seq& q) {
  if (a.splits > 1 && a.offsets && q.q1 > q.q0 + q.rows) mark_rows(a, q.q0 + q.rows, q.q1, j.part, j.parts);
}

// keys first .. last - 1 (multiples of `step` but the last) of `most` that range `split` takes; used: ranges in all
struct Range {
  int first, last, used;
};
__device__ __forceinline__ Range range_of(const Args& a, int most, int split, int step) {
  const int steps = (most + step - 1) / step;
  const int per = max(a.range / step, (steps + a.splits - 1) / a.splits);
  Range r;
  r.used = max(1, (steps + per - 1) / per);
  r.first = min(most, split * per * step);
  r.last = min(most, r.first + per * step);
  return r;
}

// (two waves a SIMD: left to itself the compiler keeps O in accumulation registers, and one wave fits at DP = 128.  The
// two-wave form's 64 KB of tiles let two workgroups run on a CU, one wave a SIMD, and its registers, 185 + 80 at DP = 128,
// allow no more.  All instances keep 18 to 31 scalars in lanes of a vector register; nothing goes to memory)
template <class T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, NW == 1 ? 2 : 1) void paged_att_split(Args a) {
  typedef Geo<T, DP> Ge;
  constexpr int kImg = kKeys * Ge::RB;  // one 32-row image
  constexpr int kStage = 2 * kImg;      // keys and values
  constexpr int NS = kStage >= 32768 ? 1 : kStage >= 16384 ? 2 : 4;  // stages of a wave's ring (at most 32 KB)
  constexpr int kIt = kImg / 1024;      // loads of one image
  constexpr int kMerge = NW > 1 ? NW * 32 * (DP + 1) * 4 : 0;
  constexpr int kLds = NW * NS * kStage > kMerge ? NW * NS * kStage : kMerge;
  static_assert(NW * NS * kStage <= 65536, "load_lds reaches 64 KB");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[kLds];
  __shared__ float s_m[NW][32], s_l[NW][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const Job job = job_of<kRowsW>(a, lane);
  const int s = job.s, kh = job.kh, split = job.split;
  if (s >= a.n) {
    rest_of_rows(a, job, Ge::EB);
    return;
  }
  const Seq q = seq_of(a, s);
  rows_behind(a, job, q);
  const int m0 = job.tile * kRowsW;
  if (m0 >= q.rows * a.G) return;  // (uniform over the workgroup)
  const int ilast = min(q.rows - 1, (m0 + kRowsW - 1) / a.G);
  const int most = a.causal ? max(0, min(q.kv, q.st + ilast + 1)) : q.kv;  // keys the tile's last row sees
  const Range rg = range_of(a, most, split, kKeys);
  if (split >= rg.used) return;
  const long long seq = a.offsets ? 0 : s;
  const unsigned char* qb = a.q + seq * a.q_seq + q.q0 * a.q_row;
  const unsigned char* kn = a.kn ? a.kn + seq * a.k_seq + q.q0 * a.k_row + (long long)kh * a.k_head : nullptr;
  const unsigned char* vn = a.vn ? a.vn + seq * a.v_seq + q.q0 * a.v_row + (long long)kh * a.v_head : nullptr;
  const int* tab = a.table + (long long)s * a.width;
  const int b0 = rg.first / kKeys, b1 = (rg.last + kKeys - 1) / kKeys;
  const int wper = (b1 - b0 + NW - 1) / NW;
  const int w0 = b0 + wave * wper, w1 = min(b1, w0 + wper);
  unsigned char* ring = lds + wave * NS * kStage;
  const uint32_t ring_at = __builtin_amdgcn_readfirstlane(lds_at(ring));
  if (a.D != DP) {
    clear_lds(ring, NS * kStage, lane, 64);
    wait_lds();
  }
  const int safe = a.kn ? max(0, min(q.kv, q.st)) : q.kv;
  Pages pg;
  uint32_t gaps = 0;  // bit of a stage: a page of its keys is outside the pool
  if (w0 < w1) pg.start(a, tab, (w0 * kKeys) >> a.sh, lane);
  const auto issue = [&](int blk) {
    const int j0 = blk * kKeys;
    pg.need(a, tab, j0 >> a.sh, (j0 + kKeys - 1) >> a.sh, lane);
    const uint32_t slot = (uint32_t)(blk - w0) % NS, at = ring_at + slot * kStage;
    const bool gap = pg.any_bad(j0 >> a.sh, (min(q.kv, j0 + kKeys) - 1) >> a.sh);
    gaps = (gaps & ~(1u << slot)) | ((uint32_t)gap << slot);
    load_tile<T, DP, kIt>(a, q, pg, kn, vn, kh, j0, 0, safe, at, at + kImg, lane);
  };
#pragma unroll
  for (int t = 0; t < NS; ++t)
    if (w0 + t < w1) issue(w0 + t);
  if (a.kn && split == 0) {  // (while the first tiles fly)
    // the tile writes the tokens whose first row it holds
    const int i0 = (m0 + a.G - 1) / a.G, i1 = min(q.rows, (m0 + kRowsW + a.G - 1) / a.G);
    write_chunk<T>(a, q, s, kn, vn, kh, i0, i1, threadIdx.x, 64 * NW);
    wait_loads<0>();  // (the loop's counts are of loads only)
  }
  Cols<T, DP> w;
  cols_init<T, DP>(w, a, q, qb, kh, m0, lane);
  bool odd = false;  // a value that is not finite was scrubbed
  const int least = a.causal ? max(0, min(q.kv, q.st + m0 / a.G + 1)) : q.kv;  // keys the tile's first row sees
  for (int blk = w0; blk < w1; ++blk) {
    unsigned char* kt = ring + (uint32_t)(blk - w0) % NS * kStage;
    unsigned char* vt = kt + kImg;
    const int j0 = blk * kKeys;
    if (blk + NS <= w1)
      wait_loads<(NS - 1) * 2 * kIt>();
    else
      wait_loads<0>();
    if (least < min(q.kv, j0 + kKeys)) odd |= scrub_image<T>(vt, kImg, lane, 64);
    f32x16 sc[1];
    sc[0] = scores<T, DP>(w, kt, lane);
    const bool gap = (gaps >> ((uint32_t)(blk - w0) % NS)) & 1u;
    if (gap || !__all(j0 + kKeys <= w.lim))
      mask_scores(sc[0], j0, w.lim, gap ? keys_there(a, tab, j0, q.kv, lane) : ~0u, lane);
    soft_step<T, DP, 1>(w, sc, a.c);
    weigh<T, DP>(w, sc[0], vt, lane);
    wait_lds();  // (the images are read: the next loads may overwrite them)
    if (blk + NS < w1) issue(blk + NS);
  }
  if (__any(odd))
    add_non_finite<T, DP>(w, a, q, kn, vn, tab, kh, max(w0, least / kKeys) * kKeys, min(most, w1 * kKeys), lane);
  cols_sum<T, DP>(w);
  if constexpr (NW > 1) {
    __syncthreads();  // (every wave is done with its images)
    if (lane < 32) {
      s_m[wave][lane] = w.m;
      s_l[wave][lane] = w.l;
    }
    __syncthreads();
    const int col = lane & 31, h = lane >> 5;
    float mx = -INFINITY;
#pragma unroll
    for (int v = 0; v < NW; ++v) mx = fmaxf(mx, s_m[v][col]);
    const float base = mx == -INFINITY ? 0.f : mx * a.c;
    float l = 0.f;
#pragma unroll
    for (int v = 0; v < NW; ++v) l += s_l[v][col] * __builtin_amdgcn_exp2f(fmaf(s_m[v][col], a.c, -base));
    const float f = __builtin_amdgcn_exp2f(fmaf(w.m, a.c, -base));
    float* os = reinterpret_cast<float*>(lds);  // (wave, row, DP + 1)
#pragma unroll
    for (int d = 0; d < Ge::OB; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        os[(wave * 32 + col) * (DP + 1) + d * 32 + 8 * (e >> 2) + 4 * h + (e & 3)] = w.o[d][e] * f;
    __syncthreads();
    if (wave != 0) return;
    w.m = mx;
    w.l = l;
#pragma unroll
    for (int d = 0; d < Ge::OB; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float t = 0.f;
#pragma unroll
        for (int v = 0; v < NW; ++v) t += os[(v * 32 + col) * (DP + 1) + d * 32 + 8 * (e >> 2) + 4 * h + (e & 3)];
        w.o[d][e] = t;
      }
  }
  if (rg.used > 1) {
    cols_part<T, DP>(w, a, q, s, kh, m0, split, rg.used, lane);
  } else {
    cols_store<T, DP>(w, a, q, s, kh, m0, lane);
    if (a.splits > 1) mark_whole(a, q, s, kh, m0, lane);
  }
}

// out = sum_i 2^(c (m_i - m)) O_i / sum_i 2^(c (m_i - m)) l_i over a row's ranges.  DP / 4 lanes hold a row's
// columns; a workgroup takes 256 / (DP / 4) rows, or (WIDE: more than 16 ranges) 32 columns of one row, whose ranges its
// 32 groups of 8 lanes share (16 rows of 512 ranges: 59 -> 5 us, 768 rows of up to 43: 12 -> 6.  Fewer ranges leave its
// groups idle: 32 rows of 12 ranges would gain 0.5 us, 4,096 of 16 lose 8)
struct JoinSum {
  float m, l;
  f32x4 o;
};
__device__ __forceinline__ void join_add(JoinSum& w, float m, float l, const f32x4& o, float c) {
  const float mn = fmaxf(w.m, m), base = mn == -INFINITY ? 0.f : mn * c;
  const float f0 = __builtin_amdgcn_exp2f(fmaf(w.m, c, -base)), f1 = __builtin_amdgcn_exp2f(fmaf(m, c, -base));
  w.m = mn;
  w.l = w.l * f0 + l * f1;
#pragma unroll
  for (int k = 0; k < 4; ++k) w.o[k] = w.o[k] * f0 + o[k] * f1;
}

template <class T, int DP, bool WIDE>
__global__ __launch_bounds__(256) void paged_att_join(Args a) {
  constexpr int kQ = WIDE ? 8 : DP / 4, kGr = 256 / kQ, kParts = WIDE ? DP / 32 : 1, kWv = 4;
  __shared__ float s_m[kWv], s_l[kWv];
  __shared__ __attribute__((aligned(16))) f32x4 s_o[kWv][kQ];
  const int gr = threadIdx.x / kQ, x = threadIdx.x % kQ;
  const int col = (WIDE ? (int)(blockIdx.x % kParts) * 32 : 0) + x * 4;
  const long long sh = a.slots * a.heads;
  const long long id = WIDE ? (long long)(blockIdx.x / kParts) : (long long)blockIdx.x * kGr + gr;
  const Part p = part_of(a, 0, DP);
  const int used = id < sh ? min(p.used[id], a.splits) : 0;  // (offsets that do not ascend leave rows unmarked)
  if (WIDE && used <= 1) return;
  JoinSum w = {-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}};
  if (used > 1) {
    const int i0 = WIDE ? gr : 0;
    constexpr int kStep = WIDE ? kGr : 1;
#pragma unroll 4
    for (int i = i0; i < used; i += kStep) {
      const float mi = p.ml[(i * sh + id) * 2], li = p.ml[(i * sh + id) * 2 + 1];
      const f32x4 v = *reinterpret_cast<const f32x4*>(p.o + (i * sh + id) * DP + col);  // (behind D: not used)
      join_add(w, mi, li, v, a.c);
    }
  }
  if constexpr (WIDE) {
#pragma unroll
    for (int d = kQ; d < 64; d <<= 1) {
      const float m = __shfl_xor(w.m, d), l = __shfl_xor(w.l, d);
      f32x4 o;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = __shfl_xor(w.o[k], d);
      join_add(w, m, l, o, a.c);
    }
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) < kQ) {
      if (x == 0) {
        s_m[wave] = w.m;
        s_l[wave] = w.l;
      }
      s_o[wave][x] = w.o;
    }
    __syncthreads();
    if (gr != 0) return;
#pragma unroll 4
    for (int i = 1; i < kWv; ++i) join_add(w, s_m[i], s_l[i], s_o[i][x], a.c);
  }
  if (used <= 1 || col >= a.D) return;
  const float inv = w.l > 0.f ? 1.f / w.l : (w.l == 0.f ? 0.f : w.l);
  float v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = w.o[k] * inv;
  store4<T>(a.out + (id * (long long)a.D + col) * (long long)sizeof(T), v);
}

constexpr int kWavesR = 4;
constexpr int kTileR = kWavesR * kRowsW;  // rows a workgroup of paged_att_rows

template <class T, int DP>
__global__ __launch_bounds__(64 * kWavesR, 2) void paged_att_rows(Args a) {
  typedef Geo<T, DP> Ge;
  constexpr int NT = Ge::EB == 2 ? 2 : 1;  // score tiles a step (64 or 32 keys)
  constexpr int kStep = NT * kKeys;
  constexpr int kImg = kStep * Ge::RB;
  constexpr int NS = 2;  // steps in the ring (three or four measured the same: the loads are not what it waits for)
  constexpr int kIt = kImg / 1024 / kWavesR;  // loads of one image a wave
  constexpr int kRowsL = kStep / kWavesR;     // image rows a wave loads
  static_assert(kIt >= 1 && NS >= 2 && NS * 2 * kImg <= 65536, "load_lds reaches 64 KB");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[NS * 2 * kImg];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Job job = job_of<kTileR>(a, lane);
  const int s = job.s, kh = job.kh, split = job.split;
  if (s >= a.n) {
    rest_of_rows(a, job, Ge::EB);
    return;
  }
  const Seq q = seq_of(a, s);
  rows_behind(a, job, q);
  const int g0 = job.tile * kTileR;
  if (g0 >= q.rows * a.G) return;
  const int ilast = min(q.rows - 1, (g0 + kTileR - 1) / a.G);
  const int most = a.causal ? max(0, min(q.kv, q.st + ilast + 1)) : q.kv;
  const Range rg = range_of(a, most, split, kStep);
  if (split >= rg.used) return;
  const int m0 = g0 + wave * kRowsW;
  const long long seq = a.offsets ? 0 : s;
  const unsigned char* qb = a.q + seq * a.q_seq + q.q0 * a.q_row;
  const unsigned char* kn = a.kn ? a.kn + seq * a.k_seq + q.q0 * a.k_row + (long long)kh * a.k_head : nullptr;
  const unsigned char* vn = a.vn ? a.vn + seq * a.v_seq + q.q0 * a.v_row + (long long)kh * a.v_head : nullptr;
  const int* tab = a.table + (long long)s * a.width;
  const int t0 = rg.first / kStep, t1 = (rg.last + kStep - 1) / kStep;
  const uint32_t at = __builtin_amdgcn_readfirstlane(lds_at(lds));
  if (a.D != DP) {
    clear_lds(lds, NS * 2 * kImg, tid, 64 * kWavesR);
    __syncthreads();
  }
  const int safe = a.kn ? max(0, min(q.kv, q.st)) : q.kv;
  Pages pg;
  uint32_t gaps = 0;  // bit of a ring slot: a page of its keys is outside the pool
  pg.start(a, tab, (t0 * kStep) >> a.sh, lane);
  const auto issue = [&](int step) {
    const int j0 = step * kStep;
    pg.need(a, tab, j0 >> a.sh, (j0 + kStep - 1) >> a.sh, lane);
    const uint32_t slot = (uint32_t)(step - t0) % NS, d = at + slot * (2 * kImg);
    const bool gap = pg.any_bad(j0 >> a.sh, (min(q.kv, j0 + kStep) - 1) >> a.sh);
    gaps = (gaps & ~(1u << slot)) | ((uint32_t)gap << slot);
    load_tile<T, DP, kIt>(a, q, pg, kn, vn, kh, j0, wave * kRowsL, safe, d, d + kImg, lane);
  };
#pragma unroll
  for (int t = 0; t < NS - 1; ++t)
    if (t0 + t < t1) issue(t0 + t);
  if (a.kn && split == 0) {
    const int i0 = (g0 + a.G - 1) / a.G, i1 = min(q.rows, (g0 + kTileR + a.G - 1) / a.G);
    write_chunk<T>(a, q, s, kn, vn, kh, i0, i1, tid, 64 * kWavesR);
    wait_loads<0>();  // (the loop's counts are of loads only)
  }
  Cols<T, DP> w;
  cols_init<T, DP>(w, a, q, qb, kh, m0, lane);
  bool odd = false;  // a value that is not finite was scrubbed
  const int least = a.causal ? max(0, min(q.kv, q.st + g0 / a.G + 1)) : q.kv;  // keys the tile's first row sees
  for (int step = t0; step < t1; ++step) {
    const uint32_t slot = (uint32_t)(step - t0) % NS;
    unsigned char* kt = lds + slot * (2 * kImg);
    unsigned char* vt = kt + kImg;
    const int j0 = step * kStep;
    if (step + NS - 1 <= t1)
      wait_loads<(NS - 2) * 2 * kIt>();
    else
      wait_loads<0>();
    if (least < min(q.kv, j0 + kStep))
      odd |= scrub_image<T>(vt + wave * kRowsL * Ge::RB, kRowsL * Ge::RB, lane, 64);  // (what the wave has loaded)
    wait_lds();
    // every wave's part of the step has landed, and every wave has read the step before: its slot is free
    wave_barrier();
    const bool gap = (gaps >> slot) & 1u;
    if (step + NS - 1 < t1) issue(step + NS - 1);
    if (__all(j0 >= w.lim)) continue;
    f32x16 sc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) sc[t] = scores<T, DP>(w, kt + t * kKeys * Ge::RB, lane);
    if (gap || !__all(j0 + kStep <= w.lim)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
        mask_scores(sc[t], j0 + t * kKeys, w.lim, gap ? keys_there(a, tab, j0 + t * kKeys, q.kv, lane) : ~0u, lane);
    }
    soft_step<T, DP, NT>(w, sc, a.c);
#pragma unroll
    for (int t = 0; t < NT; ++t) weigh<T, DP>(w, sc[t], vt + t * kKeys * Ge::RB, lane);
  }
  if (least < most && __syncthreads_or(odd))
    add_non_finite<T, DP>(w, a, q, kn, vn, tab, kh, max(t0, least / kStep) * kStep, min(most, t1 * kStep), lane);
  cols_sum<T, DP>(w);
  if (rg.used > 1) {
    cols_part<T, DP>(w, a, q, s, kh, m0, split, rg.used, lane);
  } else {
    cols_store<T, DP>(w, a, q, s, kh, m0, lane);
    if (a.splits > 1) mark_whole(a, q, s, kh, m0, lane);
  }
}

int dp_of(int64_t dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }

struct Plan {
  bool rows_kernel;
  int64_t tiles, items;  // Args::tiles; work items but for splits and key heads
  int splits, waves, range;
};

// Which kernel, and into how many ranges the keys are cut.  Measured on one MI355X, us without -> with the rule:
//   more than 32 rows a (sequence, key head): paged_att_rows; 33 .. 64 as two tiles of paged_att_split read the keys
//     twice (128 x 8 heads x 36 rows over 4,096 keys 489 -> 379; 28 x 12 x 33 over 60: 12.2 -> 9.6)
//   paged_att_split: the ranges that fill one wave a SIMD (1,024), of at least 64 keys (8 waves over 768 keys:
//     16.2 -> 9.9, over 8,192: 18.4 -> 14.2; 64 over 2,048: 17.5 -> 13.4), all of them in one round (192 over 2,048 in
//     960 waves 37, in 1,152 49).  Where that leaves a range of more than 1,024 keys, more and shorter ones
//     (of 512 keys, or 8,192 in all) even out sequences of different lengths: 24 of up to 16,384 keys in ranges of 2,731
//     would wait for the longest.  Two ranges of one row tile are two waves of one workgroup, which needs no join
//     (384 over 512 keys: 25 -> 22), but never more than two (192 over 512 keys: 17.4 in two waves, 15.2 in ranges)
//   paged_att_rows: a workgroup a CU for ranges of 128 keys and more, all that the chip holds for 384 and more (8
//     over 1,024 keys: 20.8 -> 13.2; 32 over 16,384: 71 -> 55), but some 1,024 where ranges would be longer than 1,024
//     keys, for unequal lengths again (packed chunks of up to 64 over 8,192: 68 -> 53)
Plan plan_of(const mfl_paged_attention_args* p) {
  Plan r{};
  const int64_t G = p->heads / p->kv_heads, M = p->rows * G;
  const int64_t kv = p->max_kv < 1 ? 1 : p->max_kv;
  r.rows_kernel = M > kRowsW;
  const int64_t rows = r.rows_kernel ? kTileR : kRowsW, step = r.rows_kernel ? 2 * kKeys : kKeys;
  // tiles of a sequence; packed: of all together (they share p->total rows), and one behind the last
  int64_t base;
  if (p->offsets) {
    const int64_t most = p->n * ((M + rows - 1) / rows), few = (p->total * G + rows - 1) / rows + p->n;
    base = few < most ? few : most;
    r.items = r.tiles = base + 1;
  } else {
    r.tiles = (M + rows - 1) / rows;
    base = r.items = p->n * r.tiles;
  }
  base *= p->kv_heads;
  if (base < 1) base = 1;
  const int64_t all = (1023 + base) / base;  // ranges of a tile that make 1,024 in all
  int64_t sp;
  if (!r.rows_kernel) {
    const int64_t fill = base < 1024 ? 1024 / base : 1;
    int64_t range = (kv + fill - 1) / fill;
    if (range > 1024) range = kv * base / 8192 < 512 ? 512 : kv * base / 8192;
    if (range < 2 * kKeys) range = 2 * kKeys;
    sp = (kv + range - 1) / range;
    r.waves = sp == 2 && fill > 1 ? 2 : 1;
    if (r.waves == 2) sp = 1;
  } else {
    r.waves = kWavesR;
    const int64_t slots = dp_of(p->dim) == 128 ? 512 : 768;  // workgroups the chip holds at once
    if (4 * base <= slots) {
      const int64_t cus = kv / 128 < 192 / base ? kv / 128 : 192 / base;
      const int64_t held = kv / 384 < slots / base ? kv / 384 : slots / base;
      sp = cus > held ? cus : held;
      if (sp < 1) sp = 1;
      if (kv / sp > 1024 && sp < all) sp = all;
    } else {
      const int64_t least = 2 * base < slots ? 512 : 1024;
      sp = kv / least < all ? kv / least : all;
    }
  }
  if (sp < 1 || p->rows == 0) sp = 1;
  if (sp > 512) sp = 512;
  r.splits = (int)sp;
  r.range = (int)(((kv + sp - 1) / sp + step - 1) / step * step);
  return r;
}

int64_t slots_of(const mfl_paged_attention_args* p) { return p->offsets ? p->total : p->n * p->rows; }

int eb_of(int64_t dtype) { return dtype == 0 ? 4 : (dtype == 2 || dtype == 3) ? 2 : 0; }

// a mistake in the arguments: its text is set and false returned
bool check(const mfl_paged_attention_args* p) {
  const char* who = "mfl_paged_attention";
  if (!p) return mfl_paged_error("%s: NULL arguments", who);
  const int eb = eb_of(p->dtype);
  if (!eb) return mfl_paged_error("%s: dtype tag %lld (0 float32, 2 bfloat16, 3 float16)", who, (long long)p->dtype);
  if (p->n < 0 || p->rows < 0 || p->total < 0 || p->width < 0 || p->pages < 0)
    return mfl_paged_error("%s: negative sizes", who);
  if (p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads || p->heads > 4096)
    return mfl_paged_error("%s: heads %lld not a multiple of kv_heads %lld", who, (long long)p->heads,
                           (long long)p->kv_heads);
  if (p->dim < 1 || p->dim > 128 || p->dim * eb % 16)
    return mfl_paged_error("%s: dim %lld (at most 128, a multiple of 16 bytes)", who, (long long)p->dim);
  if (p->page_size < 1 || p->page_size > 1024 || (p->page_size & (p->page_size - 1)))
    return mfl_paged_error("%s: page_size %lld is no power of two up to 1024", who, (long long)p->page_size);
  if (p->width * p->page_size > (1ll << 30) || p->pages * p->kv_heads >= (1ll << 31))
    return mfl_paged_error("%s: a table row of more than 2^30 tokens, or 2^31 pages times key heads", who);
  if (!(p->scale > 0.0) || !(p->scale < 1e30)) return mfl_paged_error("%s: scale must be positive and finite", who);
  if ((p->k_new == nullptr) != (p->v_new == nullptr))
    return mfl_paged_error("%s: k_new and v_new come together", who);
  const int64_t st[] = {p->q_seq, p->q_row, p->q_head, p->k_seq, p->k_row, p->k_head, p->v_seq, p->v_row, p->v_head};
  for (int64_t v : st)
    if (v * eb % 16) return mfl_paged_error("%s: a stride is no multiple of 16 bytes", who);
  const void* al[] = {p->q, p->k_new, p->v_new, p->k_pages, p->v_pages, p->out, p->workspace};
  for (const void* v : al)
    if (reinterpret_cast<uintptr_t>(v) & 15u) return mfl_paged_error("%s: a pointer is not 16-byte aligned", who);
  const int64_t M = p->rows * (p->heads / p->kv_heads);
  if (p->rows > (1ll << 30) || M > (1ll << 30) || p->n > (1ll << 30) || slots_of(p) * p->heads >= (1ll << 31)) return mfl_paged_error("%s: too many rows", who);
  const Plan pl = plan_of(p);
  // (a launch holds fewer than 2^32 threads)
  if (pl.items > (1ll << 30) || pl.items * pl.splits * p->kv_heads * 64 * pl.waves >= (1ll << 32) ||
      (pl.splits > 1 && (slots_of(p) * p->heads + 256) * (dp_of(p->dim) / 4) >= (1ll << 32)))
    return mfl_paged_error("%s: too many sequences and rows for one launch", who);
  return true;
}

template <class T, int DP>
int launch(const Args& a, const Plan& pl, hipStream_t st) {
  const dim3 grid((unsigned)pl.items * (unsigned)pl.splits * (unsigned)a.kvh);
  if (pl.rows_kernel)
    hipLaunchKernelGGL((paged_att_rows<T, DP>), grid, dim3(64 * kWavesR), 0, st, a);
  else if (pl.waves == 1)
    hipLaunchKernelGGL((paged_att_split<T, DP, 1>), grid, dim3(64), 0, st, a);
  else
    hipLaunchKernelGGL((paged_att_split<T, DP, 2>), grid, dim3(128), 0, st, a);
  if (pl.splits > 1) {
    const long long rows = a.slots * a.heads;
    constexpr int kGr = 256 / (DP / 4);
    if (pl.splits > 16 && rows < (1 << 22))  // (a launch holds fewer than 2^32 threads)
      hipLaunchKernelGGL((paged_att_join<T, DP, true>), dim3((unsigned)rows * (DP / 32)), dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((paged_att_join<T, DP, false>), dim3((unsigned)((rows + kGr - 1) / kGr)), dim3(256), 0, st, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    mfl_paged_error("mfl_paged_attention: launch failed: %s", hipGetErrorString(e));
    return 1;
  }
  return 0;
}

template <class T>
int launch_dim(const Args& a, const Plan& pl, int dp, hipStream_t st) {
  if (dp == 32) return launch<T, 32>(a, pl, st);
  if (dp == 64) return launch<T, 64>(a, pl, st);
  return launch<T, 128>(a, pl, st);
}

thread_local char g_err[256] = "";

}  // namespace

bool mfl_paged_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return false;
}

extern "C" {

const char* mfl_paged_last_error(void) { return g_err; }

int64_t mfl_paged_attention_workspace_bytes(const mfl_paged_attention_args* p) {
  g_err[0] = 0;
  if (!check(p)) return -1;
  const Plan pl = plan_of(p);
  if (pl.splits == 1) return 0;
  const int64_t sh = slots_of(p) * p->heads;
  return ((sh + 3) / 4 * 4 + (pl.splits * sh * 2 + 3) / 4 * 4 + pl.splits * sh * dp_of(p->dim)) * 4;
}

int mfl_paged_attention(const mfl_paged_attention_args* p, void* stream) {
  g_err[0] = 0;
  if (!check(p)) return 1;
  if (p->n == 0 || p->rows == 0) {
    if (!(p->offsets && p->zero_tail && p->total > 0)) return 0;
  }
  // (what is empty has no address: a table without sequences or columns, a pool without pages)
  if (!p->out || (p->n > 0 && (!p->q || !p->kv_lens || (p->width > 0 && !p->table) ||
                               (p->pages > 0 && (!p->k_pages || !p->v_pages))))) {
    mfl_paged_error("mfl_paged_attention: NULL pointer");
    return 1;
  }
  const Plan pl = plan_of(p);
  if (pl.splits > 1 && !p->workspace) {
    mfl_paged_error("mfl_paged_attention: NULL workspace");
    return 1;
  }
  const int eb = eb_of(p->dtype);
  Args a;
  a.q = static_cast<const unsigned char*>(p->q);
  a.kn = static_cast<const unsigned char*>(p->k_new);
  a.vn = static_cast<const unsigned char*>(p->v_new);
  a.kp = static_cast<unsigned char*>(p->k_pages);
  a.vp = static_cast<unsigned char*>(p->v_pages);
  a.out = static_cast<unsigned char*>(p->out);
  a.ws = static_cast<float*>(p->workspace);
  a.table = p->table;
  a.kv_lens = p->kv_lens;
  a.starts = p->starts;
  a.offsets = p->offsets;
  a.n = (int)p->n;
  a.rows = (int)p->rows;
  a.heads = (int)p->heads;
  a.kvh = (int)p->kv_heads;
  a.G = (int)(p->heads / p->kv_heads);
  a.D = (int)p->dim;
  a.pages = (int)p->pages;
  a.ps = (int)p->page_size;
  a.sh = __builtin_ctzll((unsigned long long)p->page_size);
  a.width = (int)p->width;
  a.causal = p->causal != 0;
  a.splits = pl.splits;
  a.tiles = (int)pl.tiles;
  a.zero_tail = p->offsets && p->zero_tail;
  a.total = p->total;
  a.slots = slots_of(p);
  a.range = pl.range;
  a.q_seq = p->q_seq * eb, a.q_row = p->q_row * eb, a.q_head = p->q_head * eb;
  a.k_seq = p->k_seq * eb, a.k_row = p->k_row * eb, a.k_head = p->k_head * eb;
  a.v_seq = p->v_seq * eb, a.v_row = p->v_row * eb, a.v_head = p->v_head * eb;
  a.c = (float)p->scale * kLog2e;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int dp = dp_of(p->dim);
  if (p->dtype == 0) return launch_dim<float>(a, pl, dp, st);
  if (p->dtype == 2) return launch_dim<__bf16>(a, pl, dp, st);
  return launch_dim<_Float16>(a, pl, dp, st);
}

}  // extern "C"
