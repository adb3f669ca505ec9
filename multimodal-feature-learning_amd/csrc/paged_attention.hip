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
// values' 16-bit type for the matrix product (relative 2^-9 / 2^-12 of each weight, against the output's
// own rounding of the same size); l sums the unrounded weights.
//
//   paged_att_split  few rows a (sequence, key head): a workgroup takes 32 rows and a range of the keys,
//                    its waves equal parts of the range; the waves' (m, l, O) meet in LDS, the ranges' in
//   paged_att_join   the workspace.
//   paged_att_rows   many rows: 4 waves of 32 rows share 64-key tiles in LDS.
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
  long long total;
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
  long long q0;          // packed: first row; else 0 (the sequence stride is in the base pointers)
};

__device__ __forceinline__ Seq seq_of(const Args& a, int s) {
  Seq q;
  q.kv = max(0, min(a.kv_lens[s], a.width * a.ps));  // (width * page_size < 2^31: checked on the host)
  q.q0 = 0;
  q.rows = a.rows;
  int len = a.rows;
  if (a.offsets) {
    const long long o0 = max(0ll, min((long long)a.offsets[s], a.total));
    const long long o1 = max(o0, min((long long)a.offsets[s + 1], a.total));
    q.q0 = o0;
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

// the rows of a wave, as MFMA columns
template <class T, int DP>
struct Cols {
  uint4 qf[Geo<T, DP>::QF];
  f32x16 o[Geo<T, DP>::OB];
  float m, l;
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

// scores of keys j0 .. j0+31 that the lane's row does not see become -inf; `there` bit kk: key j0+kk exists
__device__ __forceinline__ void mask_scores(f32x16& s, int j0, int lim, uint32_t there, int lane) {
  const int h = lane >> 5;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int kk = 8 * (e >> 2) + 4 * h + (e & 3);
    if (j0 + kk >= lim || !((there >> kk) & 1u)) s[e] = -INFINITY;
  }
}

// the online softmax's step for NT score tiles: m, l and O rescaled, s replaced by the weights
template <class T, int DP, int NT>
__device__ __forceinline__ void soft_step(Cols<T, DP>& w, f32x16 (&s)[NT], float c) {
  float mx = s[0][0];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[t][e]);
  mx = fmaxf(mx, __shfl_xor(mx, 32));
  const float mn = fmaxf(w.m, mx);
  const float base = mn == -INFINITY ? 0.f : mn * c;  // (nothing seen yet: every weight is 2^-inf = 0)
  const float al = __builtin_amdgcn_exp2f(fmaf(w.m, c, -base));
  float sum = 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[t][e] = __builtin_amdgcn_exp2f(fmaf(s[t][e], c, -base));
      sum += s[t][e];
    }
  sum += __shfl_xor(sum, 32);
  w.l = w.l * al + sum;
  w.m = mn;
#pragma unroll
  for (int d = 0; d < Geo<T, DP>::OB; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) w.o[d][e] *= al;
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

// packed rows behind the last sequence's
__device__ __forceinline__ void zero_rows(const Args& a, int part, int parts, int eb) {
  const long long r0 = max(0ll, min((long long)a.offsets[a.n], a.total));
  const long long per = (long long)a.heads * a.D * eb / 16;
  uint4* dst = reinterpret_cast<uint4*>(a.out) + r0 * per;
  for (long long e = (long long)part * blockDim.x + threadIdx.x; e < (a.total - r0) * per;
       e += (long long)parts * blockDim.x)
    dst[e] = uint4{0, 0, 0, 0};
}

// grid: x = splits * tiles (tile major), y = kv heads, z folded into x through n (x = ((s * tiles) + tile) *
// splits + split; s == n: the rows behind the last sequence)
template <class T, int DP, int NW>
__global__ __launch_bounds__(64 * NW) void paged_att_split(Args a) {
  typedef Geo<T, DP> Ge;
  constexpr int kImg = kKeys * Ge::RB;                       // one 32-row image
  constexpr int kMerge = NW > 1 ? NW * 32 * (DP + 1) * 4 : 0;
  constexpr int kLds = NW * 2 * kImg > kMerge ? NW * 2 * kImg : kMerge;
  __shared__ __attribute__((aligned(16))) unsigned char lds[kLds];
  __shared__ float s_m[NW][32], s_l[NW][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  int x = blockIdx.x;
  const int split = x % a.splits;
  x /= a.splits;
  const int tile = x % a.tiles, s = x / a.tiles, kh = blockIdx.y;
  if (s >= a.n) {
    zero_rows(a, (tile * a.splits + split) * a.kvh + kh, a.tiles * a.splits * a.kvh, Ge::EB);
    return;
  }
  const Seq q = seq_of(a, s);
  const int m0 = tile * kRowsW;
  if (m0 >= q.rows * a.G) return;  // (uniform over the workgroup; the join skips these tiles the same way)
  const long long seq = a.offsets ? 0 : s;
  const unsigned char* qb = a.q + seq * a.q_seq + q.q0 * a.q_row;
  const unsigned char* kn = a.kn ? a.kn + seq * a.k_seq + q.q0 * a.k_row + (long long)kh * a.k_head : nullptr;
  const unsigned char* vn = a.vn ? a.vn + seq * a.v_seq + q.q0 * a.v_row + (long long)kh * a.v_head : nullptr;
  Cols<T, DP> w;
  cols_init<T, DP>(w, a, q, qb, kh, m0, lane);
  // the last row of the tile sees the most keys
  const int ilast = min(q.rows - 1, (m0 + kRowsW - 1) / a.G);
  const int most = a.causal ? max(0, min(q.kv, q.st + ilast + 1)) : q.kv;
  const int nblk = (most + kKeys - 1) / kKeys;
  const int per = (nblk + a.splits - 1) / a.splits;
  const int b0 = split * per, b1 = min(nblk, b0 + per);
  const int wper = (max(0, b1 - b0) + NW - 1) / NW;
  const int w0 = b0 + wave * wper, w1 = min(b1, w0 + wper);
  unsigned char* kt = lds + wave * 2 * kImg;
  unsigned char* vt = kt + kImg;
  const int* tab = a.table + (long long)s * a.width;
  const int rb = a.D * Ge::EB, nch = rb / 16;
  constexpr int kIt = kImg / 1024;  // 16-byte loads a lane for one image
  int pbase = 0, pg = 0;
  uint4 rk[kIt], rv[kIt];
  uint32_t there = 0;
  bool odd = false;  // a value that is not finite was scrubbed
  const int least = a.causal ? max(0, min(q.kv, q.st + m0 / a.G + 1)) : q.kv;  // keys the tile's first row sees
  const auto fetch = [&](int blk) {
    const int j0 = blk * kKeys;
    const int pi0 = j0 >> a.sh;
    if (blk == w0 || pi0 - pbase + ((kKeys - 1) >> a.sh) >= 64) {  // the table's next 64 entries, one a lane
      pbase = pi0;
      const int e = pbase + lane;
      pg = e < a.width ? tab[e] : -1;
    }
#pragma unroll
    for (int t = 0; t < kIt; ++t) {
      const int ci = t * 64 + lane, row = ci / Ge::NC, cp = ci % Ge::NC;
      const int j = j0 + row;
      const int page = __shfl(pg, (j >> a.sh) - pbase);
      RowSrc r;
      row_src(a, q, kn, vn, kh, j, page, rb, r);
      const int ck = cp ^ Ge::k_swz(row), cv = cp ^ Ge::v_swz(row);
      rk[t] = ck < nch ? *reinterpret_cast<const uint4*>(r.k + ck * 16) : uint4{0, 0, 0, 0};
      rv[t] = cv < nch ? *reinterpret_cast<const uint4*>(r.v + cv * 16) : uint4{0, 0, 0, 0};
    }
    const int j = j0 + (lane & 31);
    const int page = __shfl(pg, (j >> a.sh) - pbase);
    there = (uint32_t)__ballot(j < q.kv && (unsigned)page < (unsigned)a.pages);
  };
  if (w0 < w1) fetch(w0);
  for (int blk = w0; blk < w1; ++blk) {
    if (least < min(q.kv, (blk + 1) * kKeys)) {
#pragma unroll
      for (int t = 0; t < kIt; ++t) odd |= scrub<T>(rv[t]);
    }
#pragma unroll
    for (int t = 0; t < kIt; ++t) {
      *reinterpret_cast<uint4*>(kt + (t * 64 + lane) * 16) = rk[t];
      *reinterpret_cast<uint4*>(vt + (t * 64 + lane) * 16) = rv[t];
    }
    const uint32_t now = there;
    if (blk + 1 < w1) fetch(blk + 1);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the wave's own LDS writes; no other wave reads them)
    f32x16 sc[1];
    sc[0] = scores<T, DP>(w, kt, lane);
    const bool full = now == 0xffffffffu && __all((blk + 1) * kKeys <= w.lim);
    if (!full) mask_scores(sc[0], blk * kKeys, w.lim, now, lane);
    soft_step<T, DP, 1>(w, sc, a.c);
    weigh<T, DP>(w, sc[0], vt, lane);
  }
  if (__any(odd))
    add_non_finite<T, DP>(w, a, q, kn, vn, tab, kh, max(w0, least / kKeys) * kKeys, min(most, w1 * kKeys), lane);
  if (a.kn && split == 0) {
    // the tile writes the tokens whose first row it holds
    const int i0 = (m0 + a.G - 1) / a.G, i1 = min(q.rows, (m0 + kRowsW + a.G - 1) / a.G);
    write_chunk<T>(a, q, s, kn, vn, kh, i0, i1, threadIdx.x, 64 * NW);
  }
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
  if (a.splits == 1) {
    cols_store<T, DP>(w, a, q, s, kh, m0, lane);
    return;
  }
  // partial: per (s, kh, tile, split): 32 maxima, 32 sums, then 32 rows of DP
  const long long id = (((long long)s * a.kvh + kh) * a.tiles + tile) * a.splits + split;
  float* ws = a.ws + id * (64 + 32 * DP);
  const int col = lane & 31, h = lane >> 5;
  if (h == 0) {
    ws[col] = w.m;
    ws[32 + col] = w.l;
  }
#pragma unroll
  for (int d = 0; d < Ge::OB; ++d)
#pragma unroll
    for (int b = 0; b < 4; ++b)
      *reinterpret_cast<f32x4*>(ws + 64 + col * DP + d * 32 + 8 * b + 4 * h) =
          f32x4{w.o[d][4 * b], w.o[d][4 * b + 1], w.o[d][4 * b + 2], w.o[d][4 * b + 3]};
}

// one workgroup a (sequence, key head, tile): out = sum_i 2^(c (m_i - m)) O_i / sum_i 2^(c (m_i - m)) l_i
template <class T, int DP>
__global__ __launch_bounds__(256) void paged_att_join(Args a) {
  const int tile = blockIdx.x % a.tiles, s = blockIdx.x / a.tiles, kh = blockIdx.y;
  const Seq q = seq_of(a, s);
  const int m0 = tile * kRowsW;
  const int nrow = min(kRowsW, q.rows * a.G - m0);
  if (nrow <= 0) return;
  const long long id = (((long long)s * a.kvh + kh) * a.tiles + tile) * a.splits;
  const float* ws = a.ws + id * (64 + 32 * DP);
  constexpr int kQ = DP / 4;  // quads a row
  for (int e = threadIdx.x; e < nrow * kQ; e += 256) {
    const int r = e / kQ, col = (e % kQ) * 4;
    if (col >= a.D) continue;
    float mx = -INFINITY;
    for (int i = 0; i < a.splits; ++i) mx = fmaxf(mx, ws[(long long)i * (64 + 32 * DP) + r]);
    const float base = mx == -INFINITY ? 0.f : mx * a.c;
    float l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < a.splits; ++i) {
      const float* p = ws + (long long)i * (64 + 32 * DP);
      const float f = __builtin_amdgcn_exp2f(fmaf(p[r], a.c, -base));
      l += p[32 + r] * f;
      const f32x4 v = *reinterpret_cast<const f32x4*>(p + 64 + r * DP + col);
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] += v[k] * f;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    const int row = m0 + r, i = row / a.G, g = row - i * a.G;
    const long long rr = (a.offsets ? q.q0 : (long long)s * a.rows) + i;
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = o[k] * inv;
    store4<T>(a.out + ((rr * a.heads + kh * a.G + g) * (long long)a.D + col) * (long long)sizeof(T), v);
  }
}

constexpr int kWavesR = 4;
constexpr int kTileR = kWavesR * kRowsW;  // rows a workgroup of paged_att_rows

template <class T, int DP>
__global__ __launch_bounds__(64 * kWavesR) void paged_att_rows(Args a) {
  typedef Geo<T, DP> Ge;
  constexpr int NT = Ge::EB == 2 ? 2 : 1;         // score tiles a step (64 or 32 keys)
  constexpr int kImg = NT * kKeys * Ge::RB;
  constexpr int kThreads = 64 * kWavesR;
  constexpr int kIt = kImg / (16 * kThreads);
  static_assert(kIt >= 1, "an image holds at least 16 bytes a thread");
  __shared__ __attribute__((aligned(16))) unsigned char lds[2 * kImg];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kh = blockIdx.y;
  int x = blockIdx.x;
  const int tile = a.tiles - 1 - x % a.tiles, s = x / a.tiles;  // (the longest tiles of a sequence first)
  if (s >= a.n) {
    zero_rows(a, tile * a.kvh + kh, a.tiles * a.kvh, Ge::EB);
    return;
  }
  const Seq q = seq_of(a, s);
  const int g0 = tile * kTileR;
  if (g0 >= q.rows * a.G) return;
  const int m0 = g0 + wave * kRowsW;
  const long long seq = a.offsets ? 0 : s;
  const unsigned char* qb = a.q + seq * a.q_seq + q.q0 * a.q_row;
  const unsigned char* kn = a.kn ? a.kn + seq * a.k_seq + q.q0 * a.k_row + (long long)kh * a.k_head : nullptr;
  const unsigned char* vn = a.vn ? a.vn + seq * a.v_seq + q.q0 * a.v_row + (long long)kh * a.v_head : nullptr;
  Cols<T, DP> w;
  cols_init<T, DP>(w, a, q, qb, kh, m0, lane);
  const int ilast = min(q.rows - 1, (g0 + kTileR - 1) / a.G);
  const int most = a.causal ? max(0, min(q.kv, q.st + ilast + 1)) : q.kv;
  constexpr int kStep = NT * kKeys;
  const int nstep = (most + kStep - 1) / kStep;
  const int* tab = a.table + (long long)s * a.width;
  const int rb = a.D * Ge::EB, nch = rb / 16;
  unsigned char *kt = lds, *vt = lds + kImg;
  uint4 rk[kIt], rv[kIt];
  uint32_t bad = 0;
  bool odd = false;  // a value that is not finite was scrubbed
  const int least = a.causal ? max(0, min(q.kv, q.st + g0 / a.G + 1)) : q.kv;  // keys the tile's first row sees
  const auto fetch = [&](int step) {
    const int j0 = step * kStep;
    bad = 0;
#pragma unroll
    for (int t = 0; t < kIt; ++t) {
      const int ci = t * kThreads + tid;
      const int row = ci / Ge::NC, cp = ci % Ge::NC, j = j0 + row;
      const int page = j < q.kv ? tab[j >> a.sh] : -1;
      RowSrc r;
      if (!row_src(a, q, kn, vn, kh, j, page, rb, r) && j < q.kv) bad |= 1u;
      const int ck = cp ^ Ge::k_swz(row & 31), cv = cp ^ Ge::v_swz(row);
      rk[t] = ck < nch ? *reinterpret_cast<const uint4*>(r.k + ck * 16) : uint4{0, 0, 0, 0};
      rv[t] = cv < nch ? *reinterpret_cast<const uint4*>(r.v + cv * 16) : uint4{0, 0, 0, 0};
    }
  };
  if (nstep > 0) fetch(0);
  for (int step = 0; step < nstep; ++step) {
    // (also: every wave is done with the last tiles)
    const bool any_bad = __syncthreads_or(bad != 0u);
    if (least < min(q.kv, (step + 1) * kStep)) {
#pragma unroll
      for (int t = 0; t < kIt; ++t) odd |= scrub<T>(rv[t]);
    }
#pragma unroll
    for (int t = 0; t < kIt; ++t) {
      const int ci = t * kThreads + tid;
      *reinterpret_cast<uint4*>(kt + ci * 16) = rk[t];
      *reinterpret_cast<uint4*>(vt + ci * 16) = rv[t];
    }
    __syncthreads();
    if (step + 1 < nstep) fetch(step + 1);
    const int j0 = step * kStep;
    if (__all(j0 >= w.lim)) continue;  // (nothing of this tile is visible to the wave's rows)
    f32x16 sc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) sc[t] = scores<T, DP>(w, kt + t * kKeys * Ge::RB, lane);
    const bool full = !any_bad && __all(j0 + kStep <= w.lim);
    if (!full) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        uint32_t there = 0xffffffffu;
        if (any_bad) {
          const int j = j0 + t * kKeys + (lane & 31);
          const int page = j < q.kv ? tab[j >> a.sh] : -1;
          there = (uint32_t)__ballot((unsigned)page < (unsigned)a.pages);
        }
        mask_scores(sc[t], j0 + t * kKeys, w.lim, there, lane);
      }
    }
    soft_step<T, DP, NT>(w, sc, a.c);
#pragma unroll
    for (int t = 0; t < NT; ++t) weigh<T, DP>(w, sc[t], vt + t * kKeys * Ge::RB, lane);
  }
  if (least < most && __syncthreads_or(odd))
    add_non_finite<T, DP>(w, a, q, kn, vn, tab, kh, least / kStep * kStep, most, lane);
  if (a.kn) {
    const int i0 = (g0 + a.G - 1) / a.G, i1 = min(q.rows, (g0 + kTileR + a.G - 1) / a.G);
    write_chunk<T>(a, q, s, kn, vn, kh, i0, i1, tid, kThreads);
  }
  cols_store<T, DP>(w, a, q, s, kh, m0, lane);
}

struct Plan {
  bool rows_kernel;
  int tiles, splits, waves;
};

Plan plan_of(const mfl_paged_attention_args* p) {
  Plan r{};
  const int64_t G = p->heads / p->kv_heads, M = p->rows * G;
  const int64_t kv = p->max_kv < 1 ? 1 : p->max_kv;
  r.rows_kernel = M > 2 * kRowsW;
  if (r.rows_kernel) {
    r.tiles = (int)((M + kTileR - 1) / kTileR);
    r.splits = 1;
    r.waves = kWavesR;
    return r;
  }
  r.tiles = (int)((M + kRowsW - 1) / kRowsW);
  r.waves = kv <= 2 * kKeys ? 1 : 4;
  const int64_t base = p->n * p->kv_heads * r.tiles;
  int64_t sp = base > 0 ? (512 + base - 1) / base : 1;
  const int64_t most = (kv + 4 * 2 * kKeys - 1) / (4 * 2 * kKeys);
  if (sp > most) sp = most;
  if (sp > 256) sp = 256;
  if (r.waves == 1) sp = 1;
  r.splits = (int)(sp < 1 ? 1 : sp);
  return r;
}

int dp_of(int64_t dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }

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
  if (p->width * p->page_size > (1ll << 30) || p->pages > (1ll << 30))
    return mfl_paged_error("%s: a table row of more than 2^30 tokens, or more than 2^30 pages", who);
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
  if (p->rows > (1ll << 30) || M > (1ll << 30)) return mfl_paged_error("%s: too many rows", who);
  const Plan pl = plan_of(p);
  if ((p->n + 1) * pl.tiles * pl.splits >= (1ll << 31))
    return mfl_paged_error("%s: too many sequences and rows for one launch", who);
  return true;
}

template <class T, int DP>
int launch(const Args& a, const Plan& pl, hipStream_t st) {
  const unsigned seqs = (unsigned)a.n + (a.zero_tail ? 1u : 0u);
  const dim3 grid(seqs * (unsigned)pl.tiles * (unsigned)pl.splits, (unsigned)a.kvh);
  if (pl.rows_kernel) {
    hipLaunchKernelGGL((paged_att_rows<T, DP>), grid, dim3(64 * kWavesR), 0, st, a);
  } else {
    if (pl.waves == 1)
      hipLaunchKernelGGL((paged_att_split<T, DP, 1>), grid, dim3(64), 0, st, a);
    else
      hipLaunchKernelGGL((paged_att_split<T, DP, 4>), grid, dim3(256), 0, st, a);
    if (pl.splits > 1)
      hipLaunchKernelGGL((paged_att_join<T, DP>), dim3((unsigned)a.n * (unsigned)pl.tiles, (unsigned)a.kvh), dim3(256),
                         0, st, a);
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
  return p->n * p->kv_heads * pl.tiles * pl.splits * (64 + 32 * dp_of(p->dim)) * 4;
}

int mfl_paged_attention(const mfl_paged_attention_args* p, void* stream) {
  g_err[0] = 0;
  if (!check(p)) return 1;
  if (p->n == 0 || p->rows == 0) {
    if (!(p->offsets && p->zero_tail && p->total > 0)) return 0;
  }
  // (without sequences only the rows behind them are set: an empty table has no address)
  if (!p->out || (p->n > 0 && (!p->q || !p->k_pages || !p->v_pages || !p->table || !p->kv_lens))) {
    mfl_paged_error("mfl_paged_attention: NULL pointer");
    return 1;
  }
  Plan pl = plan_of(p);
  if (pl.tiles < 1) pl.tiles = 1;
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
  a.tiles = pl.tiles;
  a.zero_tail = p->offsets && p->zero_tail;
  a.total = p->total;
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
