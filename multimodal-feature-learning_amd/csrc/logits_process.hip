// Penalties, biases and masks on logits (include/logits_process.h) for gfx950, with the row's best token and
// log-sum-exp: one pass over the logits, which bound it (each read once, each written once at most).
//
// A workgroup takes a tile of one row's vocabulary, eight tokens a thread, held in registers.  How often each
// token of the tile occurs in the row's history is counted in LDS (integer atomics: any order gives the same counts);
// the first of a token's occurrences to be seen again then penalises its logit once and leaves it in LDS, so that
// the dense pass only picks it up.  The row's history is read once per tile, out of the L2: long histories
// take tiles of 8,192 tokens (1,024 threads), short ones tiles of 2,048, of which there are more to fill the chip;
// a few rows of up to 16,384 tokens are one tile each, which needs no second launch.
// The best token goes by 64-bit keys (the value's order-preserving bits above the complement of the index: ties go to
// the lowest index, NaN above all).  Rows of one tile finish in the same launch, else logits_join merges the
// tiles' (key, sum of exponentials) pairs.
//
// Measured on one MI355X: 256 x 128,005 fp32 to fp32 with statistics, packed masks of 40 states, a bias and
// histories of up to 4,096: 70 us in logits_tile (3.8 TB/s) and 5 in logits_join, 77 to 80 a call; the histories are
// 20 of it, the masks 6 and the bias 5; with tiles of 4,096 tokens 6 us more.  While a workgroup counts and applies its
// history none of its logits are in flight, and each of a row's 16 tiles reads the history again.  112 x 10,000
// bf16, pick only: 8 us in one tile a row, 6 + 3 us in five and a join.
// Loads come before the history's phases: the bias fetched behind them cost 25 us of the large case.
//
// The arithmetic is the header's, operation by operation: contraction is off, so that equal logits stay
// equal and the pick does not depend on what the compiler fuses.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "logits_process.h"

#pragma clang fp contract(off)

namespace {

constexpr int kV = 8;                 // tokens a thread
constexpr int kFew = 256, kMany = 1024;  // threads a workgroup: short / long histories
// (tokens of history: 256 x 128,005 takes 65 us in small tiles and 68 in large ones at 800, 91 and 74 at 4,096;
// 32 x 50,000 takes 10.1 and 10.4, 15.4 and 10.9)
constexpr int kLongHistory = 2048;
// rows of up to 16,384 tokens that are one tile each: while all of their workgroups run at once, two a CU of one
// pass (512 x 3,000: 7.8 us, 9.2 in tiles and a join), one of two (256 x 10,000: 8.2, 10; 300 x 10,000: 14.1, 10.6)
constexpr int kFewRows = 512, kFewRows2 = 256;
constexpr int kTok = 4;               // tokens of the history a thread holds
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const unsigned char* logits;
  unsigned char* out;
  int64_t* best;
  float *lse, *logprob;
  const int *tokens, *token_lens;
  const float *rep, *pres, *freq, *bias;
  const unsigned char* allowed;
  const int* states;
  unsigned long long* keys;  // (n, tiles)
  float* sums;               // (n, tiles)
  int n, vocab, hist, kind, tiles, allowed_rows;
  long long logits_row, out_row, tokens_row, bias_row, allowed_row;
  float rep_s, pres_s, freq_s;
};

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(8))) float f32x8;
template <class T> struct Vec;
template <> struct Vec<float> { typedef f32x8 type; };
template <> struct Vec<__bf16> { typedef bf16x8 type; };
template <> struct Vec<_Float16> { typedef f16x8 type; };

// rows start at any multiple of the element size (odd vocabularies): vector accesses of element alignment
template <class T>
__device__ __forceinline__ void load8(const T* p, int m, float (&x)[kV]) {
  if (m >= kV) {
    typename Vec<T>::type v;
    __builtin_memcpy(&v, p, sizeof(v));
#pragma unroll
    for (int i = 0; i < kV; ++i) x[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i) x[i] = i < m ? (float)p[i] : 0.f;
  }
}
template <class T>
__device__ __forceinline__ void store8(T* p, int m, const float (&x)[kV]) {
  if (m >= kV) {
    typename Vec<T>::type v;
#pragma unroll
    for (int i = 0; i < kV; ++i) v[i] = (T)x[i];
    __builtin_memcpy(p, &v, sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i)
      if (i < m) p[i] = (T)x[i];
  }
}

// larger key = larger value, then lower index; NaN above everything
__device__ __forceinline__ unsigned long long key_of(float x, int v) {
  uint32_t u = __float_as_uint(x + 0.f);  // (-0 is +0)
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  if (x != x) u = 0xffffffffu;
  return ((unsigned long long)u << 32) | (uint32_t)~v;
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t u = (uint32_t)(k >> 32);
  if (u == 0xffffffffu) return NAN;
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ unsigned long long max_key(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

// the maximum a sum of exponentials is taken against: finite
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY || m != m || m == INFINITY ? 0.f : m; }

struct Stat {
  unsigned long long key;
  float m, s;  // maximum (NaN ignored) and sum of exp(x - base_of(m))
};

__device__ __forceinline__ float exp_diff(float x, float b) { return __builtin_amdgcn_exp2f((x - b) * kLog2e); }

__device__ __forceinline__ void merge(Stat& a, unsigned long long key, float m, float s) {
  const float mn = fmaxf(a.m, m), b = base_of(mn);
  // (a side that saw nothing has m = -inf and s = 0)
  a.s = (a.m == -INFINITY ? a.s : a.s * exp_diff(base_of(a.m), b)) + (m == -INFINITY ? s : s * exp_diff(base_of(m), b));
  a.m = mn;
  a.key = max_key(a.key, key);
}

// the wave's eight tokens a lane (the first m of them, index v and on)
__device__ __forceinline__ Stat wave_stat(const float (&x)[kV], int m, int v) {
  float mx = -INFINITY;
#pragma unroll
  for (int e = 0; e < kV; ++e) mx = fmaxf(mx, e < m ? x[e] : -INFINITY);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
  const float b = base_of(mx);
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < kV; ++e) s += e < m ? exp_diff(x[e], b) : 0.f;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  const bool nan = s != s;  // (the base is finite: only a NaN token makes one)
  int at = -1;
#pragma unroll
  for (int e = kV - 1; e >= 0; --e)
    if (e < m && (nan ? x[e] != x[e] : x[e] == mx)) at = v + e;
  const unsigned long long who = __ballot(at >= 0);  // (lanes hold ascending tokens)
  Stat t;
  t.key = who ? key_of(nan ? NAN : mx, __shfl(at, __builtin_ctzll(who))) : 0ull;
  t.m = mx;
  t.s = s;
  return t;
}

template <int THREADS>
__device__ __forceinline__ Stat block_stat(Stat t) {
  __shared__ unsigned long long sk[THREADS / 64];
  __shared__ float sm[THREADS / 64], ss[THREADS / 64];
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) sk[w] = t.key, sm[w] = t.m, ss[w] = t.s;
  __syncthreads();
  Stat r{0ull, -INFINITY, 0.f};
  if (threadIdx.x < 64) {
    const int i = threadIdx.x;
    if (i < THREADS / 64) r = Stat{sk[i], sm[i], ss[i]};
#pragma unroll
    for (int o = THREADS / 128; o > 0; o >>= 1) {
      const unsigned long long k = __shfl_xor(r.key, o);
      const float m = __shfl_xor(r.m, o), s = __shfl_xor(r.s, o);
      merge(r, k, m, s);
    }
  }
  return r;
}

__device__ __forceinline__ void finish(const Args& a, int row, const Stat& r) {
  const float top = key_value(r.key);
  float lse = base_of(r.m) + logf(r.s);
  if (top != top) lse = NAN;
  else if (top == INFINITY || top == -INFINITY) lse = top;
  if (a.best) a.best[row] = top == -INFINITY ? -1 : (int64_t)(uint32_t)~(uint32_t)r.key;
  if (a.lse) a.lse[row] = lse;
  // (a finite top is the maximum that the sum is taken against: -log s has the bits that top - lse would lose to top)
  const bool finite = top == top && top != INFINITY && top != -INFINITY;
  if (a.logprob) a.logprob[row] = finite ? 0.f - logf(r.s) : top == -INFINITY ? -INFINITY : NAN;
}

template <class T, class O, int THREADS, int NCH>
__global__ __launch_bounds__(THREADS, NCH == 1 ? 8 : 4) void logits_tile(Args a) {
  constexpr int kPass = THREADS * kV, kTile = kPass * NCH;
  __shared__ __attribute__((aligned(16))) float value[kTile];  // penalised logits, where count is not 0
  __shared__ __attribute__((aligned(16))) uint32_t count[kTile];
  const int row = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles;
  const int v0 = tile * kTile, nv = min(kTile, a.vocab - v0);
  const T* src = reinterpret_cast<const T*>(a.logits) + row * a.logits_row + v0;
  // the history's first kTok tokens a thread stay in registers, fetched with the logits
  const int len = a.hist == 0 ? 0 : a.token_lens ? max(0, min(a.token_lens[row], a.hist)) : a.hist;
  const int* tok = a.tokens + row * a.tokens_row;
  int held[kTok];
#pragma unroll
  for (int t = 0; t < kTok; ++t) {
    const int j = t * THREADS + (int)threadIdx.x;
    held[t] = j < len ? tok[j] : -1;
  }
  int mr = -1;  // mask row
  if (a.kind) {
    mr = a.states ? a.states[row] : (a.allowed_rows == 1 ? 0 : row);
    if ((unsigned)mr >= (unsigned)a.allowed_rows) mr = -1;
  }
  float x[NCH][kV], b[NCH][kV];  // everything the row needs is fetched before the history is counted
  uint32_t ok[NCH];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int i = c * kPass + (int)threadIdx.x * kV, m = max(0, min(kV, nv - i));
    ok[c] = 0xffu;
    if (m == 0) continue;
    load8(src + i, m, x[c]);
    if (a.bias) load8(a.bias + row * a.bias_row + v0 + i, m, b[c]);
    if (mr < 0) continue;
    if (a.kind == 2) {
      // (v0 and i are multiples of 8: the eight bits are one byte of a word)
      ok[c] = a.allowed[(long long)mr * a.allowed_row * 4 + (v0 + i) / 8];
    } else {
      const unsigned char* p = a.allowed + (long long)mr * a.allowed_row + v0 + i;
      unsigned long long w = 0;
      if (m == kV) {
        __builtin_memcpy(&w, p, 8);
      } else {
#pragma unroll
        for (int e = 0; e < kV; ++e)
          if (e < m) w |= (unsigned long long)p[e] << (8 * e);
      }
      ok[c] = 0;
#pragma unroll
      for (int e = 0; e < kV; ++e) ok[c] |= ((w >> (8 * e)) & 0xffu ? 1u : 0u) << e;
    }
  }
  if (len > 0) {
    const uint4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int i = c * kPass + (int)threadIdx.x * kV;
      if (i >= nv) continue;
      uint4* cp = reinterpret_cast<uint4*>(count + i);
      cp[0] = zero, cp[1] = zero;
    }
    __syncthreads();
    const auto add = [&](int v) {
      if ((unsigned)v < (unsigned)nv) atomicAdd(count + v, 1u);
    };
#pragma unroll
    for (int t = 0; t < kTok; ++t) add(held[t] - v0);
    for (int j = kTok * THREADS + threadIdx.x; j < len; j += THREADS) add(tok[j] - v0);
    const float rep = a.rep ? a.rep[row] : a.rep_s, pres = a.pres ? a.pres[row] : a.pres_s;
    const float freq = a.freq ? a.freq[row] : a.freq_s;
    __syncthreads();
    const auto apply = [&](int v) {
      if ((unsigned)v >= (unsigned)nv) return;
      const uint32_t c = atomicOr(count + v, 0x80000000u);
      if (c & 0x80000000u) return;  // (another occurrence has it)
      const float l = (float)src[v];
      float y = l > 0.f ? l / rep : l * rep;
      y = y - pres;
      value[v] = y - freq * (float)c;
    };
#pragma unroll
    for (int t = 0; t < kTok; ++t) apply(held[t] - v0);
    for (int j = kTok * THREADS + threadIdx.x; j < len; j += THREADS) apply(tok[j] - v0);
    __syncthreads();
  }
  const bool stats = a.best || a.lse || a.logprob;
  Stat t{0ull, -INFINITY, 0.f};
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int i = c * kPass + (int)threadIdx.x * kV, m = max(0, min(kV, nv - i));
    if (m > 0) {
      if (len > 0) {
        const uint4* cp = reinterpret_cast<const uint4*>(count + i);
        const uint4 n0 = cp[0], n1 = cp[1];
        const uint32_t n[kV] = {n0.x, n0.y, n0.z, n0.w, n1.x, n1.y, n1.z, n1.w};
        if (n[0] | n[1] | n[2] | n[3] | n[4] | n[5] | n[6] | n[7]) {
#pragma unroll
          for (int e = 0; e < kV; ++e) x[c][e] = n[e] ? value[i + e] : x[c][e];
        }
      }
      if (a.bias) {
#pragma unroll
        for (int e = 0; e < kV; ++e) x[c][e] = x[c][e] + b[c][e];
      }
#pragma unroll
      for (int e = 0; e < kV; ++e) x[c][e] = (ok[c] >> e) & 1u ? x[c][e] : -INFINITY;
      if (a.out) store8(reinterpret_cast<O*>(a.out) + row * a.out_row + v0 + i, m, x[c]);
    } else {
#pragma unroll
      for (int e = 0; e < kV; ++e) x[c][e] = -INFINITY;
    }
    if (stats) {
      const Stat u = wave_stat(x[c], m, v0 + i);
      if (NCH == 1)
        t = u;
      else
        merge(t, u.key, u.m, u.s);
    }
  }
  if (!stats) return;
  const Stat r = block_stat<THREADS>(t);
  if (threadIdx.x != 0) return;
  if (a.tiles == 1) {
    finish(a, row, r);
  } else {
    a.keys[(long long)row * a.tiles + tile] = r.key;
    // the sum against the tile's own maximum, which the key holds (with a NaN the sum is NaN)
    a.sums[(long long)row * a.tiles + tile] = r.s;
  }
}

__global__ __launch_bounds__(64) void logits_join(Args a) {
  const int row = blockIdx.x;
  Stat t{0ull, -INFINITY, 0.f};
  for (int i = threadIdx.x; i < a.tiles; i += 64) {
    const unsigned long long k = a.keys[(long long)row * a.tiles + i];
    const float m = key_value(k), s = a.sums[(long long)row * a.tiles + i];
    if (m != m) {  // a NaN: the row's sum is one whatever the others hold
      t.key = max_key(t.key, k);
      t.s = NAN;
    } else {
      merge(t, k, m, s);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned long long k = __shfl_xor(t.key, o);
    const float m = __shfl_xor(t.m, o), s = __shfl_xor(t.s, o);
    merge(t, k, m, s);
  }
  if (threadIdx.x == 0) finish(a, row, t);
}

thread_local char g_err[256] = "";

bool bad(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return false;
}

int esize(int64_t t) { return t == 0 ? 4 : t == 2 || t == 3 ? 2 : 0; }

struct Plan {
  int threads, passes, tiles;
};

Plan plan_of(const mfl_logits_args* p) {
  Plan r{p->hist > kLongHistory ? kMany : kFew, 1, 0};
  const int passes = p->vocab <= kMany * kV ? 1 : 2;
  if (p->n <= (passes == 1 ? kFewRows : kFewRows2) && p->vocab <= 2 * kMany * kV) {
    r.threads = p->vocab <= kFew * kV ? kFew : kMany;
    r.passes = passes;
  }
  const int64_t tile = (int64_t)r.threads * r.passes * kV;
  r.tiles = (int)((p->vocab + tile - 1) / tile);
  return r;
}

int tiles_of(const mfl_logits_args* p) { return plan_of(p).tiles; }

bool check(const mfl_logits_args* p) {
  const char* who = "mfl_logits_process";
  if (!p) return bad("%s: NULL arguments", who);
  if (p->n < 0 || p->n > (1 << 24) || p->vocab < 0 || p->vocab > (1 << 30) || p->hist < 0 || p->hist > (1 << 30))
    return bad("%s: n %lld, vocab %lld, hist %lld", who, (long long)p->n, (long long)p->vocab, (long long)p->hist);
  if (!esize(p->dtype) || !esize(p->out_dtype)) return bad("%s: dtype tag (0 float32, 2 bfloat16, 3 float16)", who);
  const Plan pl = plan_of(p);  // (a launch holds fewer than 2^32 threads)
  if (p->n * pl.tiles * pl.threads >= (1ll << 32) || p->n * 64 >= (1ll << 32)) return bad("%s: too many rows and tokens for one launch", who);
  if (p->allowed_kind < 0 || p->allowed_kind > 2) return bad("%s: allowed_kind %lld", who, (long long)p->allowed_kind);
  if (p->allowed_kind && (p->allowed_rows < 1 || p->allowed_rows > (1 << 30)))
    return bad("%s: allowed_rows %lld", who, (long long)p->allowed_rows);
  if (p->allowed_kind && !p->states && p->allowed_rows != 1 && p->allowed_rows < p->n)
    return bad("%s: %lld mask rows for %lld rows", who, (long long)p->allowed_rows, (long long)p->n);
  if (p->allowed_kind && p->allowed_rows > 1 &&
      p->allowed_row < (p->allowed_kind == 2 ? (p->vocab + 31) / 32 : p->vocab))
    return bad("%s: mask rows overlap", who);
  const float rep = (float)p->repetition;  // (the kernel divides by it)
  if (!p->repetition_rows && !(rep > 0.f && rep < INFINITY))
    return bad("%s: repetition must be positive and finite in float32", who);
  if (p->out == p->logits && p->out && (p->dtype != p->out_dtype || (p->n > 1 && p->out_row != p->logits_row)))
    return bad("%s: in place needs one type and stride", who);
  if (p->out && p->n > 1 && p->out_row < p->vocab) return bad("%s: rows of out overlap", who);
  return true;
}

template <class T, class O>
void launch_out(const Args& a, const Plan& pl, hipStream_t st) {
  const dim3 grid((unsigned)a.n * (unsigned)a.tiles);
  if (pl.passes == 2)
    hipLaunchKernelGGL((logits_tile<T, O, kMany, 2>), grid, dim3(kMany), 0, st, a);
  else if (pl.threads == kMany)
    hipLaunchKernelGGL((logits_tile<T, O, kMany, 1>), grid, dim3(kMany), 0, st, a);
  else
    hipLaunchKernelGGL((logits_tile<T, O, kFew, 1>), grid, dim3(kFew), 0, st, a);
}

template <class T>
void launch(const Args& a, int64_t out_dtype, const Plan& pl, hipStream_t st) {
  if (out_dtype == 0)
    launch_out<T, float>(a, pl, st);
  else if (out_dtype == 2)
    launch_out<T, __bf16>(a, pl, st);
  else
    launch_out<T, _Float16>(a, pl, st);
}

}  // namespace

extern "C" {

const char* mfl_logits_last_error(void) { return g_err; }

int64_t mfl_logits_workspace_bytes(const mfl_logits_args* p) {
  g_err[0] = 0;
  if (!check(p)) return -1;
  const int tiles = tiles_of(p);
  return tiles > 1 && (p->best || p->lse || p->logprob) ? p->n * tiles * 12 : 0;
}

int mfl_logits_process(const mfl_logits_args* p, void* stream) {
  g_err[0] = 0;
  if (!check(p)) return 1;
  if (p->n == 0) return 0;
  if (p->vocab == 0) {
    bad("mfl_logits_process: vocab 0");
    return 1;
  }
  if (!p->logits || (p->hist > 0 && !p->tokens) || (p->allowed_kind && !p->allowed)) {
    bad("mfl_logits_process: NULL pointer");
    return 1;
  }
  const int tiles = tiles_of(p);
  const bool stats = p->best || p->lse || p->logprob;
  if (tiles > 1 && stats && !p->workspace) {
    bad("mfl_logits_process: NULL workspace");
    return 1;
  }
  if (!stats && !p->out) return 0;
  Args a;
  a.logits = static_cast<const unsigned char*>(p->logits);
  a.out = static_cast<unsigned char*>(p->out);
  a.best = p->best, a.lse = p->lse, a.logprob = p->logprob;
  a.tokens = p->tokens, a.token_lens = p->token_lens;
  a.rep = p->repetition_rows, a.pres = p->presence_rows, a.freq = p->frequency_rows, a.bias = p->bias;
  a.allowed = static_cast<const unsigned char*>(p->allowed);
  a.states = p->states;
  a.keys = static_cast<unsigned long long*>(p->workspace);
  a.sums = reinterpret_cast<float*>(a.keys + (long long)p->n * tiles);
  a.n = (int)p->n, a.vocab = (int)p->vocab, a.hist = (int)p->hist, a.kind = (int)p->allowed_kind;
  a.tiles = tiles, a.allowed_rows = (int)p->allowed_rows;
  a.logits_row = p->logits_row, a.out_row = p->out_row, a.tokens_row = p->tokens_row;
  a.bias_row = p->bias_row, a.allowed_row = p->allowed_row;
  a.rep_s = (float)p->repetition, a.pres_s = (float)p->presence, a.freq_s = (float)p->frequency;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p->dtype == 0)
    launch<float>(a, p->out_dtype, plan_of(p), st);
  else if (p->dtype == 2)
    launch<__bf16>(a, p->out_dtype, plan_of(p), st);
  else
    launch<_Float16>(a, p->out_dtype, plan_of(p), st);
  if (tiles > 1 && stats) hipLaunchKernelGGL(logits_join, dim3((unsigned)a.n), dim3(64), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    bad("mfl_logits_process: launch failed: %s", hipGetErrorString(e));
    return 1;
  }
  return 0;
}

}  // extern "C"
