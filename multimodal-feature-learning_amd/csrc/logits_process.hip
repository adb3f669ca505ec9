// Penalties, biases and masks on logits (include/logits_process.h) for gfx950, with the row's best token and
// log-sum-exp: one pass over the logits, which bound it (each read once, each written once at most).
//
// A workgroup takes a tile of one row's vocabulary.  How often each token of the tile occurs in the row's
// history is counted in LDS (integer atomics: any order gives the same counts) — the history is read once per
// tile, out of the L2 — and the tile is streamed eight tokens a thread.  The best token is the maximum
// of 64-bit keys (the value's order-preserving bits above the complement of the index: ties go to the lowest
// index); the sum of exponentials is kept online in fp32 against a running maximum.  Rows of one tile finish in the same
// launch, else logits_join merges the tiles' (key, sum) pairs.
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

constexpr int kT = 256;
constexpr int kV = 8;           // tokens a thread takes at a time
constexpr int kTile = 8192;     // tokens a workgroup (their counts: 32 KB of LDS)

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
  float m, s;  // running maximum (NaN ignored) and sum of exp(x - base_of(m))
};

__device__ __forceinline__ void merge(Stat& a, unsigned long long key, float m, float s) {
  const float mn = fmaxf(a.m, m), b = base_of(mn);
  // (a side that saw nothing has m = -inf and s = 0)
  a.s = (a.m == -INFINITY ? a.s : a.s * expf(base_of(a.m) - b)) + (m == -INFINITY ? s : s * expf(base_of(m) - b));
  a.m = mn;
  a.key = max_key(a.key, key);
}

__device__ __forceinline__ Stat block_stat(Stat t) {
  __shared__ unsigned long long sk[kT / 64];
  __shared__ float sm[kT / 64], ss[kT / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned long long k = __shfl_xor(t.key, o);
    const float m = __shfl_xor(t.m, o), s = __shfl_xor(t.s, o);
    merge(t, k, m, s);
  }
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) sk[w] = t.key, sm[w] = t.m, ss[w] = t.s;
  __syncthreads();
  Stat r{sk[0], sm[0], ss[0]};
#pragma unroll
  for (int i = 1; i < kT / 64; ++i) merge(r, sk[i], sm[i], ss[i]);
  return r;
}

__device__ __forceinline__ void finish(const Args& a, int row, const Stat& r) {
  const float top = key_value(r.key);
  float lse = base_of(r.m) + logf(r.s);
  if (top != top) lse = NAN;
  else if (top == INFINITY || top == -INFINITY) lse = top;
  if (a.best) a.best[row] = top == -INFINITY ? -1 : (int64_t)(uint32_t)~(uint32_t)r.key;
  if (a.lse) a.lse[row] = lse;
  if (a.logprob) a.logprob[row] = top == -INFINITY ? -INFINITY : top - lse;
}

template <class T, class O>
__global__ __launch_bounds__(kT) void logits_tile(Args a) {
  __shared__ int count[kTile];
  const int row = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles;
  const int v0 = tile * kTile, nv = min(kTile, a.vocab - v0);
  bool any = false;
  if (a.hist > 0) {
    for (int i = threadIdx.x; i < nv; i += kT) count[i] = 0;
    __syncthreads();
    const int len = a.token_lens ? max(0, min(a.token_lens[row], a.hist)) : a.hist;
    const int* tok = a.tokens + row * a.tokens_row;
    for (int i = threadIdx.x; i < len; i += kT) {
      const int v = tok[i] - v0;
      if ((unsigned)v < (unsigned)nv) {
        atomicAdd(count + v, 1);
        any = true;
      }
    }
    any = __syncthreads_or(any);
  }
  const float rep = a.rep ? a.rep[row] : a.rep_s, pres = a.pres ? a.pres[row] : a.pres_s;
  const float freq = a.freq ? a.freq[row] : a.freq_s;
  const T* src = reinterpret_cast<const T*>(a.logits) + row * a.logits_row + v0;
  O* dst = a.out ? reinterpret_cast<O*>(a.out) + row * a.out_row + v0 : nullptr;
  const float* bias = a.bias ? a.bias + row * a.bias_row + v0 : nullptr;
  int mr = -1;  // mask row
  if (a.kind) {
    mr = a.states ? a.states[row] : (a.allowed_rows == 1 ? 0 : row);
    if ((unsigned)mr >= (unsigned)a.allowed_rows) mr = -1;
  }
  const bool stats = a.best || a.lse || a.logprob;
  Stat t{0ull, -INFINITY, 0.f};
  for (int i = threadIdx.x * kV; i < nv; i += kT * kV) {
    const int m = min(kV, nv - i);
    float x[kV];
    load8(src + i, m, x);
    if (any) {
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        const int c = e < m ? count[i + e] : 0;
        if (c > 0) {
          float y = x[e] > 0.f ? x[e] / rep : x[e] * rep;
          y = y - pres;
          x[e] = y - freq * (float)c;
        }
      }
    }
    if (bias) {
      float b[kV];
      load8(bias + i, m, b);
#pragma unroll
      for (int e = 0; e < kV; ++e) x[e] = x[e] + b[e];
    }
    if (mr >= 0) {
      uint32_t ok = 0;
      if (a.kind == 2) {
        // (v0 and i are multiples of 8: the eight bits are one byte of the word, in range with it)
        ok = a.allowed[(long long)mr * a.allowed_row * 4 + (v0 + i) / 8];
      } else {
        const unsigned char* p = a.allowed + (long long)mr * a.allowed_row + v0 + i;
#pragma unroll
        for (int e = 0; e < kV; ++e) ok |= (e < m && p[e] != 0 ? 1u : 0u) << e;
      }
#pragma unroll
      for (int e = 0; e < kV; ++e) x[e] = (ok >> e) & 1u ? x[e] : -INFINITY;
    }
    if (dst) store8(dst + i, m, x);
    if (stats) {
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < kV; ++e)
        if (e < m) {
          mx = fmaxf(mx, x[e]);
          t.key = max_key(t.key, key_of(x[e], v0 + i + e));
        }
      if (mx > t.m) {
        if (t.m != -INFINITY) t.s *= expf(base_of(t.m) - base_of(mx));
        t.m = mx;
      }
      const float b = base_of(t.m);
#pragma unroll
      for (int e = 0; e < kV; ++e)
        if (e < m) t.s += expf(x[e] - b);
    }
  }
  if (!stats) return;
  const Stat r = block_stat(t);
  if (threadIdx.x != 0) return;
  if (a.tiles == 1) {
    finish(a, row, r);
  } else {
    a.keys[(long long)row * a.tiles + tile] = r.key;
    // the sum against the tile's own maximum, which the key holds (NaN: the sum is NaN already)
    a.sums[(long long)row * a.tiles + tile] = r.s;
  }
}

__global__ __launch_bounds__(kT) void logits_join(Args a) {
  const int row = blockIdx.x;
  Stat t{0ull, -INFINITY, 0.f};
  for (int i = threadIdx.x; i < a.tiles; i += kT) {
    const unsigned long long k = a.keys[(long long)row * a.tiles + i];
    const float m = key_value(k), s = a.sums[(long long)row * a.tiles + i];
    if (m != m) {  // a NaN: the row's sum is one whatever the others hold
      t.key = max_key(t.key, k);
      t.s = NAN;
    } else {
      merge(t, k, m, s);
    }
  }
  const Stat r = block_stat(t);
  if (threadIdx.x == 0) finish(a, row, r);
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

int tiles_of(const mfl_logits_args* p) { return (int)((p->vocab + kTile - 1) / kTile); }

bool check(const mfl_logits_args* p) {
  const char* who = "mfl_logits_process";
  if (!p) return bad("%s: NULL arguments", who);
  if (p->n < 0 || p->n > (1 << 24) || p->vocab < 0 || p->vocab > (1 << 30) || p->hist < 0 || p->hist > (1 << 30))
    return bad("%s: n %lld, vocab %lld, hist %lld", who, (long long)p->n, (long long)p->vocab, (long long)p->hist);
  if (!esize(p->dtype) || !esize(p->out_dtype)) return bad("%s: dtype tag (0 float32, 2 bfloat16, 3 float16)", who);
  if (p->n * tiles_of(p) >= (1ll << 31)) return bad("%s: too many rows and tokens for one launch", who);
  if (p->allowed_kind < 0 || p->allowed_kind > 2) return bad("%s: allowed_kind %lld", who, (long long)p->allowed_kind);
  if (p->allowed_kind && (p->allowed_rows < 1 || p->allowed_rows > (1 << 30)))
    return bad("%s: allowed_rows %lld", who, (long long)p->allowed_rows);
  if (p->allowed_kind && !p->states && p->allowed_rows != 1 && p->allowed_rows < p->n)
    return bad("%s: %lld mask rows for %lld rows", who, (long long)p->allowed_rows, (long long)p->n);
  if (p->allowed_kind && p->allowed_rows > 1 &&
      p->allowed_row < (p->allowed_kind == 2 ? (p->vocab + 31) / 32 : p->vocab))
    return bad("%s: mask rows overlap", who);
  if (!p->repetition_rows && !(p->repetition > 0.0)) return bad("%s: repetition must be positive", who);
  if (p->out == p->logits && p->out && (p->dtype != p->out_dtype || (p->n > 1 && p->out_row != p->logits_row)))
    return bad("%s: in place needs one type and stride", who);
  if (p->out && p->n > 1 && p->out_row < p->vocab) return bad("%s: rows of out overlap", who);
  return true;
}

template <class T>
void launch(const Args& a, int64_t out_dtype, hipStream_t st) {
  const dim3 grid((unsigned)a.n * (unsigned)a.tiles);
  if (out_dtype == 0)
    hipLaunchKernelGGL((logits_tile<T, float>), grid, dim3(kT), 0, st, a);
  else if (out_dtype == 2)
    hipLaunchKernelGGL((logits_tile<T, __bf16>), grid, dim3(kT), 0, st, a);
  else
    hipLaunchKernelGGL((logits_tile<T, _Float16>), grid, dim3(kT), 0, st, a);
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
    launch<float>(a, p->out_dtype, st);
  else if (p->dtype == 2)
    launch<__bf16>(a, p->out_dtype, st);
  else
    launch<_Float16>(a, p->out_dtype, st);
  if (tiles > 1 && stats) hipLaunchKernelGGL(logits_join, dim3((unsigned)a.n), dim3(kT), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    bad("mfl_logits_process: launch failed: %s", hipGetErrorString(e));
    return 1;
  }
  return 0;
}

}  // extern "C"
