// A paged cache of keys and values as its kernels see it (bnh_kv_append, bnh_kv_select, bnh_kv_attn), with the checks of
// what the device holds: lengths, places and pages outside their buffers are cut or taken as not there.
#ifndef BNH_KV_H
#define BNH_KV_H
#include "bnh_internal.h"
#include "bnh_f16.h"

struct KvDev {
  void *k, *v;
  long long k_ps, v_ps;
  void *lo, *hi;
  const int32_t *table, *past, *start, *len;
  int pages, sh, Hk, dk, dv, ldt, T, rows;  // sh: log2 of the tokens to a page
};

// An int that all lanes have, through the scalar cache whatever the kernel has stored before: for what nothing stores to while it
// is read
__device__ __forceinline__ int kv_int(const int32_t *p, long long i) {
  typedef __attribute__((address_space(4))) const int32_t *P;
  return __builtin_amdgcn_readfirstlane(((P)(uintptr_t)p)[i]);
}
// sequence b's (the same in all lanes) first row, its rows (cut to T and to the buffers' rows) and the tokens ahead of them
__device__ __forceinline__ int kv_rows(const KvDev &c, int b, int *first, int *past) {
  b = __builtin_amdgcn_readfirstlane(b);
  const long long s = c.start ? kv_int(c.start, b) : (long long)b * c.T;
  long long n = c.len ? kv_int(c.len, b) : c.T;
  const int m = kv_int(c.past, b);
  *past = m > 0 ? m : 0;
  n = n < c.T ? n : c.T;
  if (s < 0 || s >= c.rows) n = 0;
  else n = n < c.rows - s ? n : c.rows - s;
  n = n < 0x7ffffff0 - *past ? n : 0x7ffffff0 - *past;
  *first = (int)s;
  return n < 0 ? 0 : (int)n;
}
// the page of the pool that holds page i of sequence b; -1: none
__device__ __forceinline__ int kv_page(const KvDev &c, int b, int i) {
  if ((unsigned)i >= (unsigned)c.ldt) return -1;
  const int p = c.table[(long long)b * c.ldt + i];
  return (unsigned)p < (unsigned)c.pages ? p : -1;
}
// N values of a row from its value c, zeros from value n on. V: N divides c and n and the row is aligned to the N values
// or to 16 bytes
template <typename T, int N>
using kv_vec = T __attribute__((ext_vector_type(N), aligned(sizeof(T) * N < 16 ? sizeof(T) * N : 16)));
// Where they are not: N values from a place in the row, the last ones for a c near its end, so that every load is one; and what
// kv_ld gives of them, once they are there. A row of fewer than N values is read value by value: fp16, what is there; fp32, some
// value for the others, or the tests for them cost the rows that are not so few (64 rows over up to 4,000 tokens, 12 heads of
// 127: 225 us, 313 with tests; fp16, up to 17,279 tokens: 451 us, 359 with tests)
template <typename T, int N>
__device__ __forceinline__ kv_vec<T, N> kv_raw(const T *p, int c, int n) {
  kv_vec<T, N> r;
  if (n >= N) {
    __builtin_memcpy(&r, p + (c <= n - N ? c : c < n ? n - N : 0), N * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) {
      if (sizeof(T) == 2) r[i] = c + i < n ? p[c + i] : (T)0;
      else r[i] = p[c + i < n ? c + i : 0];
    }
  }
  return r;
}
template <typename T, int N>
__device__ __forceinline__ kv_vec<T, N> kv_fix(kv_vec<T, N> r, int c, int n) {
  constexpr int W = N * sizeof(T) / 4;
  static_assert(W >= 1 && W * 4 == (int)(N * sizeof(T)), "whole words");
  typedef uint32_t Words __attribute__((ext_vector_type(W)));
  if (sizeof(T) == 4 && n < N) {
#pragma unroll
    for (int i = 0; i < N; i++) r[i] = c + i < n ? r[i] : (T)0;
  }
  Words w = __builtin_bit_cast(Words, r);
  if (n >= N && n % N) {  // the same for all lanes
    const int s = c > n - N && c < n ? (c - (n - N)) * (int)sizeof(T) : 0;  // bytes too early
    if (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < W; i++) w[i] = s & 2 ? __builtin_amdgcn_alignbit(i + 1 < W ? w[i + 1] : 0, w[i], 16) : w[i];
    }
#pragma unroll
    for (int d = 1; d < W; d *= 2)
#pragma unroll
      for (int i = 0; i < W; i++) w[i] = s & 4 * d ? (i + d < W ? w[i + d] : 0) : w[i];
  }
#pragma unroll
  for (int i = 0; i < W; i++) w[i] = c < n ? w[i] : 0;
  return __builtin_bit_cast(kv_vec<T, N>, w);
}
template <typename T, int N, bool V>
__device__ __forceinline__ kv_vec<T, N> kv_ld(const T *p, int c, int n) {
  if constexpr (V) {
    kv_vec<T, N> r;
#pragma unroll
    for (int i = 0; i < N; i++) r[i] = (T)0;
    if (c < n) r = *(const kv_vec<T, N> *)(p + c);
    return r;
  } else {
    return kv_fix<T, N>(kv_raw<T, N>(p, c, n), c, n);
  }
}

// the host's checks that every entry makes, and the device's descriptor
static inline int kv_check(const bnh_kvcache *c, int T, int B, int rows) {
  BNH_REQ(c && T > 0 && T <= (1 << 30) && B > 0 && rows > 0);
  BNH_REQ((c->f16 == 0 || c->f16 == 1) && c->Hk > 0 && c->Hk <= 65536 && (long long)B * c->Hk < (1LL << 24));
  BNH_REQ(c->dk > 0 && c->dk <= 256 && c->dv > 0 && c->dv <= 256);
  BNH_REQ(c->page >= 16 && c->page <= 1024 && (c->page & (c->page - 1)) == 0);
  BNH_REQ(c->pages > 0 && c->ldt > 0 && (long long)c->ldt * c->page < (1LL << 31) - 1024);
  return 0;
}
static inline bool kv_on(const void *q, size_t a) { return (uintptr_t)q % a == 0; }
static inline int kv_check_buffers(const bnh_kvcache *c, int T, int B, int rows, const int32_t *start, const int32_t *len) {
  BNH_REQ(c->k && c->v && c->table && c->past);
  BNH_REQ(c->k_ps >= (long long)c->Hk * c->page * c->dk && c->v_ps >= (long long)c->Hk * c->page * c->dv);
  BNH_REQ(!c->lo == !c->hi);
  BNH_REQ(start || (long long)T * B <= rows);
  const size_t es = c->f16 ? 2 : 4;
  BNH_REQ(kv_on(c->k, es) && kv_on(c->v, es) && kv_on(c->lo, es) && kv_on(c->hi, es));
  BNH_REQ(kv_on(c->table, 4) && kv_on(c->past, 4) && kv_on(start, 4) && kv_on(len, 4));
  return 0;
}
static inline KvDev kv_dev(const bnh_kvcache *c, int T, int rows, const int32_t *start, const int32_t *len) {
  return {c->k, c->v, c->k_ps, c->v_ps, c->lo, c->hi, c->table, c->past, start, len, c->pages,
          31 - __builtin_clz((unsigned)c->page), c->Hk, c->dk, c->dv, c->ldt, T, rows};
}
#endif
