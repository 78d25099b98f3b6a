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
template <typename T, int N, bool V>
__device__ __forceinline__ kv_vec<T, N> kv_ld(const T *p, int c, int n) {
  kv_vec<T, N> r;
  if (V) {
#pragma unroll
    for (int i = 0; i < N; i++) r[i] = (T)0;
    if (c < n) r = *(const kv_vec<T, N> *)(p + c);
  } else if (c + N <= n) {
    __builtin_memcpy(&r, p + c, N * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) r[i] = c + i < n ? p[c + i] : (T)0;
  }
  return r;
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
