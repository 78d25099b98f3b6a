// What the two forms of attention over a paged cache share (kern_kvattn.hip: few rows, and the join of split calls;
// kern_kvtile.hip: many rows).
#ifndef BNH_KVATTN_H
#define BNH_KVATTN_H
#include "bnh_kv.h"

struct KvaDev {
  const void *q;
  void *o;
  const int32_t *sel;
  int ldq, ldo, G, window, nsel;  // G: query heads that share one of keys
  float sc;                       // |scale| log2(e), above 0
  bool neg;                       // scale < 0: queries are taken negative
};

typedef float v4f __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ bool kv_finite(T x) { return x - x == (T)0; }

// A tile of rows: MR rows and query heads of one sequence and head of keys, heads innermost; with a selection, heads of one row
__device__ __forceinline__ void kva_row(const KvaDev &p, int tile, int m, int MR, int *t, int *h) {
  if (p.sel) {
    const int ht = (p.G + MR - 1) / MR;
    *t = tile / ht;
    *h = tile % ht * MR + m;
    if (*h >= p.G) *t = 0x7fffffff;  // nobody's
  } else {
    const long long x = (long long)tile * MR + m;
    *t = (int)(x / p.G);
    *h = (int)(x % p.G);
  }
}

// 0, or NaN where a value of x is not finite: one instruction for two of fp16
template <typename T, int N>
__device__ __forceinline__ void kv_mark(kv_vec<T, N> x, kv_vec<T, 2> &acc) {
  typedef kv_vec<T, 2> P;
#pragma unroll
  for (int i = 0; i < N; i += 2) acc = __builtin_elementwise_fma((P){x[i], x[i + 1]}, (P){(T)0, (T)0}, acc);
}

// How a call is cut
struct KvaPlan {
  bool tiled;
  int D, DK, MR, nrt, nsp;  // D: width of the sums' rows; MR: rows to a tile
  long long units;
};
// where the parts of a split lie in the workspace: each row's maximum and sum, then its products
static inline float2 *kva_ml(const KvaPlan &r, void *work) { return r.nsp > 1 ? (float2 *)work : nullptr; }
static inline float *kva_part(const KvaPlan &r, void *work) {
  return r.nsp > 1 ? (float *)((float2 *)work + r.units * r.nsp * r.MR) : nullptr;
}
// waves to a block of the tiled form (32 rows each)
static inline int kva_waves(int DK) { return DK == 256 ? 4 : 8; }
// the tiled form's launch (kern_kvtile.hip); v: everything is aligned to 16 bytes, widths too
int kva_tiles(const KvDev &c, const KvaDev &p, const KvaPlan &r, bool f16, bool v, void *work, hipStream_t s);
#endif
