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
  int want, least;                // parts of a split call in all, about, and tiles to one of them at least
  float sc;                       // |scale| log2(e), above 0 (times it, -inf is -inf), and what queries are taken times: the
  float sign;                     // scale's sign, 0 for a scale of 0
};

typedef float v4f __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ bool kv_finite(T x) { return x - x == (T)0; }

// A tile of rows: MR rows and query heads of one sequence and head of keys, heads innermost; with a selection, heads of one row
__device__ __forceinline__ void kva_row(const KvaDev &p, int tile, int m, int MR, int *t, int *h) {
  if (p.sel) {
    const unsigned ht = (unsigned)(p.G + MR - 1) / (unsigned)MR;
    *t = (int)((unsigned)tile / ht);
    *h = (int)((unsigned)tile % ht) * MR + m;
    if (*h >= p.G) *t = 0x7fffffff;  // nobody's
  } else {
    const unsigned x = (unsigned)tile * (unsigned)MR + (unsigned)m;  // below 2^31 + MR
    *t = (int)(x / (unsigned)p.G);
    *h = (int)(x - (unsigned)*t * (unsigned)p.G);
  }
}

// 0, or NaN where a value of x is not finite: one instruction for two of fp16
template <typename T, int N>
__device__ __forceinline__ void kv_mark(kv_vec<T, N> x, kv_vec<T, 2> &acc) {
  typedef kv_vec<T, 2> P;
#pragma unroll
  for (int i = 0; i < N; i += 2) acc = __builtin_elementwise_fma((P){x[i], x[i + 1]}, (P){(T)0, (T)0}, acc);
}

// The tokens that a tile of rows looks at, in tiles of TK of them
struct KvaSpan {
  int t0, t1;    // its rows: t0 past the sequence's last, none
  int j1;        // the last token
  int base, nt;  // the first tile of tokens, and how many; with a selection, tiles of the listed pages
};
__device__ __forceinline__ KvaSpan kva_span(const KvDev &c, const KvaDev &p, int tile, int MR, int TK, int n, int past) {
  KvaSpan r;
  int h;
  kva_row(p, tile, 0, MR, &r.t0, &h);
  if (p.sel) r.t1 = r.t0;
  else kva_row(p, tile, MR - 1, MR, &r.t1, &h);
  r.t1 = r.t1 < n ? r.t1 : n - 1;
  const long long cap = ((long long)c.ldt << c.sh) - 1;
  const int j0 = p.window && past + r.t0 >= p.window ? past + r.t0 - p.window + 1 : 0;
  r.j1 = past + r.t1 < cap ? past + r.t1 : (int)cap;
  r.base = j0 / TK;
  r.nt = p.sel ? (int)((((long long)p.nsel << (c.sh - 4)) + 1) >> 1) : r.j1 < j0 ? 0 : r.j1 / TK - r.base + 1;
  return r;
}

// A block's work: part sp of the tiles of tokens of a tile of rows, `per` of them, for one head of keys. How many parts there
// are is for the device to say, which knows the sequences' lengths: in a split call every block adds up the work of all sequences
// (few, or there would be no need for parts), and takes a part to be a `want`th of it, at least `least` tiles. A tile's parts
// are items one after another; they keep their sums at their place `item`
constexpr int kMostParts = 128;
struct KvaItem {
  int b, g, tile, sp, per, parts, item;
  int first, n, past;  // the sequence's, as kv_rows says
};
__device__ __forceinline__ bool kva_item(const KvDev &c, const KvaDev &p, int B, int nrt, bool split, int MR, int TK, unsigned item,
                                         KvaItem *r) {
  if (!split) {  // the last rows, which see most, of all heads and sequences first
    const unsigned sq = item / (unsigned)c.Hk, q = sq / (unsigned)B;
    if (q >= (unsigned)nrt) return false;
    *r = {(int)(sq - q * B), (int)(item - sq * c.Hk), nrt - 1 - (int)q, 0, 0x7fffffff, 1, (int)item, 0, 0, 0};
    r->n = kv_rows(c, r->b, &r->first, &r->past);
    return true;
  }
  const int lane = threadIdx.x & 63;
  const unsigned ht = (unsigned)(p.G + MR - 1) / (unsigned)MR;
  // a lane's sequence: its tiles of rows, and the most tiles of tokens that one of them looks at: the last does, but in a window,
  // where it has fewer rows than others
  const unsigned most = ((unsigned)p.window + (unsigned)(MR - 1) / (unsigned)p.G) / (unsigned)TK + 2;
  int first, past, n, tiles, nt;
  auto size = [&](int b) {
    const int i = b < B ? b : B - 1;
    const long long s = c.start ? c.start[i] : (long long)i * c.T;
    const int m = c.past[i], len = c.len ? c.len[i] : c.T;
    past = m > 0 ? m : 0;
    long long x = len < c.T ? len : c.T;
    if (s < 0 || s >= c.rows) x = 0;
    else x = x < c.rows - s ? x : c.rows - s;
    x = x < 0x7ffffff0 - past ? x : 0x7ffffff0 - past;
    n = b >= B || x < 0 ? 0 : (int)x;
    first = (int)s;
    tiles = p.sel ? (int)((unsigned)n * ht) : (int)(((unsigned)n * (unsigned)p.G + MR - 1) / (unsigned)MR);
    nt = n ? kva_span(c, p, tiles - 1, MR, TK, n, past).nt : 0;
    if (n && p.window && !p.sel) {
      const long long cap = (long long)c.ldt << c.sh;
      const unsigned all = ((unsigned)(cap < past + n ? cap : past + n) + TK - 1) / (unsigned)TK;
      nt = (int)(all < most ? all : most);
    }
  };
  float work = 0.f;
  for (int b0 = 0; b0 < B; b0 += 64) {
    size(b0 + lane);
    work += (float)tiles * (float)nt * (float)c.Hk;
  }
  for (int d = 1; d < 64 && d < B; d *= 2) work += __shfl_xor(work, d);
  if (B < 64) work = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(work)));
  const int each = (int)__builtin_ceilf(work / (float)p.want), floor = each > p.least ? each : p.least;
  unsigned before = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    if (B > 64) size(b0 + lane);
    const unsigned few = (unsigned)(nt + kMostParts - 1) / kMostParts, per = few > (unsigned)floor ? few : floor;
    const unsigned parts = (unsigned)nt > per ? ((unsigned)nt + per - 1) / per : 1, mine = (unsigned)(c.Hk * tiles) * parts;
    unsigned sum = mine;
    for (int d = 1; d < 64 && d < B; d *= 2) {
      const unsigned o = __shfl_up(sum, d);
      sum += lane >= d ? o : 0;
    }
    const unsigned long long in = __ballot(before + sum > item);
    if (in) {
      const int l = __builtin_ctzll(in);
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
      const unsigned rest = item - (before + of(sum) - of(mine)), np = of(parts), x = rest / np, y = x / (unsigned)c.Hk;
      *r = {b0 + l, (int)(x - y * c.Hk), of(tiles) - 1 - (int)y, (int)(rest - x * np), (int)((of(nt) + np - 1) / np), (int)np,
            (int)item, of(first), of(n), of(past)};
      for (int *v : {&r->b, &r->g, &r->tile, &r->sp, &r->per, &r->parts}) *v = __builtin_amdgcn_readfirstlane(*v);
      return true;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// How a call is cut
struct KvaPlan {
  bool tiled;
  int D, DK, MR, TK, nrt;  // D: width of the sums' rows; MR, TK: rows and tokens to a tile
  bool split;
  int want, least;         // parts in all, about, and tiles of tokens to one at least
  long long units, items;  // tiles of all heads and sequences; blocks: a part is a `want`th of all the work, or a tile's last
};
// what lies in the workspace of a split call: each tile's parts and the first of them, then of each part each row's maximum and
// sum, and its products
static inline int2 *kva_counts(const KvaPlan &r, void *work) { return r.split ? (int2 *)work : nullptr; }
static inline float2 *kva_ml(const KvaPlan &r, void *work) {
  return r.split ? (float2 *)((char *)work + bnh_round_up(8 * r.units, 16)) : nullptr;
}
static inline float *kva_part(const KvaPlan &r, void *work) {
  return r.split ? (float *)(kva_ml(r, work) + r.items * r.MR) : nullptr;
}
static inline size_t kva_bytes(const KvaPlan &r) {
  return r.split ? (size_t)(bnh_round_up(8 * r.units, 16) + r.items * r.MR * (4 * r.D + 8)) : 0;
}
// tokens to a tile of the tiled form, and waves to a block of it (32 rows each)
constexpr int kva_tokens(bool f16, int DK) { return f16 && DK < 256 ? 64 : 32; }
constexpr int kva_waves(bool f16, int DK) { return f16 && DK < 256 ? 8 : 4; }
// the tiled form's launch (kern_kvtile.hip); w: what everything is aligned to, widths too, in bytes: 16, 4 or 2
int kva_tiles(const KvDev &c, const KvaDev &p, const KvaPlan &r, bool f16, int w, void *work, hipStream_t s);
#endif
