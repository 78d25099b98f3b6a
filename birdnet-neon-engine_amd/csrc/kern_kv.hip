// New rows into a paged cache with their rotation (bnh_kv_append), and the pages that rows look at by the pages' bounds
// (bnh_kv_select).
#include <float.h>

#include "bnh_kv.h"

namespace {

// ---------------------------------------------------------------------------------------------- append
// Bound by HBM: q, k and v are read once and written once. A block owns the new rows of one page for one head of keys, with the
// query heads that read it, so that the page's bounds need no atomics: its threads are `nu` units of a head (VEC values,
// with their partners VEC more) side by side, times as many rows as fit 256. 24 archives of 720 rows, 12 heads of 128, 162 MB: 50 us,
// 3.2 TB/s, of which the angles are 6 (36 us for the same buffers again, which the last-level cache holds); 8 of up to 500 rows of odd
// widths in fp32, value by value: 21 us, 2.5 TB/s; live rows 6 to 7, a launch and two loads that wait for each other.
struct AppDev {
  const void *k, *v, *q;
  void *qr;
  const float *freq;
  const int32_t *pos;
  int ldk, ldv, ldq, ldr, G, rd, pairs;
};

// cos and sin of pos freq: the angle in quarters of a turn, reduced to half a one about the nearest, where the series of sin and cos
// up to x^9 and x^10 are within 2e-9. The angle (55 bits) and 2 / pi are in two parts each and whole turns go before the parts
// are joined, so that a far position's angle is as exact as that of 0. In one part of 53 bits it is off by 2^-53 of itself at each of
// three steps, five units of what 32 bits leave at position 2^31 (24 archives of 720 rows, 12 heads: 49.4 us so, 50.3 now)
__device__ __forceinline__ void turn(int pos, float freq, float *cs, float *sn) {
  constexpr double Q1 = 0x1.45f306dc9c883p-1, Q2 = -0x1.6b01ec5417056p-55;  // 2 / pi and what is left of it
  const double a1 = (double)pos * (double)freq, a2 = __builtin_fma((double)pos, (double)freq, -a1);
  const double t1 = a1 * Q1, t2 = __builtin_fma(a1, Q1, -t1) + __builtin_fma(a1, Q2, a2 * Q1);
  const double t = __builtin_fma(-4.0, __builtin_rint(0.25 * t1), t1) + t2, n = __builtin_rint(t), r = t - n;
  const int k = (int)n & 3;
  const float x = (float)(r * 1.57079632679489661923), y = x * x;
  float s = __builtin_fmaf(y, 2.7557319e-6f, -1.9841270e-4f);
  s = __builtin_fmaf(y, s, 8.3333333e-3f);
  s = __builtin_fmaf(y, s, -1.6666667e-1f);
  s = __builtin_fmaf(x * y, s, x);
  float c = __builtin_fmaf(y, -2.7557319e-7f, 2.4801587e-5f);
  c = __builtin_fmaf(y, c, -1.3888889e-3f);
  c = __builtin_fmaf(y, c, 4.1666667e-2f);
  c = __builtin_fmaf(y, c, -0.5f);
  c = __builtin_fmaf(y, c, 1.f);
  const float a = k & 1 ? s : c, b = k & 1 ? c : s;
  *cs = k == 1 || k == 2 ? -a : a;
  *sn = k >= 2 ? -b : b;
}
// the smaller and the larger of two, value by value, NaN where one is
template <typename W>
__device__ __forceinline__ W low(W a, W b) { return __builtin_elementwise_minimum(a, b); }
template <typename W>
__device__ __forceinline__ W high(W a, W b) { return __builtin_elementwise_maximum(a, b); }

// A unit: VEC values at `a` and VEC more at `b` (pairs 0: the partners; pairs 1 and values past rd: the next ones)
template <typename T, int VEC>
__global__ __launch_bounds__(256) void k_kv_append(KvDev c, AppDev p, int npt, int nu, int b0, int pt0) {
  typedef T W __attribute__((ext_vector_type(VEC), aligned(sizeof(T) * VEC)));
  __shared__ __attribute__((aligned(16))) T s_lo[512 * VEC], s_hi[512 * VEC];
  const unsigned sq = blockIdx.x / (unsigned)c.Hk;  // sequences and pages of a launch from (b0, pt0) on
  const int g = (int)(blockIdx.x - sq * c.Hk);
  const unsigned b1 = sq / (unsigned)npt, pt1 = sq - b1 * npt;
  const int b = b0 + (int)b1, pt = pt0 + (int)pt1;
  int first, past;
  const int n = kv_rows(c, b, &first, &past);
  const int pi = (past >> c.sh) + pt;                   // the sequence's page
  const long long p0 = (long long)pi << c.sh, p1 = p0 + (1 << c.sh);
  if (n == 0 || (pt && p0 - past >= n)) return;
  const int t0 = pt ? (int)(p0 - past) : 0, t1 = n < p1 - past ? n : (int)(p1 - past);  // its rows
  const int page = kv_page(c, b, pi);
  const int off = (int)(past + t0 - p0);             // the first one's place in the page
  const int tid = threadIdx.x, u = tid % nu, rl = tid / nu, RL = 256 / nu;
  // the unit's values of a head
  const int half = p.rd / 2, nr = p.pairs ? 0 : (half + VEC - 1) / VEC;  // units of partners
  const bool apart = u < nr;                                             // VEC values and their partners
  const int rest = p.pairs ? 0 : p.rd;                                   // then pairs of VEC side by side from here
  const int a = apart ? u * VEC : rest + 2 * (u - nr) * VEC, bb = apart ? a + half : a + VEC;
  const int na = apart ? half : c.dk, nb = apart ? p.rd : c.dk;          // where the values end
  W lo[2], hi[2];
#pragma unroll
  for (int i = 0; i < VEC; i++) lo[0][i] = lo[1][i] = (T)INFINITY, hi[0][i] = hi[1][i] = (T)-INFINITY;
  T *kc = (T *)c.k + (page < 0 ? 0 : page * c.k_ps + ((long long)g << c.sh) * c.dk);
  if (rl < RL) {
    for (int t = t0 + rl; t < t1; t += RL) {
      const long long r = (long long)first + t;
      float cs[VEC], sn[VEC];
      const int pos = p.pos ? p.pos[r] : past + t;
      // pairs: a unit of 2 VEC values has VEC pairs, value 2 i of the two vectors with value 2 i + 1
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        const int e = apart ? a + i : a / 2 + i;
        cs[i] = 1.f, sn[i] = 0.f;
        if (p.rd && (apart || p.pairs) && e < half) turn(pos, p.freq[e], &cs[i], &sn[i]);
      }
      auto rotate = [&](const T *src, T *dst, bool bound) {
        W x[2];
        if (VEC > 1) {
          x[0] = *(const W *)(src + a), x[1] = *(const W *)(src + bb);
        } else {
          x[0][0] = a < na ? src[a] : (T)0, x[1][0] = bb < nb ? src[bb] : (T)0;
        }
        if (apart) {
#pragma unroll
          for (int i = 0; i < VEC; i++) {
            const float y = (float)x[0][i], z = (float)x[1][i];
            x[0][i] = (T)__builtin_fmaf(y, cs[i], -(z * sn[i]));
            x[1][i] = (T)__builtin_fmaf(y, sn[i], z * cs[i]);
          }
        } else if (p.pairs && a < p.rd) {
          T w[2 * VEC];
#pragma unroll
          for (int i = 0; i < VEC; i++) w[i] = x[0][i], w[VEC + i] = x[1][i];
#pragma unroll
          for (int i = 0; i < VEC; i++) {
            if (a + 2 * i >= p.rd) continue;
            const float y = (float)w[2 * i], z = (float)w[2 * i + 1];
            w[2 * i] = (T)__builtin_fmaf(y, cs[i], -(z * sn[i]));
            w[2 * i + 1] = (T)__builtin_fmaf(y, sn[i], z * cs[i]);
          }
#pragma unroll
          for (int i = 0; i < VEC; i++) x[0][i] = w[i], x[1][i] = w[VEC + i];
        }
        if (VEC > 1) {
          *(W *)(dst + a) = x[0], *(W *)(dst + bb) = x[1];
        } else {
          if (a < na) dst[a] = x[0][0];
          if (bb < nb) dst[bb] = x[1][0];
        }
        if (bound) {
#pragma unroll
          for (int j = 0; j < 2; j++) lo[j] = low(lo[j], x[j]), hi[j] = high(hi[j], x[j]);
        }
      };
      if (page >= 0) rotate((const T *)p.k + r * p.ldk + g * c.dk, kc + (long long)(off + t - t0) * c.dk, c.lo != nullptr);
      if (p.q)
        for (int h = g * p.G; h < (g + 1) * p.G; h++)
          rotate((const T *)p.q + r * p.ldq + (long long)h * c.dk, (T *)p.qr + r * p.ldr + (long long)h * c.dk, false);
    }
  }
  if (page < 0) return;
  // values as they are, 16 bytes at a time, the last ones of a row wherever they begin
  T *vc = (T *)c.v + page * c.v_ps + (((long long)g << c.sh) + off) * c.dv;
  constexpr int VE = 16 / sizeof(T);
  if (c.dv < VE) {
    for (int i = tid; i < (t1 - t0) * c.dv; i += 256) {
      const int t = i / c.dv, e = i - t * c.dv;
      vc[(long long)t * c.dv + e] = ((const T *)p.v)[((long long)first + t0 + t) * p.ldv + g * c.dv + e];
    }
  } else {
    const int nv = (c.dv + VE - 1) / VE, step = 256 / nv, e0 = tid % nv * VE, e = VEC == VE || e0 + VE <= c.dv ? e0 : c.dv - VE;
    for (int t = tid / nv; t < t1 - t0 && tid < step * nv; t += step) {
      const T *x = (const T *)p.v + ((long long)first + t0 + t) * p.ldv + g * c.dv + e;
      if constexpr (VEC == VE) {
        *(W *)(vc + (long long)t * c.dv + e) = *(const W *)x;
      } else {
        uint4 y;
        __builtin_memcpy(&y, x, 16);
        __builtin_memcpy(vc + (long long)t * c.dv + e, &y, 16);
      }
    }
  }
  if (!c.lo) return;
  if (rl < RL) {
#pragma unroll
    for (int i = 0; i < VEC; i++) {  // [rl][value]; values past the unit's end are nobody's
      if (a + i < na) s_lo[rl * c.dk + a + i] = lo[0][i], s_hi[rl * c.dk + a + i] = hi[0][i];
      if (bb + i < nb) s_lo[rl * c.dk + bb + i] = lo[1][i], s_hi[rl * c.dk + bb + i] = hi[1][i];
    }
  }
  __syncthreads();
  // columns (two of fp16 where rows of LDS allow it), over groups of the rows and then over the groups
  constexpr int PK = VEC > 1 && sizeof(T) == 2 ? 2 : 1;
  typedef T P __attribute__((ext_vector_type(PK)));
  const int cols = c.dk / PK, groups = 256 / cols, col = tid % cols, grp = tid / cols;
  const int used = RL < t1 - t0 ? RL : t1 - t0;
  P *pl = (P *)s_lo + col, *ph = (P *)s_hi + col;
  if (grp < groups && grp < used) {
    P l = pl[grp * cols], h = ph[grp * cols];
    for (int i = grp + groups; i < used; i += groups) l = low(l, pl[i * cols]), h = high(h, ph[i * cols]);
    pl[grp * cols] = l, ph[grp * cols] = h;
  }
  __syncthreads();
  if (grp == 0) {
    const long long at = ((long long)page * c.Hk + g) * c.dk + PK * col;
    P l = pl[0], h = ph[0];
    for (int i = 1; i < groups && i < used; i++) l = low(l, pl[i * cols]), h = high(h, ph[i * cols]);
    P *gl = (P *)((T *)c.lo + at), *gh = (P *)((T *)c.hi + at);
    if (off) l = low(l, *gl), h = high(h, *gh);
    *gl = l, *gh = h;
  }
}

template <typename T, int VEC>
int append_run(const KvDev &c, const AppDev &p, int B, hipStream_t s) {
  const int npt = (int)(((long long)c.T + (1 << c.sh) - 2) >> c.sh) + 1;  // pages that T rows can touch
  const int half = p.rd / 2, nr = p.pairs ? 0 : (half + VEC - 1) / VEC, left = c.dk - (p.pairs ? 0 : p.rd);
  const int nu = nr + (left + 2 * VEC - 1) / (2 * VEC);
  const long long most = bnh_most_blocks(256);  // Hk <= 2^16
  const int np = most / c.Hk < npt ? (int)(most / c.Hk) : npt, nb = most / c.Hk / np < B ? (int)(most / c.Hk / np) : B;
  for (int b0 = 0; b0 < B; b0 += nb)
    for (int p0 = 0; p0 < npt; p0 += np) {
      const int n = npt - p0 < np ? npt - p0 : np;
      hipLaunchKernelGGL((k_kv_append<T, VEC>), dim3((unsigned)((long long)(B - b0 < nb ? B - b0 : nb) * n * c.Hk)), dim3(256), 0, s,
                         c, p, n, nu, b0, p0);
      BNH_HIP(hipGetLastError());
    }
  return 0;
}

// ---------------------------------------------------------------------------------------------- select
// A score's order as a whole number: larger for larger scores, 0 for a page that is not to be had, above that of +infinity for one
// that is always taken
typedef unsigned long long u64;
constexpr u64 ALWAYS = ~0ull;
__device__ __forceinline__ u64 order_of(double x) {
  if (x != x) x = -INFINITY;
  const u64 b = (u64)__double_as_longlong(x == 0 ? 0.0 : x);  // -0 is 0
  return b >> 63 ? ~b : b | 1ull << 63;
}
struct SelDev {
  const void *q;
  int32_t *sel;
  int ldq, H, G, window, nsel, first, last;
};
// the row's place: its sequence's pages [lo, hi) have a token that it may see. Row i of a launch is row t0 + i of sequence b0, or
// of those after it
__device__ __forceinline__ bool sel_row(const KvDev &c, int window, int b0, int t0, unsigned i, int *b, long long *row, int *lo, int *hi) {
  const unsigned x = (unsigned)t0 + i, q = x / (unsigned)c.T;
  *b = b0 + (int)q;
  const int t = (int)(x - q * (unsigned)c.T);
  int first, past;
  const int n = kv_rows(c, *b, &first, &past);
  if (t >= n) return false;
  *row = (long long)first + t;
  const int at = past + t;
  *lo = window && at >= window ? (at - window + 1) >> c.sh : 0;
  *hi = (at >> c.sh) + 1;
  return true;
}

// The scores of PPB pages for one row and head of keys: 16 lanes a page, 8 values each a step. Bound by reading the bounds
// (4 dk bytes a page and head in fp16). The products are exact in 64 bits; a sum of n of them is off by n 2^-53 of its terms' sizes
// at most, and always in the same order, which decides between scores that are closer. One row over 1,890 pages of 4 heads of 128:
// 9.4 us; 16 rows over up to 810: 14.2; 144 rows of 2 heads of 72 over up to 188, fp32: 11.4.
constexpr int PPB = 64;
template <typename T, bool V>
__global__ __launch_bounds__(256) void k_kv_score(KvDev c, SelDev p, int npb, int b0, int t0, u64 *key) {
  __shared__ __attribute__((aligned(16))) float s_q[16 * 256];  // up to 16 query heads at a time
  const unsigned x = blockIdx.x / (unsigned)npb, i = x / (unsigned)c.Hk;
  const int pb = (int)(blockIdx.x - x * npb), g = (int)(x - i * c.Hk);
  int b, lo, hi;
  long long row;
  if (!sel_row(c, p.window, b0, t0, i, &b, &row, &lo, &hi)) return;
  const int cur = hi - 1, end = hi < c.ldt ? hi : c.ldt;
  const int tid = threadIdx.x, l = tid & 15, team = tid >> 4;
  if (pb * PPB >= end) return;
  u64 *out = key + ((long long)i * c.Hk + g) * c.ldt;
  const int kd = (c.dk + 127) / 128 * 128;
  double acc[PPB / 16];
#pragma unroll
  for (int j = 0; j < PPB / 16; j++) acc[j] = 0;
  for (int h0 = 0; h0 < p.G; h0 += 16) {
    const int nh = p.G - h0 < 16 ? p.G - h0 : 16;
    if (h0) __syncthreads();
    for (int y = tid; y < nh * kd; y += 256) {
      const int h = y / kd, d = y - h * kd;
      s_q[y] = d < c.dk ? (float)((const T *)p.q)[row * p.ldq + (long long)(g * p.G + h0 + h) * c.dk + d] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PPB / 16; j++) {
      const int pi = pb * PPB + 16 * j + team;
      const int page = pi >= lo && pi < end ? kv_page(c, b, pi) : -1;
      if (page < 0) continue;
      const T *pl = (const T *)c.lo + ((long long)page * c.Hk + g) * c.dk;
      const T *ph = (const T *)c.hi + ((long long)page * c.Hk + g) * c.dk;
      for (int d0 = 0; d0 < kd; d0 += 128) {
        const int d = d0 + 8 * l;
        const kv_vec<T, 8> xl = kv_ld<T, 8, V>(pl, d, c.dk), xh = kv_ld<T, 8, V>(ph, d, c.dk);
        for (int h = 0; h < nh; h++) {
          const float4 q0 = *(const float4 *)(s_q + h * kd + d), q1 = *(const float4 *)(s_q + h * kd + d + 4);
          const float q[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
#pragma unroll
          for (int e = 0; e < 8; e++)
            acc[j] = __builtin_fma((double)q[e], (double)(float)(q[e] >= 0.f ? xh[e] : xl[e]), acc[j]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < PPB / 16; j++) {
    const int pi = pb * PPB + 16 * j + team;
    if (pi >= end) continue;
    double x = acc[j];
#pragma unroll
    for (int m = 1; m < 16; m *= 2) x += __shfl_xor(x, m);
    const bool there = pi >= lo && kv_page(c, b, pi) >= 0;
    if (l == 0) out[pi] = !there ? 0 : pi < p.first || pi > cur - p.last ? ALWAYS : order_of(x);
  }
}

// The nsel largest of a row's keys, the lower pages first where the last of them are equal, in ascending order. The bits that all
// keys agree on are passed over, then digits of 8 bits are counted until the last one needed is known; pages that are always
// taken (no more than nsel) stand aside, or they would stretch the range to all 64 bits. 512 threads hold 8 keys each, in
// order; more than 4,096 are read again for each digit. Bound by the steps, of which each waits for the one before: 1,890
// pages of a row 7.3 us, 14.8 with digits from the top (the first are the same for all) and keys read again for each.
constexpr int KEYS = 8, NTP = 512;
__global__ __launch_bounds__(NTP) void k_kv_pick(KvDev c, SelDev p, int b0, int t0, const u64 *key) {
  __shared__ int s_n[256], s_w[NTP / 64], s_t[NTP / 64], s_b[2];
  __shared__ unsigned s_lo[NTP / 64], s_hi[NTP / 64];
  const unsigned i = blockIdx.x / (unsigned)c.Hk;
  const int g = (int)(blockIdx.x - i * c.Hk);
  int b, lo, hi;
  long long row;
  if (!sel_row(c, p.window, b0, t0, i, &b, &row, &lo, &hi)) return;
  const int end = hi < c.ldt ? hi : c.ldt;
  const u64 *k = key + ((long long)i * c.Hk + g) * c.ldt;
  int32_t *out = p.sel + (row * c.Hk + g) * p.nsel;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (end - lo <= 128) {  // a key to a thread, which counts those that come before it
    __shared__ __attribute__((aligned(16))) u64 s_k[NTP];
    const int n = end - lo;
    const u64 mine = tid < n ? k[lo + tid] : 0;
    s_k[tid] = mine;
    __syncthreads();
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; j += 2) {
      const ulonglong2 x = *(const ulonglong2 *)(s_k + j);
      rank += (x.x > mine) + (x.y > mine) + (x.x == mine && j < tid) + (x.y == mine && j + 1 < tid);
    }
    const bool take = mine && rank < p.nsel;
    const u64 in = __ballot(take);
    if (lane == 0) s_w[wave] = __popcll(in);
    __syncthreads();
    int at = __popcll(in & ((1ull << lane) - 1)), done = 0;
#pragma unroll
    for (int w = 0; w < NTP / 64; w++) at += w < wave ? s_w[w] : 0, done += s_w[w];
    if (take) out[at] = lo + tid;
    for (int x = done + tid; x < p.nsel; x += NTP) out[x] = -1;
    return;
  }
  const bool once = end - lo <= KEYS * NTP;
  const int each = once ? (end - lo + NTP - 1) / NTP : KEYS;  // keys to a thread
  u64 y[KEYS];
  auto fetch = [&](int x0) {  // the thread's keys of those from x0 on; 0: none
#pragma unroll
    for (int e = 0; e < KEYS; e++) {
      const int x = x0 + tid * each + e;
      y[e] = e < each && x < end ? k[x] : 0;
    }
  };
  // the sum of a number over the block, and how much of it is in threads before this one
  auto before = [&](int n, int *total, int *s) {
    int sum = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_up(sum, d);
      sum += lane >= d ? o : 0;
    }
    if (lane == 63) s[wave] = sum;
    __syncthreads();
    int at = sum - n;
    *total = 0;
#pragma unroll
    for (int w = 0; w < NTP / 64; w++) at += w < wave ? s[w] : 0, *total += s[w];
    return at;
  };
  // the range of the upper words of the keys that are not always taken, and how many are
  unsigned least = ~0u, most = 0;
  int count = 0;  // of all, and 2^16 times of those that are always taken, of 4,096 keys at a time
  int always = 0, any = 0;
  for (int x0 = lo; x0 < end; x0 += KEYS * NTP) {
    fetch(x0);
    count = 0;
#pragma unroll
    for (int e = 0; e < KEYS; e++) {
      const unsigned w = (unsigned)(y[e] >> 32);
      count += (y[e] != 0) + ((y[e] == ALWAYS) << 16);
      if (y[e] && y[e] != ALWAYS) least = least < w ? least : w, most = most > w ? most : w;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) count += __shfl_xor(count, d);
    any += count & 0xffff, always += count >> 16;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const unsigned l = __shfl_xor(least, d), m = __shfl_xor(most, d);
    least = least < l ? least : l, most = most > m ? most : m;
  }
  if (lane == 0) s_lo[wave] = least, s_hi[wave] = most, s_w[wave] = always, s_t[wave] = any;
  __syncthreads();
  always = any = 0;
#pragma unroll
  for (int w = 0; w < NTP / 64; w++) {
    least = least < s_lo[w] ? least : s_lo[w], most = most > s_hi[w] ? most : s_hi[w];
    always += s_w[w], any += s_t[w];
  }
  any -= always;
  // taken: those that always are, those above `cut` in the bits of `mask`, and the first `need` that agree with it there
  u64 cut = 0, mask = ~0ull;
  int need = p.nsel - always;
  if (need <= 0) {
    cut = ALWAYS - 1;  // none of the others
  } else if (any > need) {
    int bits = least == most ? 32 : 64 - __builtin_clz(least ^ most);  // that are not the same for all
    mask = bits < 64 ? ~0ull << bits : 0;
    cut = (u64)most << 32 & mask;
    bool all = false;
    while (!all) {
      const int shift = bits > 8 ? bits - 8 : 0;
      if (tid < 256) s_n[tid] = 0;
      __syncthreads();
      for (int x0 = lo; x0 < end; x0 += KEYS * NTP) {
        if (!once) fetch(x0);
#pragma unroll
        for (int e = 0; e < KEYS; e++)
          if (y[e] && y[e] != ALWAYS && (y[e] & mask) == cut) atomicAdd(&s_n[(y[e] >> shift) & ((1u << (bits - shift)) - 1)], 1);
      }
      __syncthreads();
      // the digit of the last one needed: above it fewer than need, with it need or more
      if (wave == 0) {
        int n[4], sum = 0;  // digits 255 - 4 lane .. downwards
#pragma unroll
        for (int e = 0; e < 4; e++) n[e] = s_n[255 - 4 * lane - e], sum += n[e];
        int up = sum;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
          const int o = __shfl_up(up, d);
          up += lane >= d ? o : 0;
        }
        up -= sum;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (up < need && up + n[e] >= need) s_b[0] = 255 - 4 * lane - e, s_b[1] = up;
          up += n[e];
        }
      }
      __syncthreads();
      cut |= (u64)s_b[0] << shift;
      mask |= shift ? ~0ull << shift : ~0ull;
      need -= s_b[1];
      all = shift == 0 || s_n[s_b[0]] == need;
      bits = shift;
      __syncthreads();
    }
  }
  auto above = [&](u64 x) { return x == ALWAYS || (x & mask) > cut; };
  auto agrees = [&](u64 x) { return x && x != ALWAYS && (x & mask) == cut; };
  int done = 0, ties = 0;
  for (int x0 = lo; x0 < end; x0 += KEYS * NTP) {
    if (!once) fetch(x0);
    int n = 0, total;  // those above, and 2^16 times those that agree
#pragma unroll
    for (int e = 0; e < KEYS; e++)
      n += above(y[e]) + (agrees(y[e]) << 16);
    const int in = before(n, &total, s_n);
    int rank = ties + (in >> 16), at = done + (in & 0xffff) + ((rank < need ? rank : need) - (ties < need ? ties : need));
#pragma unroll
    for (int e = 0; e < KEYS; e++) {
      const bool tie = agrees(y[e]);
      if (above(y[e]) || (tie && rank < need)) out[at++] = x0 + tid * each + e;
      rank += tie;
    }
    const int now = ties + (total >> 16);
    done += (total & 0xffff) + ((now < need ? now : need) - (ties < need ? ties : need));
    ties = now;
    if (!once) __syncthreads();
  }
  for (int x = done + tid; x < p.nsel; x += NTP) out[x] = -1;
}

// rows of a launch: the scores of 64 MB at most, or of one row
long long select_rows(const bnh_kvcache *c, int T, int B) {
  const long long per = 8LL * c->Hk * c->ldt, n = (64LL << 20) / per, all = (long long)T * B;
  return n < 1 ? 1 : n < all ? n : all;
}

int select_check(const bnh_kvcache *c, const bnh_kvattn *p, int T, int B, int rows) {
  if (kv_check(c, T, B, rows)) return -1;
  BNH_REQ(p && p->H > 0 && p->H % c->Hk == 0 && p->H <= 65536 && p->nsel > 0 && p->nsel <= (1 << 20) && p->window >= 0);
  BNH_REQ((long long)rows * c->Hk < (1LL << 31));
  return 0;
}

}  // namespace

extern "C" {

int bnh_kv_append(const bnh_kvcache *c, const bnh_rotary *r, const void *k, int ldk, const void *v, int ldv, const void *q,
                  int ldq, void *qr, int ldr, int H, int T, int B, int rows, const int32_t *start, const int32_t *len,
                  void *stream) {
  if (kv_check(c, T, B, rows) || kv_check_buffers(c, T, B, rows, start, len)) return -1;
  BNH_REQ(k && v && ldk >= c->Hk * c->dk && ldv >= c->Hk * c->dv);
  BNH_REQ(!q == !qr);
  BNH_REQ(!q || (H > 0 && H <= 65536 && H % c->Hk == 0 && ldq >= H * c->dk && ldr >= H * c->dk && (q != qr || ldq == ldr)));
  BNH_REQ(!r || (r->rd >= 0 && r->rd <= c->dk && r->rd % 2 == 0 && (r->pairs == 0 || r->pairs == 1) && (!r->rd || r->freq)));
  const size_t es = c->f16 ? 2 : 4;
  BNH_REQ(kv_on(k, es) && kv_on(v, es) && kv_on(q, es) && kv_on(qr, es));
  BNH_REQ(!r || (kv_on(r->freq, 4) && kv_on(r->pos, 4)));
  const KvDev d = kv_dev(c, T, rows, start, len);
  const int rd = r ? r->rd : 0, pairs = r ? r->pairs : 0, ve = 16 / (int)es;
  const AppDev p = {k, v, q, qr, r ? r->freq : nullptr, r ? r->pos : nullptr, ldk, ldv, ldq, ldr, q ? H / c->Hk : 0, rd, pairs};
  // values of q and k at a time: as many as widths, strides and addresses allow (24 archives of 720 rows, 12 heads, fp16, us: 128
  // by eights 50, one by one 86; 120 by fours 59 and 88; 108 by twos 57 and 86; fp32, 108 by twos 83 and 129)
  auto fits = [&](int n) {
    bool x = c->dk % (2 * n) == 0 && rd % (2 * n) == 0 && c->k_ps % n == 0 && ldk % n == 0;
    x = x && (!q || (ldq % n == 0 && ldr % n == 0)) && kv_on(c->lo, 4) && kv_on(c->hi, 4);
    for (const void *y : {(const void *)c->k, k, q, (const void *)qr}) x = x && kv_on(y, n * es);
    return x;
  };
  const bool vec = fits(ve) && c->dv % ve == 0 && c->v_ps % ve == 0 && ldv % ve == 0 && kv_on(c->v, 16) && kv_on(v, 16);
  hipStream_t s = bnh_stream(stream);
  if (c->f16) {
    if (vec) return append_run<h16, 8>(d, p, B, s);
    return fits(4) ? append_run<h16, 4>(d, p, B, s) : fits(2) ? append_run<h16, 2>(d, p, B, s) : append_run<h16, 1>(d, p, B, s);
  }
  return vec ? append_run<float, 4>(d, p, B, s) : fits(2) ? append_run<float, 2>(d, p, B, s) : append_run<float, 1>(d, p, B, s);
}

size_t bnh_kv_select_work_bytes(const bnh_kvcache *c, const bnh_kvattn *p, int T, int B, int rows) {
  if (select_check(c, p, T, B, rows)) return 0;
  return (size_t)(select_rows(c, T, B) * c->Hk * c->ldt * 8);
}

int bnh_kv_select(const bnh_kvcache *c, const bnh_kvattn *p, int first, int last, int T, int B, int rows,
                  const int32_t *start, const int32_t *len, void *work, size_t work_bytes, void *stream) {
  if (select_check(c, p, T, B, rows) || kv_check_buffers(c, T, B, rows, start, len)) return -1;
  BNH_REQ(c->lo && p->q && p->sel && p->ldq >= p->H * c->dk && first >= 0 && last >= 0 && first <= p->nsel - last);
  const size_t es = c->f16 ? 2 : 4;
  BNH_REQ(kv_on(p->q, es) && kv_on(p->sel, 4));
  const long long per = select_rows(c, T, B), all = (long long)T * B;
  BNH_REQ(work && kv_on(work, 16) && work_bytes >= (size_t)(per * c->Hk * c->ldt * 8));
  const KvDev d = kv_dev(c, T, rows, start, len);
  const SelDev e = {p->q, p->sel, p->ldq, p->H, p->H / c->Hk, p->window, p->nsel, first, last};
  const bool v = c->dk % 8 == 0 && kv_on(c->lo, 16) && kv_on(c->hi, 16);
  const int npb = (int)bnh_ceil_div(c->ldt, PPB);
  // rows of a launch also by its blocks, of the scores and of the choice
  long long most = bnh_most_blocks(256) / ((long long)npb * c->Hk);
  BNH_REQ(most > 0);
  if (most > bnh_most_blocks(NTP) / c->Hk) most = bnh_most_blocks(NTP) / c->Hk;
  if (most > per) most = per;
  hipStream_t s = bnh_stream(stream);
  for (long long r0 = 0; r0 < all; r0 += most) {
    const long long n = all - r0 < most ? all - r0 : most;
    const int b0 = (int)(r0 / T), t0 = (int)(r0 % T);
    const dim3 grid((unsigned)(n * npb * c->Hk)), block(256);
    u64 *key = (u64 *)work;
    if (c->f16) {
      if (v) hipLaunchKernelGGL((k_kv_score<h16, true>), grid, block, 0, s, d, e, npb, b0, t0, key);
      else hipLaunchKernelGGL((k_kv_score<h16, false>), grid, block, 0, s, d, e, npb, b0, t0, key);
    } else {
      if (v) hipLaunchKernelGGL((k_kv_score<float, true>), grid, block, 0, s, d, e, npb, b0, t0, key);
      else hipLaunchKernelGGL((k_kv_score<float, false>), grid, block, 0, s, d, e, npb, b0, t0, key);
    }
    BNH_HIP(hipGetLastError());
    hipLaunchKernelGGL(k_kv_pick, dim3((unsigned)(n * c->Hk)), dim3(NTP), 0, s, d, e, b0, t0, key);
    BNH_HIP(hipGetLastError());
  }
  return 0;
}

}  // extern "C"
