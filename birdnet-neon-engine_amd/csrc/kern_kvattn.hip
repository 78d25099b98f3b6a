// Attention of new rows over a paged cache of keys and values (bnh_kv_attn): per row and head, over the tokens j that the row
// sees,
//   s_j = scale q . k_j,  o = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m},  m = max_j s_j,
// in one pass over the keys with the running m and sum, both in fp32 and base 2.
#include <math.h>

#include "bnh_kvattn.h"

namespace {

// 32 steps of a product: 8 of row (or column) lane & 15 in a lane, the same 8 of both operands
__device__ __forceinline__ v4f mma(kv_vec<h16, 8> a, kv_vec<h16, 8> b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mma(kv_vec<float, 8> a, kv_vec<float, 8> b, v4f c) {
#pragma unroll
  for (int e = 0; e < 8; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}
// The streaming form, for few rows and for rows with a selection: bound by reading keys and values (64 rows over up to a day,
// 1.15 GB: 224 us, 5.1 TB/s; a copy 5.1), and by the latency of its steps where there is little to read (12 heads of one row over a
// day, 106 MB: 29 us and 7 for the join; 32 pages of a week 12 and 4). Four waves of a block take tiles of 32 tokens in turn,
// straight from memory into the matrix instructions' registers: the scores' product has keys as its rows in such an order that a lane ends with the scores of 8 tokens
// in a row, 8 q4 .. 8 q4 + 7 (q4 = lane / 16), for query lane & 15, which is what the second product's operand holds; values are
// loaded as 8 tokens by CPL columns a lane and change places within the lane. Each wave has its own maximum and sums, joined at
// the end over waves, and over the blocks of a split by k_kva_join. fp16: e^{s - m} goes into the product in two parts, 22 bits,
// in units of 2^-12 so that the second part of small ones is no subnormal: the matrix cores wait for memory here.
template <typename T, int D, int MT, bool V>
__device__ __forceinline__ void kva_tile(const KvDev &c, const KvaDev &p, const KvaItem &it, int nrt, int2 *counts, float *part,
                                         float2 *pml) {
  constexpr bool F16 = sizeof(T) == 2;
  constexpr int DKT = D / 32, CPL = D / 16, MR = 16 * MT;
  constexpr float OFF = F16 ? 12.f : 0.f;
  typedef kv_vec<T, 8> FV;
  __shared__ __attribute__((aligned(16))) float s_o[4][16 * (D + 4)];
  __shared__ float s_m[4][MR], s_l[4][MR];
  const int b = it.b, g = it.g, tile = it.tile;
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int first = it.first, past = it.past, n = it.n;
  const KvaSpan span = kva_span(c, p, tile, MR, 32, n, past);
  if (span.t0 >= n) return;
  const int t0 = span.t0, t1 = span.t1, base = span.base;
  // queries
  FV qf[MT][DKT];
  int at[MT], since[MT];  // the last token that the lane's query sees, and the first
#pragma unroll
  for (int m = 0; m < MT; m++) {
    int t, h;
    kva_row(p, tile, 16 * m + lr, MR, &t, &h);
    const bool in = t < n;
    at[m] = in ? past + t : -1;
    since[m] = p.window && at[m] >= p.window ? at[m] - p.window + 1 : 0;
    const T *q = (const T *)p.q + ((long long)first + (in ? t : t0)) * p.ldq + ((long long)g * p.G + (in ? h : 0)) * c.dk;
#pragma unroll
    for (int d = 0; d < DKT; d++) {
      qf[m][d] = kv_ld<T, 8, V>(q, 32 * d + 8 * q4, in ? c.dk : 0);
      if (p.sign != 1.f) qf[m][d] *= (T)p.sign;
    }
  }
  // tokens
  const int all0 = p.window && past + t1 >= p.window ? past + t1 - p.window + 1 : 0;  // from here and ..
  const int all1 = past + t0;                                                         // .. up to here every query sees them
  const int *sel = p.sel ? p.sel + (((long long)first + t0) * c.Hk + g) * p.nsel : nullptr;
  const int kt0 = it.sp ? it.sp * it.per : 0, kt1 = it.per < span.nt - kt0 ? kt0 + it.per : span.nt;

  v4f o[MT][CPL];
  float mx[MT], l[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) {
    mx[m] = -INFINITY, l[m] = 0.f;
#pragma unroll
    for (int i = 0; i < CPL; i++) o[m][i] = (v4f){0.f, 0.f, 0.f, 0.f};
  }
  // the first tokens of a tile's two groups of 16, and their pages (-1: not there)
  auto look = [&](int kt, int (&j)[2], int (&pg)[2]) {
#pragma unroll
    for (int s = 0; s < 2; s++) {
      if (s == 1 && c.sh > 4) {
        j[1] = j[0] + 16, pg[1] = pg[0];
        break;
      }
      pg[s] = -1, j[s] = 0;
      if (kt >= kt1) continue;
      int pi;
      if (p.sel) {
        const int x = 2 * kt + s, e = x >> (c.sh - 4);
        if (e >= p.nsel) continue;
        pi = sel[e];
        if (pi < 0 || pi >= c.ldt || (e > 0 && pi <= sel[e - 1])) continue;
        j[s] = (pi << c.sh) + ((x & ((1 << (c.sh - 4)) - 1)) << 4);
      } else {
        j[s] = 32 * (base + kt) + 16 * s;
        pi = j[s] >> c.sh;
      }
      pg[s] = kv_page(c, b, pi);
    }
  };
  // piece x of a row of values: CPL columns from here, the last ones for one that the row's end cuts (those that are the piece's
  // before as well are the same twice; pieces past the end are nobody's)
  auto vcol = [&](int x) { return V || CPL * x + CPL <= c.dv || c.dv < CPL ? CPL * x : c.dv - CPL; };
  int jn[2], pn[2], bad0 = 0x7fffffff, bad1 = -1;  // tiles with values that are not finite: left out, and added at the end
  look(kt0 + wave, jn, pn);
  for (int kt = kt0 + wave; kt < kt1; kt += 4) {
    int j[2] = {jn[0], jn[1]}, pg[2] = {pn[0], pn[1]};
    look(kt + 4, jn, pn);
    if (pg[0] < 0 && pg[1] < 0) continue;
    const bool full = pg[0] >= 0 && pg[1] >= 0 && j[0] >= all0 && j[1] >= all0 && j[0] + 15 <= all1 && j[1] + 15 <= all1;
    const T *kb[2], *vb[2];
#pragma unroll
    for (int s = 0; s < 2; s++) {  // one that is not there is read where the other is
      const int x = pg[s] < 0 ? 1 - s : s;
      const long long in = ((long long)g << c.sh) + (j[x] & ((1 << c.sh) - 1));
      kb[s] = (const T *)c.k + pg[x] * c.k_ps + in * c.dk;
      vb[s] = (const T *)c.v + pg[x] * c.v_ps + in * c.dv;
    }
    const T *kp = (lr & 8 ? kb[1] : kb[0]) + (8 * (lr >> 2 & 1) + (lr & 3)) * c.dk;
    const T *vp = (q4 & 2 ? vb[1] : vb[0]) + 8 * (q4 & 1) * c.dv;
    FV kf[2][DKT];
    kv_vec<T, CPL> vr[8];
    if constexpr (V) {
#pragma unroll
      for (int d = 0; d < DKT; d++) {
        kf[0][d] = kv_ld<T, 8, V>(kp, 32 * d + 8 * q4, c.dk);
        kf[1][d] = kv_ld<T, 8, V>(kp + 4 * c.dk, 32 * d + 8 * q4, c.dk);
      }
#pragma unroll
      for (int e = 0; e < 8; e++) vr[e] = kv_ld<T, CPL, V>(vp + e * c.dv, CPL * lr, c.dv);
    } else {
      int kc = 8 * q4, vc = vcol(lr);  // what follows from them is found anew for each tile: there is no room to keep it
      asm volatile("" : "+v"(kc), "+v"(vc));
#pragma unroll
      for (int d = 0; d < DKT; d++)
        if (F16 || 32 * d < c.dk) {  // fp32: 64 rows over up to 4,000 tokens, 12 heads of 63 and 62, 90 us, 107 with those past the row read as well
          kf[0][d] = kv_raw<T, 8>(kp, 32 * d + kc, c.dk);
          kf[1][d] = kv_raw<T, 8>(kp + 4 * c.dk, 32 * d + kc, c.dk);
        }
#pragma unroll
      for (int e = 0; e < 8; e++) vr[e] = kv_raw<T, CPL>(vp + e * c.dv, vc, c.dv);
#pragma unroll
      for (int d = 0; d < DKT; d++)
        if (32 * d + 32 > c.dk && (F16 || 32 * d < c.dk)) {
          kf[0][d] = kv_fix<T, 8>(kf[0][d], 32 * d + kc, c.dk);
          kf[1][d] = kv_fix<T, 8>(kf[1][d], 32 * d + kc, c.dk);
        }
    }
    v4f s[MT][2];
#pragma unroll
    for (int m = 0; m < MT; m++) s[m][0] = s[m][1] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DKT; d++)
#pragma unroll
      for (int m = 0; m < MT && (V || F16 || 32 * d < c.dk); m++) s[m][0] = mma(kf[0][d], qf[m][d], s[m][0]), s[m][1] = mma(kf[1][d], qf[m][d], s[m][1]);
    const int jl = (q4 & 2 ? j[1] : j[0]) + 8 * (q4 & 1);  // the lane's 8 tokens
    const bool there = (q4 & 2 ? pg[1] : pg[0]) >= 0;
    kv_vec<T, 2> mk = {(T)0, (T)0};
#pragma unroll
    for (int e = 0; e < 8; e++) kv_mark<T, CPL>(vr[e], mk);
    if (__builtin_amdgcn_ballot_w64(mk[0] != mk[0] || mk[1] != mk[1])) {
      bad0 = bad0 < kt ? bad0 : kt, bad1 = kt;
#pragma unroll
      for (int e = 0; e < 8; e++)
#pragma unroll
        for (int i = 0; i < CPL; i++) vr[e][i] = kv_finite(vr[e][i]) ? vr[e][i] : (T)0;
    }
    if (!full) {
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const bool in = there && jl + e <= at[m] && jl + e >= since[m];
          s[m][e / 4][e % 4] = in ? s[m][e / 4][e % 4] : -INFINITY;
        }
    }
    FV ph[MT], pl[F16 ? MT : 1];
#pragma unroll
    for (int m = 0; m < MT; m++) {
      float top = s[m][0][0];
#pragma unroll
      for (int e = 1; e < 8; e++) top = fmaxf(top, s[m][e / 4][e % 4]);
      top = fmaxf(mx[m], top * p.sc);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float to = (top == -INFINITY ? 0.f : top) - OFF;
      if (__builtin_amdgcn_ballot_w64(top != mx[m])) {
        const float a = __builtin_amdgcn_exp2f(mx[m] - OFF - to);  // 0 from -inf
        l[m] *= a;
#pragma unroll
        for (int i = 0; i < CPL; i++) o[m][i] *= a;
      }
      mx[m] = top;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[m][e / 4][e % 4], p.sc, -to));
        l[m] += x;
        ph[m][e] = (T)x;
        if (F16) pl[m][e] = (T)(x - (float)ph[m][e]);
      }
    }
#pragma unroll
    for (int i = 0; i < CPL; i++) {
      FV a;
#pragma unroll
      for (int e = 0; e < 8; e++) a[e] = vr[e][i];
#pragma unroll
      for (int m = 0; m < MT; m++) {
        if (F16) o[m][i] = mma(a, pl[m], o[m][i]);
        o[m][i] = mma(a, ph[m], o[m][i]);
      }
    }
  }
  // Values that are not finite, for the queries that see them: within the products, 0 times them would reach the others, and
  // an infinity times a second part of 0 be none
  for (int kt = bad0; kt <= bad1; kt += 4) {
    int j[2], pg[2];
    look(kt, j, pg);
#pragma unroll 1
    for (int k = 0; k < 32; k++) {
      const int x = k >> 4, tk = (x ? j[1] : j[0]) + (k & 15), page = x ? pg[1] : pg[0];
      if (page < 0) continue;
      const long long in = ((long long)g << c.sh) + (tk & ((1 << c.sh) - 1));
      const T *v = (const T *)c.v + page * c.v_ps + in * c.dv, *kr = (const T *)c.k + page * c.k_ps + in * c.dk;
      bool bad = false;
      for (int col = lane; col < c.dv; col += 64) bad = bad || !kv_finite(v[col]);
      if (!__builtin_amdgcn_ballot_w64(bad)) continue;
#pragma unroll
      for (int m = 0; m < MT; m++) {
        float s = 0.f;
#pragma unroll
        for (int d = 0; d < DKT; d++) {
          const FV y = kv_ld<T, 8, V>(kr, 32 * d + 8 * q4, c.dk);
#pragma unroll
          for (int e = 0; e < 8; e++) s = __builtin_fmaf((float)y[e], (float)qf[m][d][e], s);
        }
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        if (tk > at[m] || tk < since[m] || s == -INFINITY) continue;
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s, p.sc, OFF - mx[m]));
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (int i = 0; i < CPL; i++) {
            const int col = vcol(4 * q4 + r) + i;
            const float z = col < c.dv ? (float)v[col] : 0.f;
            if (!kv_finite(z)) o[m][i][r] += y * z;
          }
      }
    }
  }
  if (counts && tid == 0 && it.sp == 0) counts[((long long)b * c.Hk + g) * nrt + tile] = make_int2(it.item, it.parts);
  // the four waves' sums
#pragma unroll
  for (int m = 0; m < MT; m++) {
    l[m] += __shfl_xor(l[m], 16);
    l[m] += __shfl_xor(l[m], 32);
    if (q4 == 0) s_m[wave][16 * m + lr] = mx[m], s_l[wave][16 * m + lr] = l[m];
  }
#pragma unroll
  for (int m = 0; m < MT; m++) {
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int i = 0; i < CPL; i++)
        if (V || CPL * (4 * q4 + r) < c.dv) s_o[wave][lr * (D + 4) + vcol(4 * q4 + r) + i] = o[m][i][r];
    __syncthreads();
    const int x = tid >> 4, c0 = (tid & 15) * CPL, row = 16 * m + x;
    float top = s_m[0][row], f[4], sum = 0.f;
#pragma unroll
    for (int w = 1; w < 4; w++) top = fmaxf(top, s_m[w][row]);
    const float to = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      f[w] = __builtin_amdgcn_exp2f(s_m[w][row] - to);
      sum += f[w] * s_l[w][row];
    }
    float y[CPL];
#pragma unroll
    for (int i = 0; i < CPL; i++) {
      y[i] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; w++) y[i] = __builtin_fmaf(f[w], s_o[w][x * (D + 4) + c0 + i], y[i]);
    }
    if (it.parts == 1) {
      int t, h;
      kva_row(p, tile, row, MR, &t, &h);
      if (t >= n) continue;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      T *out = (T *)p.o + ((long long)first + t) * p.ldo + ((long long)g * p.G + h) * c.dv;
      if (V) {
        kv_vec<T, CPL> z;
#pragma unroll
        for (int i = 0; i < CPL; i++) z[i] = (T)(y[i] * inv);
        if (c0 < c.dv) *(kv_vec<T, CPL> *)(out + c0) = z;
      } else {
#pragma unroll
        for (int i = 0; i < CPL; i++)
          if (c0 + i < c.dv) out[c0 + i] = (T)(y[i] * inv);
      }
    } else {
      const long long at = (long long)it.item * MR + row;
      if ((tid & 15) == 0) pml[at] = make_float2(top, sum);
      if (sum != 0.f)
#pragma unroll
        for (int i = 0; i < CPL; i += 2) *(float2 *)(part + at * D + c0 + i) = make_float2(y[i], y[i + 1]);
    }
  }
}

template <typename T, int D, int MT, bool V>
__global__ __launch_bounds__(256, sizeof(T) == 2 && D <= 128 && MT == 1 ? 3 : 1) void k_kva(KvDev c, KvaDev p, int B, int nrt, unsigned blk0, int2 *counts, float *part,
                                             float2 *pml) {
  KvaItem it;
  if (kva_item(c, p, B, nrt, counts, 16 * MT, 32, blk0 + blockIdx.x, &it)) kva_tile<T, D, MT, V>(c, p, it, nrt, counts, part, pml);
}

// The parts of a split: each row's sums over them, in order. D / 4 lanes to a row, which read up to 8 of its parts at once, for
// tiles of many rows
template <typename T, int D>
__global__ __launch_bounds__(256) void k_kva_join8(KvDev c, KvaDev p, int nrt, int MR, unsigned unit0, const int2 *counts,
                                                   const float *part, const float2 *pml) {
  constexpr int L = D / 4, R = 256 / L;  // lanes to a row; rows at a time
  const unsigned unit = unit0 + blockIdx.x, sq = unit / (unsigned)nrt, b = sq / (unsigned)c.Hk;
  const int tile = (int)(unit - sq * nrt), g = (int)(sq - b * c.Hk);
  const int col = threadIdx.x % L * 4;
  int first, past, t, h;
  const int n = kv_rows(c, b, &first, &past);
  kva_row(p, tile, 0, MR, &t, &h);
  if (t >= n) return;
  const int parts = kv_int(&counts->y, 2 * (long long)unit), item = kv_int(&counts->x, 2 * (long long)unit);
  if (parts == 1) return;
  for (int m = blockIdx.y * R + threadIdx.x / L; m < MR; m += gridDim.y * R) {
    kva_row(p, tile, m, MR, &t, &h);
    if (t >= n || col >= c.dv) continue;
    const long long at = (long long)item * MR + m;
    float top = -INFINITY, sum = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < parts; s0 += 8) {
      float2 z[8];
      float4 v[8];
#pragma unroll
      for (int s = 0; s < 8; s++) {
        z[s] = make_float2(-INFINITY, 0.f);
        if (s0 + s < parts)
          z[s] = pml[at + (long long)(s0 + s) * MR], v[s] = *(const float4 *)(part + (at + (long long)(s0 + s) * MR) * D + col);
      }
      float now = top;
#pragma unroll
      for (int s = 0; s < 8; s++) now = fmaxf(now, z[s].x);
      const float to = now == -INFINITY ? 0.f : now, a = __builtin_amdgcn_exp2f(top - to);
      sum *= a;
#pragma unroll
      for (int i = 0; i < 4; i++) y[i] *= a;
      top = now;
#pragma unroll
      for (int s = 0; s < 8; s++) {
        if (z[s].y == 0.f) continue;  // a part without a weight has stored nothing
        const float f = __builtin_amdgcn_exp2f(z[s].x - to);
        sum = __builtin_fmaf(f, z[s].y, sum);
        y[0] = __builtin_fmaf(f, v[s].x, y[0]), y[1] = __builtin_fmaf(f, v[s].y, y[1]);
        y[2] = __builtin_fmaf(f, v[s].z, y[2]), y[3] = __builtin_fmaf(f, v[s].w, y[3]);
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T *out = (T *)p.o + ((long long)first + t) * p.ldo + ((long long)g * p.G + h) * c.dv + col;
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (col + i < c.dv) out[i] = (T)(y[i] * inv);
  }
}
// For few rows: a block to a row, whose four waves share its parts
template <typename T, int D>
__global__ __launch_bounds__(256) void k_kva_join(KvDev c, KvaDev p, int nrt, int MR, unsigned unit0, const int2 *counts,
                                                  const float *part, const float2 *pml) {
  constexpr int N = D >= 64 ? D / 64 : 1;  // columns to a lane
  typedef float VN __attribute__((ext_vector_type(N)));
  __shared__ float s_f[4][kMostParts];
  __shared__ __attribute__((aligned(16))) float s_y[4][D < 64 ? 64 : D];
  const unsigned unit = unit0 + blockIdx.x, sq = unit / (unsigned)nrt, b = sq / (unsigned)c.Hk;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m = blockIdx.y, tile = (int)(unit - sq * nrt), g = (int)(sq - b * c.Hk);
  int first, past, t, h;
  const int n = kv_rows(c, b, &first, &past);
  kva_row(p, tile, m, MR, &t, &h);
  if (t >= n) return;  // the tile's first row is the sequence's if any is
  const int parts = kv_int(&counts->y, 2 * (long long)unit), item = kv_int(&counts->x, 2 * (long long)unit);
  if (parts == 1) return;
  const long long at = (long long)item * MR + m;
  // the parts' weights, in every wave
  float top = -INFINITY, sum = 0.f;
  float2 z[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    z[i] = make_float2(-INFINITY, 0.f);
    if (lane + 64 * i < parts) z[i] = pml[at + (long long)(lane + 64 * i) * MR];
    top = fmaxf(top, z[i].x);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  const float to = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const float f = z[i].y == 0.f ? 0.f : __builtin_amdgcn_exp2f(z[i].x - to);
    s_f[wave][lane + 64 * i] = f;
    sum = __builtin_fmaf(f, z[i].y, sum);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  const int col = lane * N;
  VN y = (VN)0.f;
  if (col < D)
#pragma unroll 8
    for (int s = wave; s < parts; s += 4) {
      const float f = s_f[wave][s];
      const VN v = *(const VN *)(part + (at + (long long)s * MR) * D + col);
      if (f != 0.f) y += f * v;
    }
  *(VN *)(s_y[wave] + col) = y;
  __syncthreads();
  if (wave || col >= c.dv) return;
#pragma unroll
  for (int i = 1; i < 4; i++) y += *(const VN *)(s_y[i] + col);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T *out = (T *)p.o + ((long long)first + t) * p.ldo + ((long long)g * p.G + h) * c.dv + col;
#pragma unroll
  for (int i = 0; i < N; i++)
    if (col + i < c.dv) out[i] = (T)(y[i] * inv);
}

// How a call is cut
KvaPlan plan(const bnh_kvcache *c, const bnh_kvattn *p, int T, int B) {
  KvaPlan r;
  const int d = c->dk > c->dv ? c->dk : c->dv, G = p->H / c->Hk;
  const long long m = p->nsel ? G : (long long)T * G;
  r.D = d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256;
  // The tiled form's waves have 32 rows each, and 128 or 256 to a block; the other one's time goes up at 17 rows and at 65, past 128
  // wide at 33. Tiled and the other, us, for 24 stations' caches of up to 5,000 tokens and 4 heads, and one of a day and 12 heads.
  // fp16, 64 wide: 16 rows 20.8 and 16.5, 34.1 and 21.6; 17 rows 20.8 and 25.9, 34.3 and 43.4. 128: 25.4 and 20.7, 40.9 and 30.0; 25.3
  // and 30.3, 40.8 and 57.7. 136: 32 rows 38.3 and 40.6, 86.3 and 73.6; 33 rows 39.3 and 43.8, 88.2 and 131.5. 192: 39.0 and 33.7, 87.0
  // and 62.3; 39.7 and 38.1, 89.2 and 107.9. 256: 40.5 and 36.3, 89.6 and 67.4; 40.8 and 40.0, 91.5 and 119.5. fp32, whose products
  // take as long for rows that are nobody's: 64 rows of 128 63.4 and 65.0, 167 and 150; 65 rows 63.8 and 72.5, 166 and 185
  r.tiled = !p->nsel && m > (!c->f16 ? 64 : d <= 128 ? 16 : 32);
  r.TK = 32;
  if (r.tiled) {
    r.DK = c->dk <= 64 && d <= 128 ? 64 : d <= 128 ? 128 : 256;
    r.D = c->dv <= 64 && d <= 128 ? 64 : d <= 128 ? 128 : 256;
    r.MR = 32 * kva_waves(c->f16, r.DK);
    r.TK = kva_tokens(c->f16, r.DK);
  } else {
    const int big = c->f16 ? (r.D <= 128 ? 64 : 32) : r.D <= 64 ? 64 : r.D == 128 ? 32 : 16;
    r.MR = m <= 16 ? 16 : big;
  }
  r.nrt = (int)(p->nsel ? T * bnh_ceil_div(G, r.MR) : bnh_ceil_div(m, r.MR));
  r.units = (long long)B * c->Hk * r.nrt;
  // tiles of 32 tokens that a row tile can see
  long long tok = (long long)c->ldt * c->page;
  if (p->nsel) tok = (long long)p->nsel * c->page;
  else if (p->window && (long long)p->window + r.MR < tok) tok = (long long)p->window + r.MR;
  const long long tiles = bnh_ceil_div(tok, 32) + 1;
  // parts for the compute units where tiles leave some without work: one block each of the tiled form, with room for the last
  // parts of tiles (24 chunks of up to 120 rows: 54 us with the join, 63 with 256), four of the other (64 rows over up to a day: 223 +
  // 6 us, 229 + 6 with 768, 241 + 5 with 512), of 512 tokens at least, or what is joined costs more (one row over a day: 24 + 7 us
  // in 406 parts, 23 + 9 in 732)
  r.want = r.tiled ? 192 : 1024;
  r.least = r.tiled ? 256 / r.TK : p->nsel ? 8 : 16;
  r.split = r.units < 2 * r.want && tiles > (r.tiled ? 2 * r.least * r.TK / 32 : 2 * r.least);
  r.items = r.split ? r.want + r.units + 1 : r.units;
  return r;
}
template <typename T, int D>
int join_run(const KvDev &c, const KvaDev &p, const KvaPlan &r, void *work, hipStream_t s) {
  if (!r.split) return 0;
  const long long most = bnh_most_blocks(256);
  // rows that a tile can have, as blocks, or as some passes of a few
  const long long rows = p.nsel ? p.G : (long long)c.T * p.G;
  const int R = 1024 / D, few = 16, y = r.tiled ? (r.MR / R < few ? r.MR / R : few) : (int)(rows < r.MR ? rows : r.MR);
  for (long long u0 = 0; u0 < r.units; u0 += most) {
    const dim3 grid((unsigned)(r.units - u0 < most ? r.units - u0 : most), y), block(256);
    if (r.tiled)
      hipLaunchKernelGGL((k_kva_join8<T, D>), grid, block, 0, s, c, p, r.nrt, r.MR, (unsigned)u0, kva_counts(r, work),
                         kva_part(r, work), kva_ml(r, work));
    else
      hipLaunchKernelGGL((k_kva_join<T, D>), grid, block, 0, s, c, p, r.nrt, r.MR, (unsigned)u0, kva_counts(r, work),
                         kva_part(r, work), kva_ml(r, work));
    BNH_HIP(hipGetLastError());
  }
  return 0;
}
template <typename T, int D, int MT, bool V>
int rows_run(const KvDev &c, const KvaDev &p, const KvaPlan &r, void *work, hipStream_t s) {
  const long long most = bnh_most_blocks(256);
  const int B = (int)(r.units / r.nrt / c.Hk);
  for (long long b0 = 0; b0 < r.items; b0 += most) {
    const long long n = r.items - b0 < most ? r.items - b0 : most;
    hipLaunchKernelGGL((k_kva<T, D, MT, V>), dim3((unsigned)n), dim3(256), 0, s, c, p, B, r.nrt, (unsigned)b0, kva_counts(r, work),
                       kva_part(r, work), kva_ml(r, work));
    BNH_HIP(hipGetLastError());
  }
  return join_run<T, D>(c, p, r, work, s);
}
template <typename T, int D, bool V>
int rows_go(const KvDev &c, const KvaDev &p, const KvaPlan &r, void *work, hipStream_t s) {
  constexpr int big = sizeof(T) == 2 ? (D <= 128 ? 4 : 2) : D <= 64 ? 4 : D == 128 ? 2 : 1;
  if constexpr (big > 1)
    if (r.MR > 16) return rows_run<T, D, big, V>(c, p, r, work, s);
  return rows_run<T, D, 1, V>(c, p, r, work, s);
}
template <typename T>
int tiles_run(const KvDev &c, const KvaDev &p, const KvaPlan &r, int w, void *work, hipStream_t s) {
  if (kva_tiles(c, p, r, sizeof(T) == 2, w, work, s)) return -1;
  return r.D == 64    ? join_run<T, 64>(c, p, r, work, s)
         : r.D == 128 ? join_run<T, 128>(c, p, r, work, s)
                      : join_run<T, 256>(c, p, r, work, s);
}
template <typename T, bool V>
int run(const KvDev &c, const KvaDev &p, const KvaPlan &r, void *work, hipStream_t s) {
  if (r.D == 32) return rows_go<T, 32, V>(c, p, r, work, s);
  if (r.D == 64) return rows_go<T, 64, V>(c, p, r, work, s);
  if (r.D == 128) return rows_go<T, 128, V>(c, p, r, work, s);
  return rows_go<T, 256, V>(c, p, r, work, s);
}

int attn_check(const bnh_kvcache *c, const bnh_kvattn *p, int T, int B, int rows) {
  if (kv_check(c, T, B, rows)) return -1;
  BNH_REQ(p && p->H > 0 && p->H % c->Hk == 0 && p->H <= 65536 && p->window >= 0 && p->nsel >= 0 && p->nsel <= (1 << 20));
  BNH_REQ((long long)T * p->H < (1LL << 31) && (long long)rows * c->Hk < (1LL << 31));
  return 0;
}

}  // namespace

extern "C" {

size_t bnh_kv_attn_work_bytes(const bnh_kvcache *c, const bnh_kvattn *p, int T, int B, int rows) {
  if (attn_check(c, p, T, B, rows)) return 0;
  return kva_bytes(plan(c, p, T, B));
}

int bnh_kv_attn(const bnh_kvcache *c, const bnh_kvattn *p, int T, int B, int rows, const int32_t *start, const int32_t *len,
                void *work, size_t work_bytes, void *stream) {
  if (attn_check(c, p, T, B, rows) || kv_check_buffers(c, T, B, rows, start, len)) return -1;
  BNH_REQ(!p->nsel == !p->sel);
  BNH_REQ(p->q && p->o && p->ldq >= p->H * c->dk && p->ldo >= p->H * c->dv);
  const size_t es = c->f16 ? 2 : 4;
  BNH_REQ(kv_on(p->q, es) && kv_on(p->o, es) && kv_on(p->sel, 4));
  const KvaPlan r = plan(c, p, T, B);
  const size_t need = kva_bytes(r);
  BNH_REQ(r.items < (1LL << 31));
  BNH_REQ(need == 0 || (work && kv_on(work, 16) && work_bytes >= need));
  const KvDev d = kv_dev(c, T, rows, start, len);
  const float sc = p->scale == 0 ? 1.f : fabsf(p->scale * 1.44269504f), sign = p->scale == 0 ? 0.f : p->scale < 0 ? -1.f : 1.f;
  const KvaDev a = {p->q, p->o, p->sel, p->ldq, p->ldo, p->H / c->Hk, p->window, p->nsel, r.want, r.least, sc, sign};
  const int ve = 16 / (int)es, cpl = r.tiled ? 8 : r.D / 16;
  bool v = c->dk % 8 == 0 && c->dv % cpl == 0 && c->k_ps % ve == 0 && c->v_ps % ve == 0 && p->ldq % ve == 0 &&
           p->ldo % (cpl < ve ? cpl : ve) == 0;
  for (const void *x : {p->q, (const void *)p->o, (const void *)c->k, (const void *)c->v}) v = v && kv_on(x, 16);
  hipStream_t s = bnh_stream(stream);
  if (r.tiled) {
    bool four = !c->f16 || (c->dk % 2 == 0 && c->dv % 2 == 0 && c->k_ps % 2 == 0 && c->v_ps % 2 == 0);
    for (const void *x : {(const void *)c->k, (const void *)c->v}) four = four && kv_on(x, 4);
    const int w = v ? 16 : four ? 4 : 2;
    return c->f16 ? tiles_run<h16>(d, a, r, w, work, s) : tiles_run<float>(d, a, r, w, work, s);
  }
  if (c->f16) return v ? run<h16, true>(d, a, r, work, s) : run<h16, false>(d, a, r, work, s);
  return v ? run<float, true>(d, a, r, work, s) : run<float, false>(d, a, r, work, s);
}

}  // extern "C"
