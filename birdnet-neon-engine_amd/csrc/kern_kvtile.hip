// Attention of many rows over a paged cache (bnh_kv_attn): the tiled form.
//
// Bound by the matrix cores, the exponentials and what feeds both out of LDS, at the clock that the card's power leaves: 17,280
// rows of 12 heads of 128 from an empty cache 1,290 to 1,320 us, 700 TFLOP/s of the two products and 1,050 with the weights' second
// part (a library product of 8,192 cubed 1,164), the matrix cores busy for 56% of the cycles, no bank conflict. fp32 4,000 rows 565 us,
// 87 of 153 TFLOP/s. Short calls are bound by what a block does before its first tile, about 14,000 cycles, and by the join of parts:
// 24 chunks of up to 120 rows over up to 5,000 tokens 41 + 13 us. The NW waves of a block own 32 rows each (query heads that share
// keys are rows too) and share tiles of TK tokens in LDS, which loads bring there while the tile before is multiplied (by way of
// registers for odd widths of fp16, and where values are not finite). Scores are K q^T, so that a lane has tokens of one query (lane & 31): maxima and sums stay in the lane but for
// one exchange, and the exponentials are the second product's operand as they lie, given that row m of the first product is
// token m with bits 2 and 3 exchanged. Rows of LDS are pieces of 16 bytes, exchanged by bits of the token such that neither the
// reads of 16 tokens' pieces nor the transposing reads of 4 tokens meet in a bank.
#include <math.h>

#include "bnh_kvattn.h"
#include "bnh_lds_dma.h"

namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
__device__ __forceinline__ v16f mma(kv_vec<h16, 8> a, kv_vec<h16, 8> b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v16f mma(kv_vec<float, 8> a, kv_vec<float, 8> b, v16f c) {
#pragma unroll
  for (int e = 0; e < 8; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}
// where piece x of token k's row of CH pieces lies
template <int CH>
__device__ __forceinline__ int piece(int k, int x) {
  const int f = CH == 8 ? (k >> 1 & 1) << 2 | (k >> 2 & 3) : (k & 3) << 2 | (k >> 2 & 3);
  return k * CH + (x ^ f);
}

// an address that all lanes have, as the wave's own
__device__ __forceinline__ const void *one(const void *p) {
  const uint64_t x = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
  return (const void *)(uintptr_t)((uint64_t)hi << 32 | lo);
}
// the larger of a lane's and that of the lane 32 from it
__device__ __forceinline__ float both(float x) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  const u2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// fp16: the waves of a block are two groups, one wave of each on every SIMD, half a tile apart: while one multiplies (its
// last tile's values and the next one's scores), the other takes exponentials. Waves in step would all want the matrix cores
// and then all want the exponentials: 17,280 rows of 12 heads of 128 take 1,438 us so, not 1,315. fp32 products take ten times as
// long as the exponentials, and the groups go in step.
// W: bytes of a lane's load, which everything is aligned to: 16, 4, or 2 (odd widths of fp16), where all goes through registers.
// 8,000 rows of 12 heads of 128 and 126: 332 us by fours, 595 us through registers; fp32, 16 heads of 64 and 97, 256 tokens seen:
// 53 us and 68
template <typename T, int DK, int DV, int NW, int NG, int W>
__device__ __forceinline__ void kvt_item(const KvDev &c, const KvaDev &p, const KvaItem &it, int nrt, int2 *counts, float *part,
                                         float2 *pml) {
  constexpr bool F16 = sizeof(T) == 2, PP = F16 && NW == 8, V = W == 16;
  constexpr int VE = 16 / sizeof(T), TK = kva_tokens(F16, DK), ST = TK / 32, NT = 64 * NW, MR = 32 * NW;
  constexpr int KC = DK / VE, VC = DV / VE;                    // pieces of a row
  constexpr int KP = NT / KC, VP = NT / VC;                    // tokens that one load of all threads covers
  constexpr int NK = TK / KP, NV = TK / VP, GT = TK / NG;
  constexpr int NB = DK == 256 && !F16 ? 2 : 3;                // tiles in LDS
  // Weights are in units of 2^-12, so that the second part of those down to 2^-15 of the largest is no subnormal, and nothing above
  // 2^-37 of it is lost; the running maximum may be short by GROW in the exponent before the sums are scaled anew (2^15 at most:
  // nothing overflows)
  constexpr float OFF = F16 ? 12.f : 0.f, GROW = 3.f;
  typedef kv_vec<T, 8> FV;
  typedef kv_vec<T, VE> PV;
  constexpr int KB = TK * KC * 16, VB = TK * VC * 16;          // bytes of a tile
  __shared__ PV s_kb[NB][TK * KC], s_vb[NB][TK * VC];
  __shared__ int s_bad[3];  // the first and last tile with values that are not finite; whether the outputs show any
  const int b = it.b, g = it.g, tile = it.tile;
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int first = it.first, past = it.past, n = it.n;
  int tx, hx;
  const KvaSpan span = kva_span(c, p, tile, MR, TK, n, past);
  if (span.t0 >= n) return;
  const int j1 = span.j1, end = span.base + span.nt;
  const int kt0 = it.sp ? span.base + it.sp * it.per : span.base, kt1 = it.per < end - kt0 ? kt0 + it.per : end;
  kva_row(p, tile, 32 * wave + lr, MR, &tx, &hx);
  const bool mine = tx < n;
  const int at = mine ? past + tx : -1, since = p.window && at >= p.window ? at - p.window + 1 : 0;
  FV qf[DK / 16];
  {
    const T *q = (const T *)p.q + ((long long)first + (mine ? tx : span.t0)) * p.ldq + ((long long)g * p.G + (mine ? hx : 0)) * c.dk;
#pragma unroll
    for (int d = 0; d < DK / 16; d++) {
      qf[d] = kv_ld<T, 8, V>(q, 16 * d + 8 * hi, mine ? c.dk : 0);
      if (p.sign != 1.f) qf[d] *= (T)p.sign;
    }
  }
  // this wave's rows see all of [all0, all1], and nothing outside [see0, see1]
  int w0, w1, hw;
  kva_row(p, tile, 32 * wave, MR, &w0, &hw);
  kva_row(p, tile, 32 * wave + 31, MR, &w1, &hw);
  w1 = w1 < n ? w1 : n - 1;
  const bool idle = w0 >= n;
  const int all0 = p.window && past + w1 >= p.window ? past + w1 - p.window + 1 : 0, all1 = past + w0;
  const int see0 = p.window && past + w0 >= p.window ? past + w0 - p.window + 1 : 0, see1 = past + w1;

  v16f o[DV / 32];
  float mx, l;

  // The sequence's pages, 64 of them at a time in the lanes of a register, from page pb on (-1: not there)
  int pt = -1, pb = -64;
  auto page_of = [&](int token) {
    const int x = token >> c.sh;
    if (x - pb >= 64 || x < pb) {
      pb = x;
      pt = kv_page(c, b, x + lane);
    }
    return __builtin_amdgcn_readlane(pt, x - pb);
  };
  const int inpage = (1 << c.sh) - 1;
  const T *kh = (const T *)c.k + ((long long)g << c.sh) * c.dk, *vh = (const T *)c.v + ((long long)g << c.sh) * c.dv;

  // The work on a tile
  v16f s[ST];
  // fp16: weights in two parts, 22 bits, and a product for each. In one part's 11 bits outputs whose terms cancel are off by several
  // times their own rounding (17,280 rows of 12 heads of 128: 976 us so, 1,315 with both; 24 chunks of up to 120 rows 48 and 54)
  FV ph[2 * ST], pl[F16 ? 2 * ST : 1];
  // A tile is NG groups of GT tokens that have a page each: one for pages of TK tokens or more, else groups of 16
  int pc[NG];
  auto seen = [&](int kt) {  // whether the wave has rows that see a token of the tile
    return !idle && kt * TK <= see1 && kt * TK + TK - 1 >= see0;
  };
  // Places in LDS: a lane's first one; the others of its products are that one with bits exchanged, or a fixed way behind
  typedef __attribute__((address_space(3))) const char *Lds;
  const int row = (lr & 19) | (lr & 4) << 1 | (lr & 8) >> 1;  // the token of the first product's row
  const int ka = 16 * piece<KC>(row, F16 ? hi : 2 * hi);
  // the second one's: F16, 4 tokens by 16 columns to a group of 16 lanes, which get them by column
  const int va = F16 ? 16 * piece<VC>(8 * hi + (lane >> 2 & 3), (lane >> 3 & 2) + (lane >> 1 & 1)) + 8 * (lane & 1)
                     : 16 * piece<VC>(8 * hi, lr >> 2) + 4 * (lr & 3);
  auto scores = [&](int buf) {
    const int x = ka + buf * KB;
#pragma unroll
    for (int i = 0; i < ST; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) s[i][r] = 0.f;
#pragma unroll
    for (int d = 0; d < DK / 16; d++)
#pragma unroll
      for (int i = 0; i < ST; i++) {
        typedef __attribute__((address_space(3))) const PV *L;
        FV a;
        if constexpr (F16) {
          a = *(L)((Lds)&s_kb[0][0] + (x ^ 32 * d) + 32 * i * KC * 16);
        } else {
          const PV y = *(L)((Lds)&s_kb[0][0] + (x ^ 64 * d) + 32 * i * KC * 16);
          const PV z = *(L)((Lds)&s_kb[0][0] + (x ^ (64 * d + 16)) + 32 * i * KC * 16);
          a = __builtin_shufflevector(y, z, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        s[i] = mma(a, qf[d], s[i]);
      }
  };
  auto weigh = [&](int kt) {
    const int j = kt * TK;
    bool full = j >= all0 && j + TK - 1 <= all1;
#pragma unroll
    for (int i = 0; i < NG; i++) full = full && pc[i] >= 0;
    if (!full) {
#pragma unroll
      for (int i = 0; i < ST; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const int x = j + 32 * i + 16 * (r >> 3) + 8 * hi + (r & 7);
          const bool in = x <= at && x >= since && pc[NG == 1 ? 0 : 2 * i + (r >> 3)] >= 0;
          s[i][r] = in ? s[i][r] : -INFINITY;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 0; i < ST; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) top = fmaxf(top, s[i][r]);
    top *= p.sc;
    top = both(top);
    if (__builtin_amdgcn_ballot_w64(top > mx + GROW)) {
      top = fmaxf(top, mx);
      const float a = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - top);
      l *= a;
#pragma unroll
      for (int i = 0; i < DV / 32; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[i][r] *= a;
      mx = top;
    }
    const float to = (mx == -INFINITY ? 0.f : mx) - OFF;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < ST; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][r], p.sc, -to));
        sum[r & 3] += x;
        const T y = (T)x;
        ph[2 * i + r / 8][r % 8] = y;
        if (F16) pl[2 * i + r / 8][r % 8] = (T)(x - (float)y);
      }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  };
  auto values = [&](int buf, auto between) {
    const int x = va + buf * VB;
#pragma unroll
    for (int k = 0; k < 2 * ST; k++)
#pragma unroll
      for (int v = 0; v < DV / 32; v++) {
        FV a;
        if constexpr (F16) {
          typedef short v4s __attribute__((ext_vector_type(4)));
          typedef short v8s __attribute__((ext_vector_type(8)));
          typedef __attribute__((address_space(3))) v4s *L;
          const Lds y = (Lds)&s_vb[0][0] + 16 * k * VC * 16;
          const v4s z0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L)(y + (x ^ 64 * v)));
          const v4s z1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L)(y + (x ^ (64 * v + 16)) + 4 * VC * 16));
          const v8s z = __builtin_shufflevector(z0, z1, 0, 1, 2, 3, 4, 5, 6, 7);
          a = __builtin_bit_cast(FV, z);
        } else {
          typedef __attribute__((address_space(3))) const float *L;
#pragma unroll
          for (int e = 0; e < 8; e++)
            a[e] = *(L)((Lds)&s_vb[0][0] + (x ^ 16 * (8 * v ^ ((e & 3) << 2 | e >> 2))) + (16 * k + e) * VC * 16);
        }
        if (F16) o[v] = mma(a, pl[k], o[v]);
        o[v] = mma(a, ph[k], o[v]);
        if (v == DV / 32 - 1) between(k);
      }
  };

  auto clear = [&]() {
    mx = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < DV / 32; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) o[i][r] = 0.f;
  };
  clear();
  if (tid == 0) s_bad[0] = 0x7fffffff, s_bad[1] = -1, s_bad[2] = 0;
  __syncthreads();
  bool careful = W == 2;
  if constexpr (W > 2) {
    // Tiles go from memory into LDS by themselves. Unit u is the keys of tile u and the values of tile u - LAG, LAG 1 where the
    // second product is a tile behind the first. A load of all threads covers KP (VP) tokens; a lane's piece of it lands in the
    // order of the lanes, so the lane asks for the piece that belongs there. Columns past a row's end are its first piece once
    // more (queries have zeros there, and nobody takes such outputs). Pages that are not there and, in the last tile, tokens that
    // no row sees are zeros once their place has been filled from somewhere, by the lanes that did. Keys and values that are not
    // finite show in the outputs: the rows are done again then
    constexpr int LAG = PP ? 1 : 0;
    constexpr int E = W / (int)sizeof(T), PE = VE / E;           // elements of a load, loads of a piece
    constexpr int KL = KC * PE, VL = VC * PE;                    // loads of a row
    constexpr int KP = NT / KL, VP = NT / VL, NK = TK / KP, NV = TK / VP;
    constexpr int KF = NG == 1 ? 1 : KP < 16 ? NG : NK, VF = NG == 1 ? 1 : VP < 16 ? NG : NV;  // loads that begin in groups of their own
    int pk[NG], pv[NG], pw[NG];  // the pages of unit u's keys, and of the two before
#pragma unroll
    for (int i = 0; i < NG; i++) pk[i] = pv[i] = pw[i] = -1;
    const int vk = tid / VL;
    const int kg = wave * 64 / KL / 16, vg = wave * 64 / VL / 16;  // a wave's part of a load lies in one group of 16 tokens
    auto page = [&](const int (&pg)[NG], int i, int P, int w) {
      if (NG == 1) return pg[0];
      int r = pg[i * P / 16];
#pragma unroll
      for (int x = 1; x < P / 16; x++) r = w == x ? pg[(i * P / 16 + x) % NG] : r;
      return r;
    };
    // the lane's part of load i: its token within the tile is i P + tid / L
    uint32_t ko[NK], vo[NV];
#pragma unroll
    for (int i = 0; i < NK; i++) {
      const int k = i * KP + tid / KL, x = (piece<KC>(k, tid % KL / PE) - k * KC) * VE + tid % PE * E;
      ko[i] = (uint32_t)(((NG == 1 ? k : k & 15) * c.dk + (x < c.dk ? x : 0)) * sizeof(T));
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int k = i * VP + vk, x = (piece<VC>(k, tid % VL / PE) - k * VC) * VE + tid % PE * E;
      vo[i] = (uint32_t)(((NG == 1 ? k : k & 15) * c.dv + (x < c.dv ? x : 0)) * sizeof(T));
    }
    // the next unit's pages and where its loads begin; then load i of it (of a tile before the first or past the last from some
    // page; clean() has zeros for it)
    const void *kfrom[KF], *vfrom[VF];
    auto prepare = [&](int u) {
#pragma unroll
      for (int i = 0; i < NG; i++) {
        pw[i] = pv[i], pv[i] = pk[i];
        pk[i] = u < kt1 ? page_of(u * TK + GT * i) : -1;
      }
#pragma unroll
      for (int f = 0; f < KF; f++) {
        const int i = f * (NK / KF), pg = page(pk, i, KP, kg), in = (u * TK + (NG == 1 ? 0 : i * KP / 16 + kg) * GT) & inpage;
        kfrom[f] = one(kh + (pg < 0 ? 0 : pg) * c.k_ps + in * c.dk);
      }
#pragma unroll
      for (int f = 0; f < VF; f++) {
        const int i = f * (NV / VF), pg = LAG ? page(pv, i, VP, vg) : page(pk, i, VP, vg);
        const int in = ((u - LAG) * TK + (NG == 1 ? 0 : i * VP / 16 + vg) * GT) & inpage;
        vfrom[f] = one(vh + (pg < 0 ? 0 : pg) * c.v_ps + in * c.dv);
      }
    };
    auto fire = [&](int i, int kbuf, int vbuf) {
      const int j = i < NK ? i : i - NK;
      const void *from = i < NK ? kfrom[j / (NK / KF) % KF] : vfrom[j / (NV / VF) % VF];
      const uint32_t off = i < NK ? ko[j % NK] : vo[j % NV];
      const lds_i8 *to = (const lds_i8 *)(i < NK ? (Lds)&s_kb[0][0] + kbuf * KB : (Lds)&s_vb[0][0] + vbuf * VB) + (j * NT + wave * 64) * W;
      if constexpr (V) rq_dma16s(from, off, to);
      else rq_dma4s(from, off, to);
    };
    auto issue = [&](int u, int kbuf, int vbuf) {
      prepare(u);
#pragma unroll
      for (int i = 0; i < NK + NV; i++) fire(i, kbuf, vbuf);
    };
    // A unit has landed, keys of pages pku and values of tile kt, of pages pvu: what of it has no page, or is no row's
    auto clean = [&](int kt, int kbuf, int vbuf, const int (&pku)[NG], const int (&pvu)[NG]) {
      typedef kv_vec<T, E> Part;
      const Part zero = (Part)(T)0;
      Part *kz = (Part *)&s_kb[kbuf][0] + tid, *vz = (Part *)&s_vb[vbuf][0] + tid;
      bool whole = true, seen = kt * TK + TK - 1 <= j1;
#pragma unroll
      for (int i = 0; i < NG; i++) whole = whole && pku[i] >= 0, seen = seen && pvu[i] >= 0;
      if (!whole) {
#pragma unroll
        for (int i = 0; i < NK; i++)
          if (page(pku, i, KP, kg) < 0) kz[i * NT] = zero;
      }
      if (!seen) {
#pragma unroll
        for (int i = 0; i < NV; i++)
          if (page(pvu, i, VP, vg) < 0 || kt * TK + i * VP + vk > j1) vz[i * NT] = zero;
      }
    };
    if (kt0 < kt1) {
      if constexpr (PP) {
        // Phases end with a barrier. The first group multiplies tile kt - 1's values and tile kt's scores in phase 2 kt (of
        // kt - kt0) and takes tile kt's exponentials in the next; the second does so a phase later. Unit u is read in phases 2 u and
        // 2 u + 1, so its place (u % 3) is free from phase 2 u - 4 on. Both groups ask for unit kt + 2 between the products of tile
        // kt, and have waited for theirs of unit kt + 1 at the end of them, in phase 2 (kt + 1) - 1 at the latest
        const int late = wave >> 2;
        bool was = false;
        int q = 0;  // (kt - kt0) % 3: the place of tile kt's keys and values
        auto next = [](int x, int n) { return (x + n) % 3; };
#pragma unroll
        for (int i = 0; i < 2 * ST; i++)
#pragma unroll
          for (int e = 0; e < 8; e++) ph[i][e] = pl[i][e] = (T)0;
        // tile kt0 - 1's values, which have no page and are zeros, lie in the last place
        issue(kt0, 0, 2);
        issue(kt0 + 1, 1, 0);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NK + NV) : "memory");
        clean(kt0 - 1, 0, 2, pv, pw);
        prepare(kt0 + 2);
        __syncthreads();
        if (late) __syncthreads();
        for (int kt = kt0; kt <= kt1; kt++) {
          // a tile that the wave sees nothing of has weights of 0
          const bool on = kt < kt1 && seen(kt);
          const int q1 = next(q, 1), q2 = next(q, 2);
          if (on || was) {
            values(q2, [&](int k) {
              constexpr int F = (NK + NV + 2 * ST - 1) / (2 * ST);
#pragma unroll
              for (int i = 0; i < F; i++)
                if (k * F + i < NK + NV) fire(k * F + i, q2, q1);
            });
            scores(q);
            // operands ahead of the products: 8 reads, then as many after each product as it takes
            __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
            for (int i = 0; i < 2 * ST * (DV / 32); i++) {
              __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
              __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            }
#pragma unroll
            for (int i = 0; i < ST * (DK / 16) - 8; i++) {
              __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x8, 8, 0);
          } else {
#pragma unroll
            for (int i = 0; i < NK + NV; i++) fire(i, q2, q1);
          }
          // unit kt + 1 has landed
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NK + NV) : "memory");
          clean(kt, q1, q, pv, pw);
          __syncthreads();
#pragma unroll
          for (int i = 0; i < NG; i++) pc[i] = pw[i];
          prepare(kt + 3);
          if (on) weigh(kt);
          if (was && !on) {
#pragma unroll
            for (int i = 0; i < 2 * ST; i++)
#pragma unroll
              for (int e = 0; e < 8; e++) ph[i][e] = pl[i][e] = (T)0;
          }
          was = on;
          __syncthreads();
          q = q1;
        }
        RQ_WAIT_VM(0);
        if (!late) __syncthreads();
      } else {
        int q = 0;
        issue(kt0, 0, 0);
        if (NB == 3 && kt0 + 1 < kt1) issue(kt0 + 1, 1, 1);
        for (int kt = kt0; kt < kt1; kt++) {
          if (NB == 3 && kt + 1 < kt1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NK + NV) : "memory");
          else RQ_WAIT_VM(0);
#pragma unroll
          for (int i = 0; i < NG; i++) pc[i] = NB == 3 && kt + 1 < kt1 ? pv[i] : pk[i];
          clean(kt, q, q, pc, pc);
          __syncthreads();  // the tile is there, and the one before is done with
          const int to = NB == 3 ? (q + 2) % 3 : q ^ 1;
          if (kt + NB - 1 < kt1) issue(kt + NB - 1, to, to);
          if (seen(kt)) {
            scores(q);
            weigh(kt);
            values(q, [](int) {});
          }
          q = NB == 3 ? (q + 1) % 3 : q ^ 1;
        }
      }
    }
    float odd = 0.f;
#pragma unroll
    for (int i = 0; i < DV / 32; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) odd = __builtin_fmaf(o[i][r], 0.f, odd);
    if (odd != 0.f) s_bad[2] = 1;
    __syncthreads();
    careful = s_bad[2] != 0;
  }
  if (careful) {
    // Tile by tile through registers, where what is not finite is taken out of the values, and pieces need no alignment
    clear();
    const int kk = tid / KC, kx = tid % KC, vk = tid / VC, vx = tid % VC;
    PV kn[NK], vn[NV];
    bool kin[NK], vin[NV];  // whether there is a page
    auto load = [&](int kt) {
#pragma unroll
      for (int i = 0; i < NK; i++) {
        const int j = kt * TK + i * KP + kk, pg = kv_page(c, b, j >> c.sh);
        kn[i] = kv_raw<T, VE>(kh + (pg < 0 ? 0 : pg) * c.k_ps + (j & inpage) * c.dk, kx * VE, c.dk);
        kin[i] = pg >= 0;
      }
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const int j = kt * TK + i * VP + vk, pg = kv_page(c, b, j >> c.sh);
        vn[i] = kv_raw<T, VE>(vh + (pg < 0 ? 0 : pg) * c.v_ps + (j & inpage) * c.dv, vx * VE, c.dv);
        vin[i] = pg >= 0;
      }
    };
    if (kt0 < kt1) load(kt0);
    for (int kt = kt0; kt < kt1; kt++) {
#pragma unroll
      for (int i = 0; i < NG; i++) pc[i] = page_of(kt * TK + GT * i);
#pragma unroll
      for (int i = 0; i < NK; i++) kn[i] = kv_fix<T, VE>(kn[i], kin[i] ? kx * VE : c.dk, c.dk);
#pragma unroll
      for (int i = 0; i < NV; i++) vn[i] = kv_fix<T, VE>(vn[i], vin[i] ? vx * VE : c.dv, c.dv);
      kv_vec<T, 2> mk = {(T)0, (T)0};
#pragma unroll
      for (int i = 0; i < NV; i++) kv_mark<T, VE>(vn[i], mk);
      if (mk[0] != mk[0] || mk[1] != mk[1]) {
        atomicMin(&s_bad[0], kt), atomicMax(&s_bad[1], kt);
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
          for (int e = 0; e < VE; e++) vn[i][e] = kv_finite(vn[i][e]) ? vn[i][e] : (T)0;
      }
      const int q = kt & 1;  // read until the barrier of the tile after next
#pragma unroll
      for (int i = 0; i < NK; i++) s_kb[q][piece<KC>(i * KP + kk, kx)] = kn[i];
#pragma unroll
      for (int i = 0; i < NV; i++) s_vb[q][piece<VC>(i * VP + vk, vx)] = vn[i];
      if (kt + 1 < kt1) load(kt + 1);
      __syncthreads();
      if (!seen(kt)) continue;
      scores(q);
      weigh(kt);
      values(q, [](int) {});
    }
    __syncthreads();
  }
  // values that are not finite, for the queries that see them (0 times them would reach the others)
  for (int kt = s_bad[0]; kt <= s_bad[1] && !idle; kt++) {
#pragma unroll 1
    for (int k = 0; k < TK; k++) {
      const int tk = kt * TK + k, page = page_of(tk);
      if (page < 0 || tk > see1 || tk < see0) continue;
      const long long in = ((long long)g << c.sh) + (tk & inpage);
      const T *v = (const T *)c.v + page * c.v_ps + in * c.dv, *kr = (const T *)c.k + page * c.k_ps + in * c.dk;
      bool bad = false;
      for (int col = lane; col < c.dv; col += 64) bad = bad || !kv_finite(v[col]);
      if (!__builtin_amdgcn_ballot_w64(bad)) continue;
      float x = 0.f;
#pragma unroll
      for (int d = 0; d < DK / 16; d++) {
        const FV y = kv_ld<T, 8, V>(kr, 16 * d + 8 * hi, c.dk);
#pragma unroll
        for (int e = 0; e < 8; e++) x = __builtin_fmaf((float)y[e], (float)qf[d][e], x);
      }
      x += __shfl_xor(x, 32);
      if (tk > at || tk < since || x == -INFINITY) continue;
      const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(x, p.sc, OFF - mx));
#pragma unroll
      for (int i = 0; i < DV / 32; i++) {
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const int col = 32 * i + 8 * (r >> 2) + 4 * hi + (r & 3);
          const float z = col < c.dv ? (float)v[col] : 0.f;
          if (!kv_finite(z)) o[i][r] += y * z;
        }
        asm volatile("" ::: "memory");  // no more loads than these at a time
      }
    }
  }
  l += __shfl_xor(l, 32);
  if (counts && tid == 0 && it.sp == 0) counts[((long long)b * c.Hk + g) * nrt + tile] = make_int2(it.item, it.parts);
  if (!mine) return;
  if (it.parts == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T *out = (T *)p.o + ((long long)first + tx) * p.ldo + ((long long)g * p.G + hx) * c.dv;
#pragma unroll
    for (int v = 0; v < DV / 32; v++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int col = 32 * v + 8 * i + 4 * hi;
        kv_vec<T, 4> z;
#pragma unroll
        for (int e = 0; e < 4; e++) z[e] = (T)(o[v][4 * i + e] * inv);
        if (V) {
          if (col < c.dv) *(kv_vec<T, 4> *)(out + col) = z;
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (col + e < c.dv) out[col + e] = z[e];
        }
      }
  } else {
    const long long x = (long long)it.item * MR + 32 * wave + lr;
    if (hi == 0) pml[x] = make_float2(mx, l);
    if (l != 0.f)
#pragma unroll
      for (int v = 0; v < DV / 32; v++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          *(float4 *)(part + x * DV + 32 * v + 8 * i + 4 * hi) =
              make_float4(o[v][4 * i], o[v][4 * i + 1], o[v][4 * i + 2], o[v][4 * i + 3]);
  }
}

template <typename T, int DK, int DV, int NW, int NG, int W>
__global__ __launch_bounds__(64 * NW, NW / 4) void k_kvt(KvDev c, KvaDev p, int B, int nrt, unsigned blk0, int2 *counts,
                                                         float *part, float2 *pml) {
  KvaItem it;
  if (kva_item(c, p, B, nrt, counts, 32 * NW, kva_tokens(sizeof(T) == 2, DK), blk0 + blockIdx.x, &it))
    kvt_item<T, DK, DV, NW, NG, W>(c, p, it, nrt, counts, part, pml);
}

template <typename T, int DK, int DV, int NG, int W>
int run(const KvDev &c, const KvaDev &p, const KvaPlan &r, void *work, hipStream_t s) {
  constexpr int NW = kva_waves(sizeof(T) == 2, DK);
  const long long most = bnh_most_blocks(64 * NW);
  const int B = (int)(r.units / r.nrt / c.Hk);
  for (long long b0 = 0; b0 < r.items; b0 += most) {
    const long long n = r.items - b0 < most ? r.items - b0 : most;
    hipLaunchKernelGGL((k_kvt<T, DK, DV, NW, NG, W>), dim3((unsigned)n), dim3(64 * NW), 0, s, c, p, B, r.nrt, (unsigned)b0,
                       kva_counts(r, work), kva_part(r, work), kva_ml(r, work));
    BNH_HIP(hipGetLastError());
  }
  return 0;
}
template <typename T, bool ONE, int W>
int widths(const KvDev &c, const KvaDev &p, const KvaPlan &r, void *work, hipStream_t s) {
  constexpr int NG = ONE ? 1 : kva_tokens(sizeof(T) == 2, 128) / 16;
  if (r.DK == 256) return run<T, 256, 256, ONE ? 1 : 2, W>(c, p, r, work, s);
  if (r.DK == 64) return r.D == 64 ? run<T, 64, 64, NG, W>(c, p, r, work, s) : run<T, 64, 128, NG, W>(c, p, r, work, s);
  return r.D == 64 ? run<T, 128, 64, NG, W>(c, p, r, work, s) : run<T, 128, 128, NG, W>(c, p, r, work, s);
}
template <typename T, int W>
int pages(const KvDev &c, const KvaDev &p, const KvaPlan &r, void *work, hipStream_t s) {
  return 1 << c.sh >= kva_tokens(sizeof(T) == 2, r.DK) ? widths<T, true, W>(c, p, r, work, s) : widths<T, false, W>(c, p, r, work, s);
}

}  // namespace

int kva_tiles(const KvDev &c, const KvaDev &p, const KvaPlan &r, bool f16, int w, void *work, hipStream_t s) {
  if (!f16) return w == 16 ? pages<float, 16>(c, p, r, work, s) : pages<float, 4>(c, p, r, work, s);
  if (w == 2) return widths<h16, false, 2>(c, p, r, work, s);
  return w == 16 ? pages<h16, 16>(c, p, r, work, s) : pages<h16, 4>(c, p, r, work, s);
}
