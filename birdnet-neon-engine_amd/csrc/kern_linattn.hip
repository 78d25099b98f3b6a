// Linear attention with a decay for each head (bnh_linattn): per sequence and head, over its rows t
//   S = exp(g_t) S + k_t v_t^T,  o_t = scale q_t^T S,
// S [dk][dv] in fp32.
//
// k_la_step, the recurrence itself, for sequences of few rows: bound by reading and writing the states (8 dk dv bytes a
// sequence and head, against 2 (2 dk + 2 dv) bytes a row). A block owns 4 LANES columns of one state: LANES lanes, four
// columns each (16 bytes), side by side over the 256 / LANES groups that share its rows; a thread keeps its rows' columns
// in registers over all rows of the sequence. 64 sequences of 12 heads of 128 x 128, a row each: 18.4 us (101 MB, 5.5
// TB/s: part of the states is in the last-level cache).
#include "bnh_internal.h"
#include "bnh_f16.h"

namespace {

struct LaDev {
  const void *q, *k, *v;
  void *o;
  const float *g, *s0;
  float *s1;
  const int32_t *start, *len, *slot;
  int ldq, ldk, ldv, ldo, ldg, H, rq, rk, rv, dk, dv, slots, T, rows;  // rq: heads that share a q head
  int b0;  // the launch's first sequence
  float scale;
};

// e^g of this g is 0 in 64 bits too: a row at or below it starts the state anew, whatever it holds (0 times an infinity or a
// NaN would keep it)
constexpr float kAnew = -746.f;

// sequence b's first row and its rows, cut to T and to the buffers' rows
__device__ __forceinline__ int la_rows(const LaDev &p, int b, int *first) {
  const long long s = p.start ? p.start[b] : (long long)b * p.T;
  long long n = p.len ? p.len[b] : p.T;
  n = n < p.T ? n : p.T;
  if (s < 0 || s >= p.rows) n = 0;
  else n = n < p.rows - s ? n : p.rows - s;
  *first = (int)s;
  return n < 0 ? 0 : (int)n;
}
__device__ __forceinline__ int la_slot(const LaDev &p, int b) {  // -1: none
  const int s = p.slot ? p.slot[b] : b;
  return s >= 0 && s < p.slots ? s : -1;
}

template <typename T, int LANES, int KR, bool VS>
__global__ __launch_bounds__(256) void k_la_step(LaDev p, int nsl) {
  constexpr int RG = 256 / LANES;  // row groups
  __shared__ float s_q[2][256], s_k[2][256];
  __shared__ __attribute__((aligned(16))) float s_r[2][4][4 * LANES];
  const int tid = threadIdx.x, ln = tid % LANES, rg = tid / LANES;
  const int sl = (int)(blockIdx.x % nsl), h = (int)(blockIdx.x / nsl % p.H);
  const int b = p.b0 + (int)(blockIdx.x / nsl / p.H);
  const int col = sl * 4 * LANES + 4 * ln;
  int first;
  const int n = la_rows(p, b, &first);
  const int slot = la_slot(p, b);
  const long long at = ((long long)slot * p.H + h) * p.dk * p.dv;
  float s[KR][4];
#pragma unroll
  for (int i = 0; i < KR; i++) {
    const int kk = rg + RG * i;
#pragma unroll
    for (int j = 0; j < 4; j++) s[i][j] = 0.f;
    if (p.s0 && slot >= 0 && kk < p.dk) {
      const float *q = p.s0 + at + (long long)kk * p.dv + col;
      if (VS) {
        if (col < p.dv) {
          const float4 t = *(const float4 *)q;
          s[i][0] = t.x, s[i][1] = t.y, s[i][2] = t.z, s[i][3] = t.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (col + j < p.dv) s[i][j] = q[j];
      }
    }
  }
  const int hq = h / p.rq * p.dk, hk = h / p.rk * p.dk, hv = h / p.rv * p.dv;
  for (int t = 0; t < n; t++) {
    const long long r = (long long)first + t;
    const int u = t & 1;
    if (tid < p.dk) {
      s_q[u][tid] = (float)((const T *)p.q)[r * p.ldq + hq + tid];
      s_k[u][tid] = (float)((const T *)p.k)[r * p.ldk + hk + tid];
    }
    float v[4], a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = col + j < p.dv ? (float)((const T *)p.v)[r * p.ldv + hv + col + j] : 0.f;
    const float g = p.g[r * p.ldg + h], d = expf(g);
    if (g <= kAnew) {
#pragma unroll
      for (int i = 0; i < KR; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) s[i][j] = 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KR; i++) {
      const int kk = rg + RG * i;
      if (kk >= p.dk) continue;
      const float qq = s_q[u][kk], kv = s_k[u][kk];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        s[i][j] = __builtin_fmaf(d, s[i][j], kv * v[j]);
        a[j] = __builtin_fmaf(qq, s[i][j], a[j]);
      }
    }
    // the row groups' sums: within the wave, then over the four waves
#pragma unroll
    for (int j = 0; j < 4; j++) {
#pragma unroll
      for (int m = LANES; m < 64; m *= 2) a[j] += __shfl_xor(a[j], m);
      if ((tid & 63) < LANES) s_r[u][tid >> 6][4 * ln + j] = a[j];
    }
    __syncthreads();
    if (tid < 4 * LANES && sl * 4 * LANES + tid < p.dv) {
      const float o = (s_r[u][0][tid] + s_r[u][1][tid]) + (s_r[u][2][tid] + s_r[u][3][tid]);
      ((T *)p.o)[r * p.ldo + (long long)h * p.dv + sl * 4 * LANES + tid] = (T)(p.scale * o);
    }
  }
  if (!p.s1 || slot < 0) return;
#pragma unroll
  for (int i = 0; i < KR; i++) {
    const int kk = rg + RG * i;
    if (kk >= p.dk) continue;
    float *q = p.s1 + at + (long long)kk * p.dv + col;
    if (VS) {
      if (col < p.dv) *(float4 *)q = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (col + j < p.dv) q[j] = s[i][j];
    }
  }
}

template <typename T, int LANES, bool VS>
int step_run(LaDev d, int B, hipStream_t s) {
  constexpr int RG = 256 / LANES;
  const int nsl = (int)bnh_ceil_div(d.dv, 4 * LANES), kr = (int)bnh_ceil_div(d.dk, RG);
  const int most = (int)(bnh_most_blocks(256) / ((long long)nsl * d.H));  // sequences; H <= 2^16, dv <= 2^8: 16 at least
  for (long long b0 = 0; b0 < B; b0 += most) {
    d.b0 = (int)b0;
    const dim3 grid((unsigned)((long long)nsl * d.H * (B - b0 < most ? B - b0 : most))), block(256);
#define GO(KR) hipLaunchKernelGGL((k_la_step<T, LANES, KR, VS>), grid, block, 0, s, d, nsl)
    if (kr <= 256 / RG / 4) GO(256 / RG / 4);
    else if (kr <= 256 / RG / 2) GO(256 / RG / 2);
    else GO(256 / RG);
#undef GO
    BNH_HIP(hipGetLastError());
  }
  return 0;
}

// Columns to a block: 128, or 32 where 128 leave compute units without one (or dv has no more). Eight rows of 12 heads of
// 128 x 128: one sequence 20.3 us with 128, 13.0 with 32; 64 sequences 35 and 53.
template <typename T>
int step_go(const LaDev &d, int B, bool vs, hipStream_t s) {
  if (d.dv <= 32 || (long long)B * d.H * bnh_ceil_div(d.dv, 128) < 256)
    return vs ? step_run<T, 8, true>(d, B, s) : step_run<T, 8, false>(d, B, s);
  return vs ? step_run<T, 32, true>(d, B, s) : step_run<T, 32, false>(d, B, s);
}

// The chunked form, for sequences of many rows. Over a chunk of C rows with the running sums c_i of g within it:
//   o_i = scale (e^{c_i} q_i^T S + sum_{j <= i} e^{c_i - c_j} (q_i . k_j) v_j^T),
//   S <- e^{c_C} S + sum_j e^{c_C - c_j} k_j v_j^T,
// four matrix products on MFMA. Every exponent is a sum of g over the rows in between, at most 0 where g is, so nothing is
// divided by a small decay; c is kept in 64 bits because differences of its values matter where c itself has grown
// large, and g below -1e4 (whose e^g is 0) counts as -1e4, so that a reset's infinity does not cancel another's.
//
// A block of four or eight waves owns 64 or 128 columns of one state over one piece of one sequence. The state stays in the
// accumulators of the waves (16 columns each, all of dk): their layout is, for pairs of 16-row tiles, that of the first operand
// of the product with q's rows, so it never passes through LDS. q, k and v of the next chunk are loaded into registers while this
// one's are multiplied out of LDS; k's and v's transposes come out of LDS through ds_read_b64_tr_b16.
//
// fp16 rows: the factors of a product have to be fp16, its sums are fp32. Scores, the state and what is added to it go in as
// two fp16 parts each, 22 bits, against the exact v, q and k. Scores are scaled row by row and the state column by column by
// powers of two first (their largest to 2^12..2^13), so neither overflows. The state itself is not rounded: its update takes
// v_j e^{c_C - c_j}, the largest of the chunk's by column scaled to 2^14..2^15 (the state's own unit from then on). With one
// part for scores and state the outputs' relative error was 2.9e-4 instead of the 2.1e-4 of fp16 outputs as such, and several
// times the outputs' own rounding where their terms cancel; the second parts cost 17 us of the 141 below, and 12 of the 136.
// fp32 rows run on the fp32 MFMA, unscaled and unsplit.
//
// 12 heads of 128 x 128 in fp16: 17,280 rows of one sequence 136 us (21 pieces of 13 chunks: what the pieces add 38, the
// join 10, the outputs 89; 214 MB would take 42), 24 sequences of up to 720 rows 141 us. A chunk takes a block 12,000 to
// 13,000 cycles, 2,000 of them on the matrix cores: its phases (scores, state product, update, outputs) wait on LDS and on
// each other, with two waves a SIMD at 210 registers; four waves of 128 registers spill and take 1.5 times as long. The
// blocks of an XCD are neighbours in the sequences' order (bnh_xcd_block): with sequences of unequal lengths that lie sorted,
// as in the second of these, the XCD of the longest has 23 chunks one after another where an even spread would have 12.
//
// A row's v that is not finite would reach earlier rows of its chunk as 0 x inf; it is taken out of the product and added to
// the rows that see it one by one (a wave that finds none skips this). A row that starts the state anew (e^g is 0) takes
// what was before it times 0; where the state or a row of such a chunk is not finite, the chunk ends ahead of that row, and
// the next one begins with it and no state.

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v8f __attribute__((ext_vector_type(8)));
typedef h16 v8h __attribute__((ext_vector_type(8)));
typedef h16 v4h __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));

// A fragment: 8 of the 32 steps of a product for row (or column) lane & 15, the same 8 of both operands in a lane
template <typename T>
struct Frag;
template <>
struct Frag<h16> {
  typedef v8h V;   // a fragment
  typedef v4h H;   // four values
};
template <>
struct Frag<float> {
  typedef v8f V;
  typedef v4f H;
};
__device__ __forceinline__ v4f mma(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4f mma(v8f a, v8f b, v4f c) {
#pragma unroll
  for (int e = 0; e < 8; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}
// steps 8 q + e (q = lane >> 4) of a row at p = its step 8 q
template <typename T>
__device__ __forceinline__ typename Frag<T>::V row8(const T *p) {
  return *(const typename Frag<T>::V *)p;
}
// steps 4 q + e and 16 + 4 q + e of a row at p = its step 4 q
template <typename T>
__device__ __forceinline__ typename Frag<T>::V row44(const T *p) {
  const typename Frag<T>::H a = *(const typename Frag<T>::H *)p, b = *(const typename Frag<T>::H *)(p + 16);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
// the same steps of column lane & 15 of a matrix at p whose rows (a step each) are `ld` apart: a group of 16 lanes reads 4
// rows of 16 values and gets them by column; rows an odd number of 32 bytes apart fall on different banks
__device__ __forceinline__ v8h col44(const h16 *p, int ld, int lane) {
  const h16 *a = p + (4 * (lane >> 4) + ((lane & 15) >> 2)) * ld + 4 * (lane & 3);
  typedef __attribute__((address_space(3))) v4s L;
  const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L *)a), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L *)(a + 16 * ld));
  typedef short v8s __attribute__((ext_vector_type(8)));
  const v8s z = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(v8h, z);
}
__device__ __forceinline__ v8f col44(const float *p, int ld, int lane) {
  v8f r;
#pragma unroll
  for (int e = 0; e < 8; e++) r[e] = p[(4 * (lane >> 4) + e + (e < 4 ? 0 : 12)) * ld + (lane & 15)];
  return r;
}
// 2^-e that takes a largest value m to 2^12..2^13: 0 and infinities are left as they are, and nothing grows past 2^126
__device__ __forceinline__ int scale_exp(float m) {
  const int e = (int)(__float_as_uint(m) >> 23 & 255) - 127 - 12;
  return m == 0.f || e > 127 - 12 ? 0 : e < -126 ? -126 : e;
}

// 16 bytes of a row of `cols` values from its value c, zeros past the end; V: all of them are in or out, 16-byte aligned
template <typename T, bool V>
__device__ __forceinline__ uint4 row16(const T *p, int c, int cols) {
  constexpr int VE = 16 / sizeof(T);
  uint4 r = make_uint4(0, 0, 0, 0);
  if (V) {
    if (c < cols) r = *(const uint4 *)(p + c);
  } else if (c + VE <= cols) {
    __builtin_memcpy(&r, p + c, 16);
  } else if (c < cols) {
    T t[VE] = {};
#pragma unroll
    for (int i = 0; i < VE; i++)
      if (c + i < cols) t[i] = p[c + i];
    __builtin_memcpy(&r, t, 16);
  }
  return r;
}

// One piece of one sequence by NW waves, 16 of the state's columns each. OUT: the outputs, from the state before the piece,
// and s1 from the sequence's last; else the state that every piece but the last adds (the first one's includes s0), into
// part, and its whole decay. s1 may lie over s0, and the output launch's blocks run in any order: the launch before it keeps
// the state before the first piece in part's last place, and a first piece that is not also the last starts from there.
// fp32 rows of dk up to 64 are held to registers of which two blocks of eight waves fit a compute unit (8 sequences of up to
// 500 rows, 16 heads of 64 x 97: 73 us, 88 with one).
template <typename T, int DKT, int NW, int C, bool V, bool OUT>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 4 && DKT <= 2 ? 4 : 1) void k_la_chunk(LaDev p, int nsl, int npc, int pcr,
                                                                                          float *part, float *pdec) {
  constexpr bool F16 = sizeof(T) == 2;
  constexpr int VE = 16 / sizeof(T), KD = 32 * DKT, DV = 16 * NW, NT = 64 * NW, SQ = KD + VE, SP = C + VE;
  constexpr int SK = KD + (F16 ? 16 : 4), SV = DV + (F16 ? 16 : 4);
  constexpr int RK = NT * VE / KD, RV = NT * VE / DV;                          // rows that one load of all threads covers
  constexpr int NK = C / RK > 0 ? C / RK : 1, NV = C / RV > 0 ? C / RV : 1;
  typedef typename Frag<T>::V FV;
  typedef typename Frag<T>::H FH;
  __shared__ __attribute__((aligned(16))) T s_q[OUT ? C * SQ : 1], s_k[C * SK], s_v[C * SV], s_p[2][OUT ? C * SP : 1],
      s_l[2][OUT && F16 ? C * SP : 1];                         // F16: the scores' second parts
  __shared__ double s_c[2][64];                              // c_i
  __shared__ __attribute__((aligned(16))) float s_w[2][64];  // e^{c_C - c_j}
  __shared__ float s_e[2][64], s_d[2];                       // e^{c_i}; e^{c_C}
  __shared__ int s_x[2][2][64];                              // the scores' scale by step of 32 columns and row
  __shared__ int s_bad;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, q4 = lane >> 4;
  unsigned lb = bnh_xcd_block(blockIdx.x, gridDim.x);
  const int sl = (int)(lb % nsl), h = (int)(lb / nsl % p.H);
  lb /= nsl * p.H;
  const int pc = (int)(lb % (OUT ? npc : npc - 1)), b = p.b0 + (int)(lb / (OUT ? npc : npc - 1));
  int first;
  const int n = la_rows(p, b, &first), slot = la_slot(p, b);
  const int r0 = pc * pcr;
  if (OUT ? pc > 0 && r0 >= n : r0 + pcr >= n) return;  // no such piece, or a last one, whose state nobody takes
  const int rows = n - r0 < pcr ? n - r0 : pcr;         // of this piece; 0: only a state to copy
  const int c0 = sl * DV + wave * 16;                   // this wave's columns
  const long long pst = ((((long long)b * p.H + h) * nsl + sl) * npc) * (KD * DV);  // this state's pieces
  const long long at = ((long long)slot * p.H + h) * p.dk * p.dv;

  v4f S[2 * DKT];     // times 2^ux: rows 16 t + 4 q4 + r, column c0 + lr
  int ux = 0;
  float most = 0.f;   // F16: no finite value of the column is larger
#pragma unroll
  for (int t = 0; t < 2 * DKT; t++) S[t] = (v4f){0.f, 0.f, 0.f, 0.f};
  const bool keep = p.s0 && p.s1 && slot >= 0 && n > pcr;  // another block than the first piece's stores s1
  if (OUT && (pc > 0 || keep)) {
    const float *w = part + pst + (long long)(pc > 0 ? pc - 1 : npc - 1) * (KD * DV) + wave * (KD * 16) + 4 * lane;
#pragma unroll
    for (int t = 0; t < 2 * DKT; t++) S[t] = *(const v4f *)(w + 256 * t);
  } else if (pc == 0 && p.s0 && slot >= 0) {
#pragma unroll
    for (int t = 0; t < 2 * DKT; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int kk = 16 * t + 4 * q4 + r, col = c0 + lr;
        if (kk < p.dk && col < p.dv) S[t][r] = p.s0[at + (long long)kk * p.dv + col];
      }
  }
  if (!OUT && keep && pc == 0) {
    float *w = part + pst + (long long)(npc - 1) * (KD * DV) + wave * (KD * 16) + 4 * lane;
#pragma unroll
    for (int t = 0; t < 2 * DKT; t++) *(v4f *)(w + 256 * t) = S[t];
  }
  if (F16) {
#pragma unroll
    for (int t = 0; t < 2 * DKT; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) most = fmaxf(most, S[t][r] - S[t][r] == 0.f ? fabsf(S[t][r]) : 0.f);
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
  }
  if (OUT) {  // the blocks right of the diagonal that a step of 32 reads
    for (int i = tid; i < C / 32 * 256; i += NT)
      s_p[0][(i / 256 * 32 + i % 256 / 16) * SP + i / 256 * 32 + 16 + i % 16] =
          s_p[1][(i / 256 * 32 + i % 256 / 16) * SP + i / 256 * 32 + 16 + i % 16] = (T)0.f;
    if (F16)
      for (int i = tid; i < C / 32 * 256; i += NT)
        s_l[0][(i / 256 * 32 + i % 256 / 16) * SP + i / 256 * 32 + 16 + i % 16] =
            s_l[1][(i / 256 * 32 + i % 256 / 16) * SP + i / 256 * 32 + 16 + i % 16] = (T)0.f;
  }

  const int kr = tid / (KD / VE), kc = tid % (KD / VE) * VE, vr = tid / (DV / VE), vc = tid % (DV / VE) * VE;
  const int vcols = p.dv - sl * DV;
  const T *qp = (const T *)p.q + ((long long)first + r0) * p.ldq + h / p.rq * p.dk;
  const T *kp = (const T *)p.k + ((long long)first + r0) * p.ldk + h / p.rk * p.dk;
  const T *vp = (const T *)p.v + ((long long)first + r0) * p.ldv + h / p.rv * p.dv + sl * DV;
  uint4 qn[OUT ? NK : 1], kn[NK], vn[NV];
  // the chunk from row t0 into registers. V: rows and columns outside come from a row and a column inside, and put() has
  // zeros for them; no load waits on a branch
  auto load = [&](int t0) {
    if (t0 >= rows) return;
#pragma unroll
    for (int i = 0; i < NK; i++) {
      const int r = t0 + kr + RK * i;
      if (V) {
        const int rc = r < rows ? r : rows - 1, cc = kc < p.dk ? kc : 0;
        if (OUT) qn[i] = *(const uint4 *)(qp + (long long)rc * p.ldq + cc);
        kn[i] = *(const uint4 *)(kp + (long long)rc * p.ldk + cc);
      } else {
        if (OUT) qn[i] = r < rows ? row16<T, false>(qp + (long long)r * p.ldq, kc, p.dk) : make_uint4(0, 0, 0, 0);
        kn[i] = r < rows ? row16<T, false>(kp + (long long)r * p.ldk, kc, p.dk) : make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int r = t0 + vr + RV * i;
      if (V) vn[i] = *(const uint4 *)(vp + (long long)(r < rows ? r : rows - 1) * p.ldv + (vc < vcols ? vc : 0));
      else vn[i] = r < rows ? row16<T, false>(vp + (long long)r * p.ldv, vc, vcols) : make_uint4(0, 0, 0, 0);
    }
  };
  auto put = [&](int t0) {
    if (V && (t0 + C > rows || p.dk < KD || vcols < DV)) {
#pragma unroll
      for (int i = 0; i < NK; i++) {
        const bool in = t0 + kr + RK * i < rows && kc < p.dk;
        if (OUT && !in) qn[i] = make_uint4(0, 0, 0, 0);
        if (!in) kn[i] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < NV; i++)
        if (t0 + vr + RV * i >= rows || vc >= vcols) vn[i] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < NK; i++) {
      if (RK > C && kr >= C) break;
      if (OUT) *(uint4 *)(s_q + (kr + RK * i) * SQ + kc) = qn[i];
      *(uint4 *)(s_k + (kr + RK * i) * SK + kc) = kn[i];
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
      if (RV > C && vr >= C) break;
      *(uint4 *)(s_v + (vr + RV * i) * SV + vc) = vn[i];
    }
  };
  // c of the chunk from row t0 and what follows from it, by the last wave (every wave has g, for the rows that start the state
  // anew); rows past the end count as g = 0
  double ctot = 0, cpre = 0;  // with and without the chunk's
  bool anew = false;          // a row of the piece starts the state anew
  float gn = 0.f;
  auto gload = [&](int t0) {
    gn = 0.f;
    if (lane < C && t0 + lane < rows) gn = p.g[((long long)first + r0 + t0 + lane) * p.ldg + h];
  };
  auto sums = [&](int u) {
    double c = gn < -1e4f ? -1e4f : gn;
#pragma unroll
    for (int d = 1; d < C; d *= 2) {
      const double o = __shfl_up(c, d);
      c = lane >= d ? c + o : c;
    }
    const double last = __shfl(c, C - 1);
    const float w = expf((float)(last - c));
    if (lane < C) {
      s_c[u][lane] = c;
      s_e[u][lane] = expf((float)c);
      s_w[u][lane] = w;
      if (lane == C - 1) s_d[u] = expf((float)c);
    }
    cpre = ctot;
    ctot += last;
  };
  // The rows to take of the chunk in qn, kn and vn, of which `at` start the state anew: all of it where everything is
  // finite, else what lies ahead of such a row
  auto rows_to_new = [&](int t0, int u, uint64_t at) {
    bool bad = !(gn <= kAnew) && gn - gn != 0.f;
    auto odd = [&](uint4 x) {
      T y[VE];
      __builtin_memcpy(y, &x, 16);
#pragma unroll
      for (int e = 0; e < VE; e++) bad = bad || y[e] - y[e] != (T)0.f;
    };
#pragma unroll
    for (int i = 0; i < NK; i++)
      if (t0 + kr + RK * i < rows && kc < p.dk) odd(kn[i]);
#pragma unroll
    for (int i = 0; i < NV; i++)
      if (t0 + vr + RV * i < rows && vc < vcols) odd(vn[i]);
#pragma unroll
    for (int t = 0; t < 2 * DKT; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) bad = bad || S[t][r] - S[t][r] != 0.f;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    if (bad) s_bad = 1;
    __syncthreads();
    if (!s_bad) return C;
    if (at & 1) {
      most = 0.f;
#pragma unroll
      for (int t = 0; t < 2 * DKT; t++) S[t] = (v4f){0.f, 0.f, 0.f, 0.f};
    }
    const uint64_t next = at & ~1ull;
    const int len = next ? __builtin_ctzll(next) : C;
#pragma unroll
    for (int i = 0; i < NK; i++)
      if (kr + RK * i >= len) kn[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < NV; i++)
      if (vr + RV * i >= len) vn[i] = make_uint4(0, 0, 0, 0);
    if (wave == NW - 1) {
      ctot = at & 1 ? 0 : cpre;
      if (lane >= len || (lane == 0 && (at & 1))) gn = 0.f;
      sums(u);
    }
    return len;
  };

  load(0);
  gload(0);
  if (wave == NW - 1) sums(0);
  int u = 0, end;
  for (int t0 = 0; t0 < rows; t0 = end, u ^= 1) {
    const uint64_t at = __builtin_amdgcn_ballot_w64(gn <= kAnew);
    end = t0 + C;
    if (at) {
      anew = true;
      end = t0 + rows_to_new(t0, u, at);
    }
    put(t0);
    __syncthreads();
    load(end);
    gload(end);

    if constexpr (OUT) {  // scores of 16 rows and 32 columns a unit, a row a lane and four columns in each block of 16
      constexpr int UN = C == 64 ? 6 : 2;
#pragma unroll 1
      for (int un = wave; un < UN; un += NW) {
        const int ib = C == 64 ? 0x021233 >> 4 * un & 15 : 1 - un, jj = C == 64 ? 0x010010 >> 4 * un & 15 : 0;
        const int i = 16 * ib + lr;
        const bool two = 2 * jj + 1 <= ib;  // the second block is not all right of the diagonal
        const double ci = s_c[u][i];
        v4f a[2] = {(v4f){0.f, 0.f, 0.f, 0.f}, (v4f){0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int d = 0; d < DKT; d++) {
          const FV x = row8<T>(s_q + i * SQ + 32 * d + 8 * q4);
          a[0] = mma(row8<T>(s_k + (32 * jj + lr) * SK + 32 * d + 8 * q4), x, a[0]);
          a[1] = mma(row8<T>(s_k + (32 * jj + 16 + lr) * SK + 32 * d + 8 * q4), x, a[1]);
        }
        float m = 0.f;
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const int j = 32 * jj + 16 * c + 4 * q4 + r;
            a[c][r] = j <= i ? a[c][r] * __expf((float)(ci - s_c[u][j])) : 0.f;
            m = fmaxf(m, fabsf(a[c][r]));
          }
        float dn = 1.f;
        uint64_t keep = ~0ull;  // an infinity has no second part, nor has its row
        if (F16) {
          m = fmaxf(m, __shfl_xor(m, 16));
          m = fmaxf(m, __shfl_xor(m, 32));
          keep = m - m == 0.f ? ~0ull : 0;
          const int x = scale_exp(m);
          dn = ldexpf(1.f, -x);
          if (q4 == 0) s_x[u][jj][i] = x;
        }
#pragma unroll
        for (int c = 0; c < 2; c++) {
          FH y, z;
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const float x = F16 ? a[c][r] * dn : a[c][r];
            y[r] = (T)x;
            if (F16) z[r] = (T)(x - (float)y[r]);
          }
          if (c == 0 || two) {
            *(FH *)(s_p[u] + i * SP + 32 * jj + 16 * c + 4 * q4) = y;
            if constexpr (F16)
              *(uint64_t *)(s_l[u] + i * SP + 32 * jj + 16 * c + 4 * q4) = __builtin_bit_cast(uint64_t, z) & keep;
          }
        }
      }
    }
    if (wave == NW - 1 && end < rows) sums(u ^ 1);
    FV vf[C / 32];
#pragma unroll
    for (int j = 0; j < C / 32; j++) vf[j] = col44(s_v + 32 * j * SV + wave * 16, SV, lane);
    // whether a value of v is not finite
    bool odd = false;
    if constexpr (F16) {
      typedef unsigned short u2 __attribute__((ext_vector_type(2)));
      u2 m = {0, 0};
#pragma unroll
      for (int j = 0; j < C / 32; j++)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const u2 x = {(unsigned short)(hbits(vf[j][e]) & 0x7fff), (unsigned short)(hbits(vf[j][e + 1]) & 0x7fff)};
          m = __builtin_elementwise_max(m, x);
        }
      odd = m[0] >= 0x7c00 || m[1] >= 0x7c00;
    } else {
#pragma unroll
      for (int j = 0; j < C / 32; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) odd = odd || vf[j][e] - vf[j][e] != 0.f;
    }
    odd = __builtin_amdgcn_ballot_w64(odd) != 0;
    // the state's part of the outputs, before the state moves on
    v4f a[C / 16];
    float xs[4];  // 2^x of the accumulators' columns 4 q4 + r
    if constexpr (OUT) {
      float dn = 1.f;
      uint32_t keep = ~0u;
      if (F16) {
        float m = 0.f;
#pragma unroll
        for (int t = 0; t < 2 * DKT; t++)
#pragma unroll
          for (int r = 0; r < 4; r++) m = fmaxf(m, fabsf(S[t][r]));
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        const int x = scale_exp(m);
        keep = m - m == 0.f ? ~0u : 0;
        const float up = ldexpf(1.f, x + ux);
        dn = ldexpf(1.f, -x);
#pragma unroll
        for (int r = 0; r < 4; r++) xs[r] = __shfl(up, 4 * q4 + r);
      }
#pragma unroll
      for (int ib = 0; ib < C / 16; ib++) a[ib] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < DKT; d++) {
        FV sf, sl, x[C / 16];
#pragma unroll
        for (int ib = 0; ib < C / 16; ib++) x[ib] = row44<T>(s_q + (16 * ib + lr) * SQ + 32 * d + 4 * q4);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float y = F16 ? S[2 * d + e / 4][e % 4] * dn : S[2 * d + e / 4][e % 4];
          sf[e] = (T)y;
          if (F16) sl[e] = (T)(y - (float)sf[e]);
        }
#pragma unroll
        for (int ib = 0; ib < C / 16; ib++) a[ib] = mma(sf, x[ib], a[ib]);
        if constexpr (F16) {
          typedef uint32_t u4 __attribute__((ext_vector_type(4)));
          sl = __builtin_bit_cast(FV, __builtin_bit_cast(u4, sl) & (u4){keep, keep, keep, keep});
#pragma unroll
          for (int ib = 0; ib < C / 16; ib++) a[ib] = mma(sl, x[ib], a[ib]);
        }
      }
    }
    // the state's update
    FV hi[C / 32], lo[C / 32];
    float dec = s_d[u];
    if constexpr (F16) {
      float y[C / 32][8], m = 0.f;  // v_j e^{c_C - c_j}; the largest of the column
#pragma unroll
      for (int j = 0; j < C / 32; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          y[j][e] = __builtin_fmaf((float)vf[j][e], s_w[u][32 * j + 4 * q4 + e + (e < 4 ? 0 : 12)], 0.f);
          m = fmaxf(m, fabsf(y[j][e]));
        }
      m = fmaxf(m, __shfl_xor(m, 16));
      m = fmaxf(m, __shfl_xor(m, 32));
      // k is below 2^16. The state in its unit stays below 2^126, whatever it came with
      most = __builtin_fmaf(m, 65536.f * C, fmaxf(most * dec, 0.f));
      const int e = (int)(__float_as_uint(m) >> 23 & 255) - 127, low = (int)(__float_as_uint(most) >> 23 & 255) - 127 - 125;
      int x = m == 0.f ? ux : e > 127 ? 0 : e - 14;  // the largest to 2^14..2^15
      x = x > low ? x : low;
      dec = ldexpf(dec, ux - x);
      ux = x;
#pragma unroll
      for (int j = 0; j < C / 32; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float z = ldexpf(y[j][e], -x);
          hi[j][e] = (T)z;
          lo[j][e] = (T)(z - (float)hi[j][e]);
        }
    } else {
#pragma unroll
      for (int j = 0; j < C / 32; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) hi[j][e] = (T)((float)vf[j][e] * s_w[u][32 * j + 4 * q4 + e + (e < 4 ? 0 : 12)]);
    }
    if (F16 && odd) {  // an infinity has no second part
#pragma unroll
      for (int j = 0; j < C / 32; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) lo[j][e] = hi[j][e] - hi[j][e] == (T)0.f ? lo[j][e] : (T)0.f;
    }
    // two tiles of the state's rows at a time, whose sums do not wait on each other
#pragma unroll
    for (int t = 0; t < 2 * DKT; t += 2) {
      FV kf[2][C / 32];
#pragma unroll
      for (int g = 0; g < 2; g++) {
#pragma unroll
        for (int j = 0; j < C / 32; j++) kf[g][j] = col44(s_k + 32 * j * SK + 16 * (t + g), SK, lane);
#pragma unroll
        for (int r = 0; r < 4; r++) S[t + g][r] *= dec;
      }
#pragma unroll
      for (int j = 0; j < C / 32; j++) {
        if (F16)
#pragma unroll
          for (int g = 0; g < 2; g++) S[t + g] = mma(kf[g][j], lo[j], S[t + g]);
#pragma unroll
        for (int g = 0; g < 2; g++) S[t + g] = mma(kf[g][j], hi[j], S[t + g]);
      }
    }
    __syncthreads();  // the scores are there, and this chunk's q, k and v are free
    if constexpr (OUT) {
      if (odd) {  // v without what is not finite, which the rows that see it get below
#pragma unroll
        for (int j = 0; j < C / 32; j++)
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const T y = vf[j][e];
            vf[j][e] = y - y == (T)0.f ? y : (T)0.f;
            hi[j][e] = y - y == (T)0.f ? (T)0.f : y;
          }
      }
#pragma unroll
      for (int ib = 0; ib < C / 16; ib++) {  // the state's part and each step of 32 columns have a unit of their own
        const int i = 16 * ib + lr;
        const float ec = s_e[u][i];
        v4f y0 = mma(vf[0], row44<T>(s_p[u] + i * SP + 4 * q4), (v4f){0.f, 0.f, 0.f, 0.f});
        if (F16) y0 = mma(vf[0], row44<T>(s_l[u] + i * SP + 4 * q4), y0);
        const float u0 = F16 ? ldexpf(1.f, s_x[u][0][i]) : 1.f;
        if (C == 64 && ib >= 2) {
          v4f y1 = mma(vf[C / 32 - 1], row44<T>(s_p[u] + i * SP + 32 + 4 * q4), (v4f){0.f, 0.f, 0.f, 0.f});
          if (F16) y1 = mma(vf[C / 32 - 1], row44<T>(s_l[u] + i * SP + 32 + 4 * q4), y1);
          const float u1 = F16 ? ldexpf(1.f, s_x[u][1][i]) : 1.f;
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const float y = F16 ? __builtin_fmaf(y1[r], u1, y0[r] * u0) : y0[r] + y1[r];
            a[ib][r] = p.scale * __builtin_fmaf(F16 ? a[ib][r] * xs[r] : a[ib][r], ec, y);
          }
        } else {
#pragma unroll
          for (int r = 0; r < 4; r++)
            a[ib][r] = p.scale * __builtin_fmaf(F16 ? a[ib][r] * xs[r] : a[ib][r], ec, F16 ? y0[r] * u0 : y0[r]);
        }
      }
      if (odd) {
#pragma unroll
        for (int j = 0; j < C / 32; j++)
#pragma unroll
          for (int e = 0; e < 8; e++)
#pragma unroll 1
            for (int q = 0; q < 4; q++) {
              const int jr = 32 * j + 4 * q + e + (e < 4 ? 0 : 12);
              float y[4];
#pragma unroll
              for (int r = 0; r < 4; r++) y[r] = __shfl((float)hi[j][e], 16 * q + 4 * q4 + r);
#pragma unroll
              for (int ib = 2 * j; ib < C / 16; ib++) {
                const int i = 16 * ib + lr;
                if (jr > i) continue;
                const float x = p.scale * ldexpf((float)s_p[u][i * SP + jr], F16 ? s_x[u][j][i] : 0);
#pragma unroll
                for (int r = 0; r < 4; r++)
                  if (y[r] != 0.f) a[ib][r] += x * y[r];
              }
            }
      }
#pragma unroll
      for (int ib = 0; ib < C / 16; ib++) {
        const int i = 16 * ib + lr, col = c0 + 4 * q4;
        if (t0 + i >= rows || t0 + i >= end) continue;
        T *o = (T *)p.o + ((long long)first + r0 + t0 + i) * p.ldo + (long long)h * p.dv + col;
        FH y;
#pragma unroll
        for (int r = 0; r < 4; r++) y[r] = (T)a[ib][r];
        if (V) {
          if (col < p.dv) *(FH *)o = y;
        } else {
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (col + r < p.dv) o[r] = y[r];
        }
      }
    }
  }
  if (F16) {
    const float up = ldexpf(1.f, ux);
#pragma unroll
    for (int t = 0; t < 2 * DKT; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) S[t][r] *= up;
  }
  if (!OUT) {
    float *w = part + pst + (long long)pc * (KD * DV) + wave * (KD * 16) + 4 * lane;
#pragma unroll
    for (int t = 0; t < 2 * DKT; t++) *(v4f *)(w + 256 * t) = S[t];
    if (wave == NW - 1 && lane == 0)
      pdec[(((long long)b * p.H + h) * nsl + sl) * (npc - 1) + pc] = anew ? -1.f : expf((float)ctot);
  } else if (p.s1 && slot >= 0 && r0 + pcr >= n) {
#pragma unroll
    for (int t = 0; t < 2 * DKT; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int kk = 16 * t + 4 * q4 + r, col = c0 + lr;
        if (kk < p.dk && col < p.dv) p.s1[at + (long long)kk * p.dv + col] = S[t][r];
      }
  }
}

// The states before each piece from what the pieces add: part[i] <- part[i] + pdec[i] part[i - 1], in order, four values
// a thread; a pdec below 0 is a piece that starts the state anew
__global__ __launch_bounds__(256) void k_la_scan(LaDev p, int npc, int pcr, int quads, int nsl, float *part,
                                                 const float *pdec) {
  const int st = (int)(blockIdx.y), b = st / (nsl * p.H);
  int first;
  const int n = la_rows(p, b, &first);
  const int np = (n + pcr - 1) / pcr - 1;  // pieces whose state a later one takes
  const int i = (int)(blockIdx.x * 256 + threadIdx.x);
  if (i >= quads || np < 2) return;
  float4 *w = (float4 *)(part + (long long)st * npc * 4 * quads) + i;
  const float *d = pdec + (long long)st * (npc - 1);
  float4 s = w[0];
  for (int k = 1; k < np; k++) {
    const float4 x = w[(long long)k * quads];
    const float y = d[k];
    s = y < 0.f ? x : make_float4(__builtin_fmaf(y, s.x, x.x), __builtin_fmaf(y, s.y, x.y), __builtin_fmaf(y, s.z, x.z),
                                  __builtin_fmaf(y, s.w, x.w));
    w[(long long)k * quads] = s;
  }
}

// How a call is cut: dk and dv in tiles, and rows in pieces
struct Plan {
  bool chunk;
  int dkt, nw, c, nsl, npc, pcr;
  long long states, floats;  // of a state
};
Plan plan(const bnh_la *p, int T, int B) {
  Plan r;
  // the recurrence takes a row at a time, 2.3 us each for 64 sequences of 12 heads of 128 x 128 (T 8: 35 us, T 12: 45) and
  // 1.2 for 8 or fewer (14 and 19); the first chunk costs 43 and 13 whatever its rows
  r.chunk = T > 8;
  r.dkt = p->dk <= 32 ? 1 : p->dk <= 64 ? 2 : p->dk <= 128 ? 4 : 8;
  r.nw = p->dv > 64 ? 8 : 4;
  r.c = p->f16 ? 64 : 32;
  r.nsl = (int)bnh_ceil_div(p->dv, 16 * r.nw);
  r.states = (long long)B * p->H * r.nsl;
  r.floats = 32LL * r.dkt * 16 * r.nw;
  r.npc = 1;
  r.pcr = T;
  if (r.chunk) {
    // pieces for about as many blocks as the card holds at once (one a compute unit where a block's registers and LDS take half
    // of it or more), rounded up to a whole number for each state
    long long want = bnh_ceil_div(p->f16 && r.dkt >= 4 ? 256 : 512, r.states);
    const long long most = bnh_ceil_div(T, 4 * r.c);
    if (want > most) want = most;
    r.pcr = (int)bnh_round_up(bnh_ceil_div(T, want), r.c);
    r.npc = (int)bnh_ceil_div(T, r.pcr);
  }
  return r;
}
size_t plan_bytes(const Plan &r) {
  if (r.npc < 2) return 0;
  // what each piece but the last adds and the state before the first, then the pieces' decays
  return (size_t)(bnh_round_up(4 * r.states * r.npc * r.floats, 256) + bnh_round_up(4 * r.states * (r.npc - 1), 256));
}

template <typename T, int DKT, int NW, int C, bool V>
int chunk_run(LaDev d, const Plan &r, int B, void *work, hipStream_t s) {
  float *part = (float *)work;
  float *pdec = part ? (float *)((char *)work + bnh_round_up(4 * r.states * r.npc * r.floats, 256)) : nullptr;
  const dim3 block(64 * NW);
  if (r.npc > 1) {
    hipLaunchKernelGGL((k_la_chunk<T, DKT, NW, C, V, false>), dim3((unsigned)(r.states * (r.npc - 1))), block, 0, s, d, r.nsl,
                       r.npc, r.pcr, part, pdec);
    BNH_HIP(hipGetLastError());
    if (r.npc > 2) {
      const int quads = (int)(r.floats / 4);
      hipLaunchKernelGGL(k_la_scan, dim3((unsigned)bnh_ceil_div(quads, 256), (unsigned)r.states), dim3(256), 0, s, d, r.npc,
                         r.pcr, quads, r.nsl, part, pdec);
      BNH_HIP(hipGetLastError());
    }
  }
  // sequences a launch; those in pieces are far fewer (states of 512 blocks at most), and go in one
  const long long per = (long long)r.nsl * d.H * r.npc;
  const int most = (int)(bnh_most_blocks(64 * NW) / per);
  for (long long b0 = 0; b0 < B; b0 += most) {
    d.b0 = (int)b0;
    hipLaunchKernelGGL((k_la_chunk<T, DKT, NW, C, V, true>), dim3((unsigned)(per * (B - b0 < most ? B - b0 : most))), block, 0,
                       s, d, r.nsl, r.npc, r.pcr, part, pdec);
    BNH_HIP(hipGetLastError());
  }
  return 0;
}
template <typename T, int NW, int C, bool V>
int chunk_dk(const LaDev &d, const Plan &r, int B, void *work, hipStream_t s) {
  if (r.dkt == 1) return chunk_run<T, 1, NW, C, V>(d, r, B, work, s);
  if (r.dkt == 2) return chunk_run<T, 2, NW, C, V>(d, r, B, work, s);
  if (r.dkt == 4) return chunk_run<T, 4, NW, C, V>(d, r, B, work, s);
  return chunk_run<T, 8, NW, C, V>(d, r, B, work, s);
}
template <typename T, int C>
int chunk_go(const LaDev &d, const Plan &r, int B, bool v, void *work, hipStream_t s) {
  if (r.nw == 8) return v ? chunk_dk<T, 8, C, true>(d, r, B, work, s) : chunk_dk<T, 8, C, false>(d, r, B, work, s);
  return v ? chunk_dk<T, 4, C, true>(d, r, B, work, s) : chunk_dk<T, 4, C, false>(d, r, B, work, s);
}

int la_check(const bnh_la *p, int T, int B) {
  BNH_REQ(p && T > 0 && T <= (1 << 30) && B > 0 && p->H > 0 && p->Hq > 0 && p->Hk > 0 && p->Hv > 0);
  BNH_REQ(p->H % p->Hq == 0 && p->H % p->Hk == 0 && p->H % p->Hv == 0);
  BNH_REQ(p->dk > 0 && p->dk <= 256 && p->dv > 0 && p->dv <= 256 && (p->f16 == 0 || p->f16 == 1));
  BNH_REQ((long long)B * p->H < (1LL << 24) && p->H <= 65536);
  return 0;
}

}  // namespace

extern "C" {

size_t bnh_linattn_work_bytes(const bnh_la *p, int T, int B) {
  if (la_check(p, T, B)) return 0;
  return plan_bytes(plan(p, T, B));
}

int bnh_linattn(const bnh_la *p, int T, int B, int rows, const int32_t *start, const int32_t *len, void *work,
                size_t work_bytes, void *stream) {
  if (la_check(p, T, B)) return -1;
  BNH_REQ(p->q && p->k && p->v && p->o && p->g && rows > 0 && p->slots >= 0);
  BNH_REQ(start || (long long)T * B <= rows);
  BNH_REQ(p->ldq >= p->Hq * p->dk && p->ldk >= p->Hk * p->dk && p->ldv >= p->Hv * p->dv && p->ldo >= p->H * p->dv);
  BNH_REQ(p->ldg == 0 || p->ldg >= p->H);
  BNH_REQ(p->slot || p->slots >= B || (!p->s0 && !p->s1));
  const size_t es = p->f16 ? 2 : 4;
  auto on = [](const void *q, size_t a) { return (uintptr_t)q % a == 0; };
  BNH_REQ(on(p->q, es) && on(p->k, es) && on(p->v, es) && on(p->o, es) && on(p->g, 4) && on(p->s0, 4) && on(p->s1, 4));
  BNH_REQ(on(p->slot, 4) && on(start, 4) && on(len, 4));
  LaDev d = {p->q, p->k, p->v, p->o, p->g, p->s0, p->s1, start, len, p->slot, p->ldq, p->ldk, p->ldv, p->ldo, p->ldg,
             p->H, p->H / p->Hq, p->H / p->Hk, p->H / p->Hv, p->dk, p->dv, p->slots, T, rows, 0, p->scale};
  const bool vs = p->dv % 4 == 0 && on(p->s0, 16) && on(p->s1, 16);
  hipStream_t s = bnh_stream(stream);
  const Plan r = plan(p, T, B);
  if (r.chunk) {
    const size_t need = plan_bytes(r);
    BNH_REQ(need == 0 || (work && on(work, 16) && work_bytes >= need));
    BNH_REQ(r.states * r.npc < (1LL << 31) && (r.npc < 3 || r.states < 65536));
    const int ve = 16 / (int)es;
    const bool v = on(p->q, 16) && on(p->k, 16) && on(p->v, 16) && on(p->o, 16) && p->ldq % ve == 0 && p->ldk % ve == 0 &&
                   p->ldv % ve == 0 && p->ldo % ve == 0 && p->dk % ve == 0 && p->dv % ve == 0;
    return p->f16 ? chunk_go<h16, 64>(d, r, B, v, work, s) : chunk_go<float, 32>(d, r, B, v, work, s);
  }
  return p->f16 ? step_go<h16>(d, B, vs, s) : step_go<float>(d, B, vs, s);
}

}  // extern "C"
