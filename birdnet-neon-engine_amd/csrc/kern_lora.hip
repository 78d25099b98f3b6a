// A shared fp16 projection with low-rank adapters of many requests beside it (bnh_pw_lora):
//   out = act(W x + bias + s_j B_j (A_j x)) (+ res), j the adapter of the row's window.
//
// Two launches. k_lora_down computes t = s_j A_j x for every row with an adapter, as two fp16 parts (22 bits): factors that
// the matrix instruction of the second product takes. A row's t is scaled by a power of two first (its largest to 2^14..2^15),
// so that it keeps them whatever its size; the row's product takes the unit back in fp32. Up to 16 ranks both parts fit
// one matrix instruction, against b's ranks twice; more ranks take each product again (4,096 rows, 1,536 x 1,536, rank 64 63 us,
// 57 with one part). k_lora_gemm computes W x on fp16 MFMA with fp32 sums and adds the product
// of t with the adapter's B to the sums it has, so that the adapter costs no pass over the output. Rows of one matrix
// instruction are independent of each other, so a block of 16 rows whose adapters differ multiplies all of them by each of
// the adapters in it and every row keeps its own: nothing of another request's adapter, not even an infinity or a NaN,
// reaches it. Up to 64 rows, where w's bytes are the bound, k_lora_few computes slices of K beside the first products and
// k_lora_few_out adds them up.
//
// Measured: 17,280 rows, K 1,536, N 6,144, rank 16 of 24 stations in 394 to 450 us by the card's clock (419: 0.79 PFLOP/s; a
// library product of the same size without adapters 350): k_lora_down 18, the rest k_lora_gemm, of which the adapters'
// products, an idx, t and b read a tile, are about 15 (394 with adapters and 361 without, on one card). 24 rows of 24
// stations, 1,536 x 1,536: 7.1 us and 6.1, the latencies of two short launches (w is 1 us).
#include <type_traits>

#include "bnh_internal.h"
#include "bnh_f16.h"
#include "bnh_lds_dma.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef h16 v8h __attribute__((ext_vector_type(8)));

// eight halves from p, of which the first n are inside; V: all or none of them are, and p is 16-byte aligned
template <bool V>
__device__ __forceinline__ v8h ld8(const uint16_t *p, int n) {
  v8h r = {};
  if (V) {
    if (n > 0) r = *(const v8h *)p;
  } else if (n >= 8) {
    __builtin_memcpy(&r, p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 7; i++)
      if (i < n) r[i] = hfrom(p[i]);
  }
  return r;
}
__device__ __forceinline__ v4f mma(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// f(0) ... f(N - 1), each with its index as a constant: accumulators indexed by it stay in registers
template <int N, typename F>
__device__ __forceinline__ void each(F f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

struct LoraDev {
  const uint16_t *x, *w, *a, *b;
  const float *bias, *scale;
  const int32_t *idx;
  uint16_t *t;
  float *u;  // the unit of each row of t
  long long x_ws;
  int lda, ldw, M, N, K, n, r, half, r32;  // t's row: r32 values, its first parts from 0 and its second ones from half
  bool line;                         // x's windows follow each other: rows lda apart throughout
  long long rows;
  double rM;
};

__device__ __forceinline__ int lora_id(const LoraDev &p, int win) {  // -1: none
  const int j = p.idx[win];
  return j >= 0 && j < p.n ? j : -1;
}

// t of the 16 rows from 16 tile for the which-th different adapter among them; the block's four waves take every fourth
// step of 32 of K. RT: 16-column tiles of half a row of t; s: 768 RT floats of LDS
template <int RT, bool V>
__device__ __forceinline__ void lora_down(const LoraDev &p, long long tile, unsigned which, float *s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, kc = (lane >> 4) * 8;
  const long long row = tile * 16 + lr < p.rows ? tile * 16 + lr : p.rows - 1;
  const int win = bnh_div(row, p.M, p.rM);
  const int id = lora_id(p, win);
  // the first rows of the different adapters, and of those the one that is asked for
  bool dup = false;
#pragma unroll
  for (int j = 0; j < 15; j++) {
    const int o = __builtin_amdgcn_readlane(id, j);
    dup = dup || (j < lr && o == id);
  }
  uint32_t lead = (uint32_t)(__builtin_amdgcn_ballot_w64(lane < 16 && !dup && id >= 0));
  for (unsigned i = 0; i < which; i++) lead &= lead - 1;
  if (!lead) return;
  const int j = __builtin_amdgcn_readlane(id, __builtin_ctz(lead));
  const uint16_t *xp = p.x + win * p.x_ws + (long long)(row - (long long)win * p.M) * p.lda + kc;
  const uint16_t *ap[RT];
#pragma unroll
  for (int t = 0; t < RT; t++)  // past the last rank: any row, whose results are not kept
    ap[t] = p.a + ((long long)j * p.r + (16 * t + lr < p.r ? 16 * t + lr : p.r - 1)) * p.K + kc;
  v4f acc[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) acc[t] = (v4f){0.f, 0.f, 0.f, 0.f};
  int k = 32 * wave;
#pragma unroll 4
  for (; k + 32 <= p.K; k += 128) {
    const v8h x = ld8<V>(xp + k, 8);
#pragma unroll
    for (int t = 0; t < RT; t++) acc[t] = mma(x, ld8<V>(ap[t] + k, 8), acc[t]);
  }
  if (k < p.K) {
    const v8h x = ld8<V>(xp + k, p.K - k - kc);
#pragma unroll
    for (int t = 0; t < RT; t++) acc[t] = mma(x, ld8<V>(ap[t] + k, p.K - k - kc), acc[t]);
  }
  if (wave) {
#pragma unroll
    for (int t = 0; t < RT; t++) *(v4f *)(s + ((wave - 1) * RT + t) * 256 + 4 * lane) = acc[t];
  }
  __syncthreads();
  if (wave) return;
  const float sc = p.scale ? p.scale[j] : 1.f;
  v4f most = {0.f, 0.f, 0.f, 0.f};  // of each of the lane's four rows
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const float *q = s + t * 256 + 4 * lane;
    acc[t] += *(const v4f *)q + (*(const v4f *)(q + RT * 256) + *(const v4f *)(q + 2 * RT * 256));
#pragma unroll
    for (int e = 0; e < 4; e++) {
      acc[t][e] *= sc;
      if (16 * t + lr < p.r) most[e] = fmaxf(most[e], fabsf(acc[t][e]));
    }
  }
#pragma unroll
  for (int e = 0; e < 4; e++) {
#pragma unroll
    for (int d = 1; d < 16; d *= 2) most[e] = fmaxf(most[e], __shfl_xor(most[e], d));
    const int m = 4 * (lane >> 4) + e, rid = __shfl(id, m);
    const long long r = tile * 16 + m;
    if (r >= p.rows || rid != j) continue;
    const int x = most[e] == 0.f || most[e] - most[e] != 0.f ? 0 : (int)(__float_as_uint(most[e]) >> 23) - 127 - 14;
    if (lr == 0) p.u[r] = ldexpf(1.f, x);
#pragma unroll
    for (int t = 0; t < RT; t++) {
      const int c = 16 * t + lr;
      if (c >= p.half) continue;
      const float y = c < p.r ? ldexpf(acc[t][e], -x) : 0.f;
      const h16 hi = (h16)y;
      p.t[r * p.r32 + c] = hbits(hi);
      p.t[r * p.r32 + p.half + c] = hbits(y - y == 0.f ? (h16)(y - (float)hi) : (h16)0.f);
    }
  }
}
template <int RT, bool V>
__global__ __launch_bounds__(256) void k_lora_down(LoraDev p, long long tile0) {
  __shared__ __attribute__((aligned(16))) float s[768 * RT];
  lora_down<RT, V>(p, tile0 + blockIdx.x, blockIdx.y, s);
}

__device__ __forceinline__ float lora_act(float y, int act) {
  if (act == 1) return y * __builtin_amdgcn_rcpf(1.f + __expf(-y));
  return act == 2 ? bnh_relu_f32(y) : y;
}

struct EpiDev {
  int act, ldo, ldr;
  uint16_t *out;
  const uint16_t *res;
  long long out_ws, res_ws;
  bool line;  // so do the windows of out and res
};
// row r of rows ld apart in windows of M rows ws apart
__device__ __forceinline__ long long lora_row(const LoraDev &p, bool line, long long r, long long ws, int ld) {
  if (line) return r * ld;
  const int w = bnh_div(r, p.M, p.rM);
  return w * ws + (r - (long long)w * p.M) * ld;
}

// Up to 64 rows: bound by reading w. The first nd blocks compute t (as k_lora_down), the others the shared product of all
// rows with 32 channels over one of `ks` slices of K, into part [ks][rows][Np]; k_lora_few_out adds the slices and the
// adapters' products. RW: 16-row tiles.
template <int RT, int RW, bool V>
__global__ __launch_bounds__(256) void k_lora_few(LoraDev p, int nd, int dy, int nn, int ks, int Np, float *part) {
  constexpr int LF = RT > 2 * RW ? 768 * RT : 768 * 2 * RW;
  __shared__ __attribute__((aligned(16))) float s[LF];
  if ((int)blockIdx.x < nd) {
    lora_down<RT, V>(p, blockIdx.x / dy, blockIdx.x % dy, s);
    return;
  }
  const int blk = (int)blockIdx.x - nd, sl = blk / nn, n0 = blk % nn * 32;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, kc = (lane >> 4) * 8;
  const uint16_t *xp[RW], *wp[2];
#pragma unroll
  for (int i = 0; i < RW; i++) {
    const int row = 16 * i + lr < p.rows ? 16 * i + lr : (int)p.rows - 1;
    const int w = row / p.M;
    xp[i] = p.x + w * p.x_ws + (long long)(row - w * p.M) * p.lda + kc;
  }
#pragma unroll
  for (int j = 0; j < 2; j++) wp[j] = p.w + (long long)(n0 + 16 * j + lr < p.N ? n0 + 16 * j + lr : p.N - 1) * p.ldw + kc;
  v4f acc[2][RW];
#pragma unroll
  for (int j = 0; j < 2; j++)
#pragma unroll
    for (int i = 0; i < RW; i++) acc[j][i] = (v4f){0.f, 0.f, 0.f, 0.f};
  int k = 32 * (4 * sl + wave);
#pragma unroll 4
  for (; k + 32 <= p.K; k += 128 * ks) {
    const v8h w0 = ld8<V>(wp[0] + k, 8), w1 = ld8<V>(wp[1] + k, 8);
#pragma unroll
    for (int i = 0; i < RW; i++) {
      const v8h x = ld8<V>(xp[i] + k, 8);
      acc[0][i] = mma(w0, x, acc[0][i]);
      acc[1][i] = mma(w1, x, acc[1][i]);
    }
  }
  if (k < p.K) {
    const v8h w0 = ld8<V>(wp[0] + k, p.K - k - kc), w1 = ld8<V>(wp[1] + k, p.K - k - kc);
#pragma unroll
    for (int i = 0; i < RW; i++) {
      const v8h x = ld8<V>(xp[i] + k, p.K - k - kc);
      acc[0][i] = mma(w0, x, acc[0][i]);
      acc[1][i] = mma(w1, x, acc[1][i]);
    }
  }
  if (wave) {
#pragma unroll
    for (int i = 0; i < 2 * RW; i++) *(v4f *)(s + ((wave - 1) * 2 * RW + i) * 256 + 4 * lane) = acc[i / RW][i % RW];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int i = 0; i < 2 * RW; i++) {
    const float *q = s + i * 256 + 4 * lane;
    const v4f y = acc[i / RW][i % RW] + (*(const v4f *)q + (*(const v4f *)(q + 512 * RW) + *(const v4f *)(q + 1024 * RW)));
    const int row = 16 * (i % RW) + lr, n = n0 + 16 * (i / RW) + (lane >> 4) * 4;
    if (row < p.rows && n < p.N) *(v4f *)(part + ((long long)sl * p.rows + row) * Np + n) = y;  // Np: N rounded up to 4
  }
}
// four channels of one row a thread
template <bool VR, bool VO>
__global__ __launch_bounds__(256) void k_lora_few_out(LoraDev p, EpiDev e, int ks, int Np, const float *part) {
  const int i = (int)(blockIdx.x * 256 + threadIdx.x), nq = Np / 4;
  const int row = i / nq, n = i % nq * 4;
  if (row >= p.rows) return;
  const int w = row / p.M, m = row - w * p.M;
  const int id = p.idx ? lora_id(p, w) : -1;
  v4f y = (v4f){0.f, 0.f, 0.f, 0.f}, u = y;
#pragma unroll 4
  for (int k = 0; k < ks; k++) y += *(const v4f *)(part + ((long long)k * p.rows + row) * Np + n);
  if (id >= 0) {
    const uint16_t *t = p.t + (long long)row * p.r32, *b = p.b + ((long long)id * p.N + n) * p.r;
    for (int k = 0; k < p.r; k += 8) {
      const v8h x = *(const v8h *)(t + k), xl = *(const v8h *)(t + p.half + k);
#pragma unroll
      for (int c = 0; c < 4; c++) {
        if (n + c >= p.N) continue;
        const v8h z = ld8<VR>(b + (long long)c * p.r + k, p.r - k);
#pragma unroll
        for (int l = 0; l < 8; l++) u[c] = __builtin_fmaf((float)x[l] + (float)xl[l], (float)z[l], u[c]);
      }
    }
    const float un = p.u[row];
#pragma unroll
    for (int c = 0; c < 4; c++) y[c] = __builtin_fmaf(u[c], un, y[c]);
  }
  uint16_t *o = e.out + w * e.out_ws + (long long)m * e.ldo + n;
  const uint16_t *rs = e.res ? e.res + w * e.res_ws + (long long)m * e.ldr + n : nullptr;
  typedef h16 v4h __attribute__((ext_vector_type(4)));
  v4h z = {}, q;
  if (VO && rs) z = *(const v4h *)rs;
#pragma unroll
  for (int c = 0; c < 4; c++) {
    if (!VO && n + c >= p.N) continue;
    if (!VO && rs) z[c] = hfrom(rs[c]);
    const float v = lora_act(y[c] + (p.bias ? p.bias[n + c] : 0.f), e.act);
    q[c] = (h16)(rs ? v + (float)z[c] : v);
    if (!VO) o[c] = hbits(q[c]);
  }
  if (VO) *(v4h *)o = q;
}

// The tile of rows [r0, ...) x channels [n0, ...) of logical block lb: blocks that follow each other (and so run under one
// XCD's L2) form groups of 8 row tiles that share their channels' weights
__device__ __forceinline__ void lora_tile(unsigned lb, int nm, int nn, int *tm, int *tn) {
  const unsigned g = lb / (8u * nn), i = lb % (8u * nn);
  const unsigned gm = nm - 8 * g < 8 ? nm - 8 * g : 8;
  *tm = (int)(8 * g + i % gm);
  *tn = (int)(i / gm);
}

// BM rows x BN channels a block of WM x WN waves. The operands' steps of BK values of K (a 128-byte line of each row: half
// lines cost twice the L2 reads) pass through a ring of LDS stages that global loads fill directly (DMA: rows that are
// 16-byte aligned), with one barrier a step; the loads are issued between the products, not in one go ahead of the
// LDS reads. Without DMA through registers into two stages. A row's 16-byte chunks lie in LDS at chunk ^ f(row), so that the
// 16 rows of a fragment's read fall on different banks (the loads write 16 bytes a lane in lane order, so the lane's chunk of the
// row is permuted instead). The first operand of the matrix instruction is the weights': a lane's accumulators are
// four channels of one row.
template <int BM, int BN, int WM, int WN, int BK, int RING, bool DMA, bool VR, bool VO>
__global__ __launch_bounds__(64 * WM * WN) void k_lora_gemm(LoraDev p, EpiDev e, int tm0, int nm, int nn) {
  constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, CH = BK / 8, RPI = 64 / CH;
  constexpr int NL = (BM + BN) * CH / 64 / NW, ST = DMA ? RING : 2, SH = (BM + BN) * BK;  // loads a wave; stages, their halves
  constexpr int XS = 16 * TN + 4;                                                   // an exchange row, floats
  static_assert((BM + BN) * CH % (64 * NW) == 0 && BM % RPI == 0, "");
  constexpr int LDS = ST * SH * 2 > NW * 16 * XS * 4 ? ST * SH * 2 : NW * 16 * XS * 4;
  __shared__ __attribute__((aligned(16))) char s_raw[LDS];
  uint16_t *s = (uint16_t *)s_raw;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, q4 = lane >> 4;
  int tm, tn;
  lora_tile(bnh_xcd_block(blockIdx.x, gridDim.x), nm, nn, &tm, &tn);
  const long long r0 = (long long)(tm0 + tm) * BM;
  const int n0 = tn * BN;
  auto fx = [](int row) { return CH == 4 ? (row >> 2) & 3 : (row >> 1) & 7; };

  // this lane's chunks of a step: load i of the wave fills LDS rows (i NW + wave) RPI ..., x's first and then w's
  static_assert(NW * RPI % 16 == 0, "fx is the same for every load of a lane");
  const int gk = (lane % CH ^ fx(wave * RPI + lane / CH)) * 8;
  const uint16_t *gp[NL];
#pragma unroll
  for (int i = 0; i < NL; i++) {
    const int row = (i * NW + wave) * RPI + lane / CH;
    if (row < BM) {
      const long long r = r0 + row < p.rows ? r0 + row : p.rows - 1;
      gp[i] = p.x + lora_row(p, p.line, r, p.x_ws, p.lda) + gk;
    } else {
      const int n = n0 + row - BM < p.N ? n0 + row - BM : p.N - 1;
      gp[i] = p.w + (long long)n * p.ldw + gk;
    }
  }
  v4f acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; j++)
#pragma unroll
    for (int i = 0; i < TM; i++) acc[j][i] = (v4f){0.f, 0.f, 0.f, 0.f};
  const int wm = wave / WN * (TM * 16), wn = wave % WN * (TN * 16);
  int id[TM];  // the adapters of the wave's rows, row lr of each tile of 16; looked at when the products are done
  each<TM>([&](auto tile) {
    constexpr int i = decltype(tile)::value;
    const long long row = r0 + wm + 16 * i + lr < p.rows ? r0 + wm + 16 * i + lr : p.rows - 1;
    id[i] = p.idx ? p.idx[bnh_div(row, p.M, p.rM)] : -1;
  });
  // the adapters' operands: values k to k + 31 of t of the wave's rows, and b of the first adapter among them for their ranks
  const int rank = p.half == 16 ? 8 * (q4 & 1) : 8 * q4;  // half is 16 or a multiple of 32
  uint32_t bp[TN];  // into an adapter's b: N < 2^24, r <= 2^8
#pragma unroll
  for (int j = 0; j < TN; j++)
    bp[j] = (uint32_t)(n0 + wn + 16 * j + lr < p.N ? n0 + wn + 16 * j + lr : p.N - 1) * (uint32_t)p.r + (uint32_t)rank;
  v8h ax[TM], bn[TN];
  float un[TM];
  uint32_t todo[TM];
  int next = -1;
  auto pick = [&](int k) {  // the next adapter of a row that has not had its own, -1 when all have; its b on the way
    next = -1;
    each<TM>([&](auto tile) {
      constexpr int i = decltype(tile)::value;
      if (next < 0 && todo[i]) next = __builtin_amdgcn_readlane(id[i], __builtin_ctz(todo[i]));
    });
    if (next >= 0) {
      const int from = k < p.half ? k : k - p.half;
      each<TM>([&](auto tile) {
        constexpr int i = decltype(tile)::value;
        todo[i] &= ~(uint32_t)__builtin_amdgcn_ballot_w64(lane < 16 && id[i] == next);
      });
#pragma unroll
      for (int j = 0; j < TN; j++) bn[j] = ld8<VR>(p.b + (long long)next * p.N * p.r + from + bp[j], p.r - from - rank);
    }
  };
  auto ahead = [&](int k) {
    each<TM>([&](auto tile) {
      constexpr int i = decltype(tile)::value;
      if (id[i] >= p.n) id[i] = -1;
      todo[i] = (uint32_t)__builtin_amdgcn_ballot_w64(lane < 16 && id[i] >= 0);
      const long long row = r0 + wm + 16 * i + lr < p.rows ? r0 + wm + 16 * i + lr : p.rows - 1;
      ax[i] = *(const v8h *)(p.t + row * p.r32 + 8 * q4 + k);
      un[i] = p.u[row];
    });
    pick(k);
  };
  struct Ops {
    v8h x[TM], w[TN];
  };
  auto read = [&](const uint16_t *st, int k, Ops &o) {  // the 32 values of K from 32 k of a stage
    const int c = ((4 * k + q4) ^ fx(lr)) * 8;
#pragma unroll
    for (int j = 0; j < TN; j++) o.w[j] = *(const v8h *)(st + (BM + wn + 16 * j + lr) * BK + c);
#pragma unroll
    for (int i = 0; i < TM; i++) o.x[i] = *(const v8h *)(st + (wm + 16 * i + lr) * BK + c);
  };
  auto multiply = [&](const Ops &o, auto between) {  // between(i): after the products of row tile i
    each<TM>([&](auto tile) {
      constexpr int i = decltype(tile)::value;
#pragma unroll
      for (int j = 0; j < TN; j++) acc[j][i] = mma(o.w[j], o.x[i], acc[j][i]);
      between(i);
    });
  };
  auto nothing = [](int) {};
  auto step = [&](const uint16_t *st) {
#pragma unroll
    for (int k = 0; k < BK / 32; k++) {
      Ops o;
      read(st, k, o);
      multiply(o, nothing);
    }
  };
  auto put = [&](uint16_t *st, const v8h *v) {
#pragma unroll
    for (int i = 0; i < NL; i++) *(v8h *)(st + (i * NW + wave) * 512 + lane * 8) = v[i];
  };
  const int full = p.K / BK;
  if constexpr (DMA) {
    auto issue = [&](int t, int stage, int from, int to) {
#pragma unroll
      for (int i = 0; i < NL; i++)
        if (i >= from && i < to)
          rq_dma16((const int8_t *)(gp[i] + (long long)t * BK), (const lds_i8 *)(s + stage * SH + (i * NW + wave) * 512));
    };
    static_assert((ST == 2 || (ST == 3 && NL == 4)) && BK == 64, "the waits and halves below");
    // step t's stage is full, and every read of step t - 1's, which the next loads take, is done
    auto turn = [&](int t) {
      if (ST == 2 || t + 1 >= full) RQ_WAIT_VM(0);
      else RQ_WAIT_VM(4);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      RQ_BARRIER();
    };
    for (int t = 0; t < ST - 1 && t < full; t++) issue(t, t, 0, NL);
    int at = 0;
    if constexpr (ST == 2) {
      constexpr int PG = (NL + TM - 1) / TM;  // loads a row tile, so that they do not queue up ahead of the reads
      for (int t = 0; t < full; t++) {
        turn(t);
        if (t + 1 == full && p.r32) ahead(0);  // nothing else is on its way now
        Ops o;
        read(s + at * SH, 0, o);
        __builtin_amdgcn_sched_barrier(0);
        multiply(o, [&](int i) { if (t + 1 < full) issue(t + 1, at ^ 1, PG * i, PG * i + PG); });
        read(s + at * SH, 1, o);
        multiply(o, nothing);
        at ^= 1;
      }
    } else {
      for (int t = 0; t < full; t++) {
        turn(t);
        if (t + 1 == full && p.r32) ahead(0);
        if (t + 2 < full) issue(t + 2, at ? at - 1 : ST - 1, 0, NL);
        step(s + at * SH);
        at = at + 1 < ST ? at + 1 : 0;
      }
    }
  } else {
    v8h v[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) v[i] = ld8<false>(gp[i], p.K - gk);
    for (int t = 0; t < full; t++) {
      put(s + (t & 1) * SH, v);
      const int k = (t + 1) * BK;
#pragma unroll
      for (int i = 0; i < NL; i++)
        if (k + gk < p.K) v[i] = ld8<false>(gp[i] + k, p.K - k - gk);
      __syncthreads();
      step(s + (t & 1) * SH);
    }
  }
  if (full * BK < p.K) {  // the last values of K, zeros past them
    v8h v[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) v[i] = ld8<DMA>(gp[i] + full * BK, p.K - full * BK - gk);
    __syncthreads();
    put(s, v);
    __syncthreads();
    step(s);
  }
  __syncthreads();

  // The adapters: one of those among the wave's rows a turn, its b read once for all of them while the one before is
  // multiplied. Every row takes the product in its unit or keeps what it has, so that one request's infinities stay its own.
  for (int k = 0; k < p.r32; k += 32) {
    if (k || !DMA || full == 0) ahead(k);
    while (next >= 0) {
      const int a = next;
      v8h b[TN];
#pragma unroll
      for (int j = 0; j < TN; j++) b[j] = bn[j];
      pick(k);
      each<TM>([&](auto tile) {
        constexpr int i = decltype(tile)::value;
        if (__builtin_amdgcn_ballot_w64(lane < 16 && id[i] == a)) {
#pragma unroll
          for (int j = 0; j < TN; j++) {
            const v4f u = mma(b[j], ax[i], (v4f){0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int q = 0; q < 4; q++) acc[j][i][q] = id[i] == a ? __builtin_fmaf(u[q], un[i], acc[j][i][q]) : acc[j][i][q];
          }
        }
      });
    }
  }
  float *xch = (float *)s_raw + wave * 16 * XS;
  float bias[TN][4];
#pragma unroll
  for (int j = 0; j < TN; j++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int n = n0 + wn + 16 * j + 4 * q4 + r;
      bias[j][r] = p.bias && n < p.N ? p.bias[n] : 0.f;
    }
  each<TM>([&](auto tile) {
    constexpr int i = decltype(tile)::value;
    const long long rb = r0 + wm + 16 * i;
    if (rb >= p.rows) return;
#pragma unroll
    for (int j = 0; j < TN; j++) {
      v4f y;
#pragma unroll
      for (int r = 0; r < 4; r++) y[r] = lora_act(acc[j][i][r] + bias[j][r], e.act);
      *(v4f *)(xch + lr * XS + 16 * j + 4 * q4) = y;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    // eight channels a lane where rows are aligned, else one: 64 lanes side by side along the row either way
    constexpr int VC = VO ? 8 : 1, LPR = 16 * TN / VC;  // lanes to a row
#pragma unroll
    for (int h = 0; h < 16 * LPR; h += 64) {
      const int m = (h + lane) / LPR, c = (h + lane) % LPR * VC, n = n0 + wn + c;
      const long long r = rb + m;
      if (m >= 16 || r >= p.rows || n >= p.N) continue;
      const float *y = xch + m * XS + c;
      uint16_t *o = e.out + lora_row(p, e.line, r, e.out_ws, e.ldo) + n;
      const uint16_t *rs = e.res ? e.res + lora_row(p, e.line, r, e.res_ws, e.ldr) + n : nullptr;
      if constexpr (VO) {
        v8h z = {};
        if (rs) z = *(const v8h *)rs;
        v8h t;
#pragma unroll
        for (int k = 0; k < 8; k++) t[k] = (h16)(rs ? y[k] + (float)z[k] : y[k]);
        *(v8h *)o = t;
      } else {
        *o = hbits((h16)(rs ? *y + (float)hfrom(*rs) : *y));
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  });
}

// ALL: for rows, ranks and outputs of every alignment, else for aligned ones alone
template <int BM, int BN, int WM, int WN, int BK, int RING, bool ALL>
int lora_tiles(const LoraDev &p, const EpiDev &d, bool v, bool vr, bool vo, hipStream_t s) {
  const long long nm = bnh_ceil_div(p.rows, BM), nn = bnh_ceil_div(p.N, BN);
  const long long most = bnh_most_blocks(64 * WM * WN) / nn;  // N < 2^24: 16 at least
  const dim3 block(64 * WM * WN);
  for (long long m0 = 0; m0 < nm; m0 += most) {
    const int n = (int)(nm - m0 < most ? nm - m0 : most);
    const dim3 grid((unsigned)(n * nn));
#define GO(V, VR, VO) \
  hipLaunchKernelGGL((k_lora_gemm<BM, BN, WM, WN, BK, RING, V, VR, VO>), grid, block, 0, s, p, d, (int)m0, n, (int)nn)
    if constexpr (ALL) {
      if (v && vr && vo) GO(true, true, true);
      else if (v && vo) GO(true, false, true);
      else if (v) GO(true, false, false);
      else if (vo) GO(false, false, true);
      else GO(false, false, false);
    } else {
      GO(true, true, true);
    }
#undef GO
    BNH_HIP(hipGetLastError());
  }
  return 0;
}
// Rows up to which the few-row form runs, for its four row tiles: 32 rows, 1,536 x 1,536 12.8 us and 25.8 on the tiles; 64 rows,
// 1,536 x 6,144 19.9 and 26.2; 64 rows, 1,536 x 1,536 14.6, and 66 rows on the tiles 24.0. Where it would stop being the
// faster one has not been measured: it is still ahead at 64.
constexpr long long few = 64;
// slices of K of the few-row form: two blocks a compute unit, and a step of 32 a wave at least
long long few_slices(int N, int K) {
  const long long want = bnh_ceil_div(512, bnh_ceil_div(N, 32)), most = bnh_ceil_div(K, 128);
  return want < most ? want : most;
}
int lora_half(int r) { return r == 0 ? 0 : r <= 16 ? 16 : (int)bnh_round_up(r, 32); }
long long lora_t_bytes(long long rows, int r) { return bnh_round_up(rows * 2 * lora_half(r) * 2, 256); }
long long lora_tu_bytes(long long rows, int r) { return lora_t_bytes(rows, r) + (r ? bnh_round_up(rows * 4, 256) : 0); }

int lora_few(const LoraDev &p, const EpiDev &d, int dy, bool v, bool vr, bool vo, void *work, hipStream_t s) {
  const int Np = (int)bnh_round_up(p.N, 4), nn = (int)bnh_ceil_div(p.N, 32), ks = (int)few_slices(p.N, p.K);
  const int nd = dy * (int)bnh_ceil_div(p.rows, 16);
  float *part = (float *)((char *)work + lora_tu_bytes(p.rows, p.r));
  const dim3 grid((unsigned)(nd + nn * ks)), block(256);
#define GO2(RT, RW)                                                                                            \
  do {                                                                                                         \
    if (v) hipLaunchKernelGGL((k_lora_few<RT, RW, true>), grid, block, 0, s, p, nd, dy, nn, ks, Np, part);     \
    else hipLaunchKernelGGL((k_lora_few<RT, RW, false>), grid, block, 0, s, p, nd, dy, nn, ks, Np, part);      \
  } while (0)
#define GO(RW)                       \
  do {                               \
    if (p.r <= 16) GO2(1, RW);       \
    else if (p.r <= 64) GO2(4, RW);  \
    else GO2(16, RW);                \
  } while (0)
  if (p.rows <= 16) GO(1);
  else if (p.rows <= 32) GO(2);
  else GO(4);
#undef GO
#undef GO2
  BNH_HIP(hipGetLastError());
  const dim3 og((unsigned)bnh_ceil_div(p.rows * (Np / 4), 256));
  if (vr && vo) hipLaunchKernelGGL((k_lora_few_out<true, true>), og, block, 0, s, p, d, ks, Np, part);
  else if (vr) hipLaunchKernelGGL((k_lora_few_out<true, false>), og, block, 0, s, p, d, ks, Np, part);
  else if (vo) hipLaunchKernelGGL((k_lora_few_out<false, true>), og, block, 0, s, p, d, ks, Np, part);
  else hipLaunchKernelGGL((k_lora_few_out<false, false>), og, block, 0, s, p, d, ks, Np, part);
  BNH_HIP(hipGetLastError());
  return 0;
}
// The largest tile that still gives every compute unit one: a large tile reads its operands from L2 and LDS less often.
// Over 17,280 x 6,144 outputs and K 1,536 (no adapters) 256 x 192 takes 382 us, 128 x 128 398, 64 x 64 530; over 1,024 x
// 6,144 40, 31 and 33 us; over 2,048 x 1,536 38, 26 and 18. Rows that are not 16-byte aligned pass through registers,
// which the largest tile has none left for; it is not built for ranks that are no multiple of 8 either (rank 12 of the
// first: 440 us on 128 x 128, 414 on 256 x 192).
int lora_gemm(const LoraDev &p, const EpiDev &d, bool v, bool vr, bool vo, hipStream_t s) {
  if (v && vr && vo && bnh_ceil_div(p.rows, 256) * bnh_ceil_div(p.N, 192) >= 256)
    return lora_tiles<256, 192, 4, 2, 64, 2, false>(p, d, v, vr, vo, s);
  if (bnh_ceil_div(p.rows, 128) * bnh_ceil_div(p.N, 128) >= 256) return lora_tiles<128, 128, 2, 2, 64, 2, true>(p, d, v, vr, vo, s);
  return lora_tiles<64, 64, 2, 2, 64, 3, true>(p, d, v, vr, vo, s);
}

}  // namespace

extern "C" {

size_t bnh_pw_lora_work_bytes(int M, int B, int N, int K, int r) {
  if (M <= 0 || B <= 0 || N <= 0 || K <= 0 || r < 0 || r > 256 || (long long)M * B >= (1LL << 31) || N >= (1 << 24)) {
    bnh_fail("bnh_pw_lora_work_bytes: parameter check failed");
    return 0;
  }
  const long long rows = (long long)M * B;
  return (size_t)(lora_tu_bytes(rows, r) + (rows <= few ? 4 * few_slices(N, K) * rows * bnh_round_up(N, 4) : 0));
}

int bnh_pw_lora(const uint16_t *x, long long x_ws, int lda, int M, int B, const uint16_t *w, int ldw, int N, int K,
                const float *bias, const bnh_lora *L, const int32_t *idx, const bnh_epi16 *e, void *work,
                size_t work_bytes, void *stream) {
  BNH_REQ(x && w && e && e->out && M > 0 && B > 0 && N > 0 && K > 0 && (long long)M * B < (1LL << 31));
  BNH_REQ(N < (1 << 24) && K < (1 << 24) && lda >= K && ldw >= K && (unsigned)e->act <= 2 && e->opad == 0);
  BNH_REQ(e->ldo >= N && (B == 1 || e->out_ws >= (long long)(M - 1) * e->ldo + N) && (!e->res || e->ldr >= N));
  BNH_REQ(!L || (L->n >= 0 && L->r > 0 && L->r <= 256 && (L->n == 0 || (L->a && L->b)) && idx));
  auto on = [](const void *q, size_t a) { return (uintptr_t)q % a == 0; };
  BNH_REQ(on(x, 2) && on(w, 2) && on(bias, 4) && on(idx, 4) && on(e->out, 2) && on(e->res, 2));
  const bool ad = L && L->n > 0;
  if (ad) BNH_REQ(on(L->a, 2) && on(L->b, 2) && on(L->scale, 4));
  const size_t need = bnh_pw_lora_work_bytes(M, B, N, K, ad ? L->r : 0);
  BNH_REQ(need == 0 || (work && on(work, 16) && work_bytes >= need));
  LoraDev p = {x, w, ad ? L->a : nullptr, ad ? L->b : nullptr, bias, ad ? L->scale : nullptr, ad ? idx : nullptr,
               (uint16_t *)work, ad ? (float *)((char *)work + lora_t_bytes((long long)M * B, L->r)) : nullptr, x_ws, lda, ldw,
               M, N, K, ad ? L->n : 0, ad ? L->r : 0, ad ? lora_half(L->r) : 0, ad ? 2 * lora_half(L->r) : 0,
               B == 1 || x_ws == (long long)M * lda, (long long)M * B, 1.0 / M};
  EpiDev d = {e->act, e->ldo, e->ldr, e->out, e->res, e->out_ws, e->res_ws,
              B == 1 || (e->out_ws == (long long)M * e->ldo && (!e->res || e->res_ws == (long long)M * e->ldr))};
  hipStream_t s = bnh_stream(stream);
  const bool vx = K % 8 == 0 && lda % 8 == 0 && on(x, 16) && (B == 1 || x_ws % 8 == 0);
  const bool v = vx && ldw % 8 == 0 && on(w, 16), va = ad && vx && on(L->a, 16), vr = ad && L->r % 8 == 0 && on(L->b, 16);
  // different adapters among 16 rows in a line: at most the windows that they touch
  const int dy = M >= 15 ? 2 : (14 + M) / M + 1 < 16 ? (14 + M) / M + 1 : 16;
  const bool vo = N % 8 == 0 && e->ldo % 8 == 0 && on(e->out, 16) && (B == 1 || e->out_ws % 8 == 0) &&
                  (!e->res || (e->ldr % 8 == 0 && on(e->res, 16) && (B == 1 || e->res_ws % 8 == 0)));
  if (p.rows <= few) return lora_few(p, d, ad ? dy : 0, v && (!ad || va), vr || !ad, vo, work, s);
  if (ad) {
    const long long tiles = bnh_ceil_div(p.rows, 16), most = bnh_most_blocks(256);
    for (long long t0 = 0; t0 < tiles; t0 += most) {
      const dim3 grid((unsigned)(tiles - t0 < most ? tiles - t0 : most), (unsigned)dy);
#define GO(RT)                                                                       \
  if (va) hipLaunchKernelGGL((k_lora_down<RT, true>), grid, dim3(256), 0, s, p, t0); \
  else hipLaunchKernelGGL((k_lora_down<RT, false>), grid, dim3(256), 0, s, p, t0)
      if (p.r <= 16) GO(1);
      else if (p.r <= 32) GO(2);
      else if (p.r <= 64) GO(4);
      else if (p.r <= 128) GO(8);
      else GO(16);
#undef GO
      BNH_HIP(hipGetLastError());
    }
  }
  return lora_gemm(p, d, v, vr || !ad, vo, s);
}

}  // extern "C"
