// A shared fp16 projection with low-rank adapters of many requests beside it (bnh_pw_lora):
//   out = act(W x + bias + s_j B_j (A_j x)) (+ res), j the adapter of the row's window.
//
// Two launches. k_lora_down computes t = s_j A_j x for every row with an adapter (rounded to fp16: the factor that the
// matrix instruction of the second product takes; |t| past 65504 becomes infinite). k_lora_gemm computes W x on fp16 MFMA
// with fp32 sums and carries the K loop on over the r values of t with the adapter's B, so that the adapter costs no pass
// over the output. Rows of one matrix instruction are independent of each other, so a block of 16 rows whose adapters
// differ multiplies all of them by each of the adapters in it and every row keeps its own: nothing of another request's
// adapter, not even an infinity or a NaN, reaches it.
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

struct LoraDev {
  const uint16_t *x, *w, *a, *b;
  const float *bias, *scale;
  const int32_t *idx;
  uint16_t *t;
  long long x_ws;
  int lda, ldw, M, N, K, n, r, r32;  // r32: r rounded up to 32, t's row
  long long rows;
  double rM;
};

__device__ __forceinline__ int lora_id(const LoraDev &p, int win) {  // -1: none
  const int j = p.idx[win];
  return j >= 0 && j < p.n ? j : -1;
}

// t of 16 rows for the blockIdx.y-th different adapter among them; the block's four waves take every fourth step of 32
// of K. RT: 16-column tiles of r32.
template <int RT, bool V>
__global__ __launch_bounds__(256) void k_lora_down(LoraDev p) {
  __shared__ float s_t[3][RT][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, kc = (lane >> 4) * 8;
  const long long row = (long long)blockIdx.x * 16 + lr < p.rows ? (long long)blockIdx.x * 16 + lr : p.rows - 1;
  const int win = bnh_div(row, p.M, p.rM);
  const int id = lora_id(p, win);
  // the first rows of the different adapters, and of those the one that is this block's
  bool dup = false;
#pragma unroll
  for (int j = 0; j < 15; j++) {
    const int o = __builtin_amdgcn_readlane(id, j);
    dup = dup || (j < lr && o == id);
  }
  uint32_t lead = (uint32_t)(__builtin_amdgcn_ballot_w64(lane < 16 && !dup && id >= 0));
  for (unsigned i = 0; i < blockIdx.y; i++) lead &= lead - 1;
  if (!lead) return;
  const int j = __builtin_amdgcn_readlane(id, __builtin_ctz(lead));
  const uint16_t *xp = p.x + win * p.x_ws + (long long)(row - (long long)win * p.M) * p.lda + kc;
  const uint16_t *ap = p.a + (long long)j * p.r * p.K + kc;
  v4f acc[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) acc[t] = (v4f){0.f, 0.f, 0.f, 0.f};
  for (int k = 32 * wave; k < p.K; k += 128) {
    const v8h x = ld8<V>(xp + k, p.K - k - kc);
#pragma unroll
    for (int t = 0; t < RT; t++) {
      const int c = 16 * t + lr;
      const v8h a = c < p.r ? ld8<V>(ap + (long long)c * p.K + k, p.K - k - kc) : (v8h){};
      acc[t] = mma(x, a, acc[t]);
    }
  }
  if (wave) {
#pragma unroll
    for (int t = 0; t < RT; t++) *(v4f *)&s_t[wave - 1][t][4 * lane] = acc[t];
  }
  __syncthreads();
  if (wave) return;
  const float sc = p.scale ? p.scale[j] : 1.f;
#pragma unroll
  for (int t = 0; t < RT; t++) {
    acc[t] += *(v4f *)&s_t[0][t][4 * lane] + (*(v4f *)&s_t[1][t][4 * lane] + *(v4f *)&s_t[2][t][4 * lane]);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int m = 4 * (lane >> 4) + e;
      const long long r = (long long)blockIdx.x * 16 + m;
      const int rid = __shfl(id, m);
      if (r < p.rows && rid == j && 16 * t + lr < p.r32) p.t[r * p.r32 + 16 * t + lr] = 16 * t + lr < p.r ? hbits((h16)(sc * acc[t][e])) : 0;
    }
  }
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
};

// The tile of rows [r0, ...) x channels [n0, ...) of logical block lb: blocks that follow each other (and so run under one
// XCD's L2) form groups of 8 row tiles that share their channels' weights
__device__ __forceinline__ void lora_tile(unsigned lb, int nm, int nn, int *tm, int *tn) {
  const unsigned g = lb / (8u * nn), i = lb % (8u * nn);
  const unsigned gm = nm - 8 * g < 8 ? nm - 8 * g : 8;
  *tm = (int)(8 * g + i % gm);
  *tn = (int)(i / gm);
}

// BM rows x BN channels a block of WM x WN waves. The operands' steps of BK values of K pass through a ring of LDS stages
// that global loads fill directly (DMA: rows that are 16-byte aligned), three ahead, with one barrier a step; without DMA
// through registers into two stages. A row's 16-byte chunks lie in LDS at chunk ^ f(row), so that the 16 rows of a
// fragment's read fall on different banks (the loads write 16 bytes a lane in lane order, so the lane's chunk of the
// row is permuted instead). The first operand of the matrix instruction is the weights': a lane's accumulators are
// four channels of one row.
template <int BM, int BN, int WM, int WN, int BK, bool DMA, bool VR, bool VO>
__global__ __launch_bounds__(64 * WM * WN) void k_lora_gemm(LoraDev p, EpiDev e, int nm, int nn) {
  constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, CH = BK / 8, RPI = 64 / CH;
  constexpr int NL = (BM + BN) * CH / 64 / NW, ST = DMA ? 4 : 2, SH = (BM + BN) * BK;  // loads a wave; stages, their halves
  constexpr int XS = 16 * TN + 4;                                                   // an exchange row, floats
  static_assert((BM + BN) * CH % (64 * NW) == 0 && BM % RPI == 0, "");
  constexpr int LDS = ST * SH * 2 > NW * 16 * XS * 4 ? ST * SH * 2 : NW * 16 * XS * 4;
  __shared__ __attribute__((aligned(16))) char s_raw[LDS];
  uint16_t *s = (uint16_t *)s_raw;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, q4 = lane >> 4;
  int tm, tn;
  lora_tile(bnh_xcd_block(blockIdx.x, gridDim.x), nm, nn, &tm, &tn);
  const long long r0 = (long long)tm * BM;
  const int n0 = tn * BN;
  auto fx = [](int row) { return CH == 4 ? (row >> 2) & 3 : (row >> 1) & 7; };

  // this lane's chunks of a step: load i of the wave fills LDS rows (i NW + wave) RPI ..., x's first and then w's
  const uint16_t *gp[NL];
  int gk[NL];
#pragma unroll
  for (int i = 0; i < NL; i++) {
    const int row = (i * NW + wave) * RPI + lane / CH;
    gk[i] = (lane % CH ^ fx(row)) * 8;
    if (row < BM) {
      const long long r = r0 + row < p.rows ? r0 + row : p.rows - 1;
      const int w = bnh_div(r, p.M, p.rM);
      gp[i] = p.x + w * p.x_ws + (long long)(r - (long long)w * p.M) * p.lda + gk[i];
    } else {
      const int n = n0 + row - BM < p.N ? n0 + row - BM : p.N - 1;
      gp[i] = p.w + (long long)n * p.ldw + gk[i];
    }
  }
  v4f acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; j++)
#pragma unroll
    for (int i = 0; i < TM; i++) acc[j][i] = (v4f){0.f, 0.f, 0.f, 0.f};
  const int wm = wave / WN * (TM * 16), wn = wave % WN * (TN * 16);
  auto step = [&](const uint16_t *st) {
#pragma unroll
    for (int k = 0; k < BK / 32; k++) {
      const int c = ((4 * k + q4) ^ fx(lr)) * 8;
      v8h x[TM], w[TN];
#pragma unroll
      for (int j = 0; j < TN; j++) w[j] = *(const v8h *)(st + (BM + wn + 16 * j + lr) * BK + c);
#pragma unroll
      for (int i = 0; i < TM; i++) x[i] = *(const v8h *)(st + (wm + 16 * i + lr) * BK + c);
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[j][i] = mma(w[j], x[i], acc[j][i]);
    }
  };
  auto put = [&](uint16_t *st, const v8h *v) {
#pragma unroll
    for (int i = 0; i < NL; i++) *(v8h *)(st + (i * NW + wave) * 512 + lane * 8) = v[i];
  };
  const int full = p.K / BK;
  if constexpr (DMA) {
    auto issue = [&](int t) {
#pragma unroll
      for (int i = 0; i < NL; i++)
        rq_dma16((const int8_t *)(gp[i] + (long long)t * BK), (const lds_i8 *)(s + (t & 3) * SH + (i * NW + wave) * 512));
    };
    for (int t = 0; t < 3 && t < full; t++) issue(t);
    for (int t = 0; t < full; t++) {
      if (t + 2 < full) {
        if constexpr (NL == 2) RQ_WAIT_VM(4);
        else if constexpr (NL == 4) RQ_WAIT_VM(8);
        else RQ_WAIT_VM(0);
      } else {
        RQ_WAIT_VM(0);
      }
      // every read of step t - 1's stage is done, which step t + 3 takes
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      RQ_BARRIER();
      if (t + 3 < full) issue(t + 3);
      step(s + (t & 3) * SH);
    }
  } else {
    v8h v[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) v[i] = ld8<false>(gp[i], p.K - gk[i]);
    for (int t = 0; t < full; t++) {
      put(s + (t & 1) * SH, v);
      const int k = (t + 1) * BK;
#pragma unroll
      for (int i = 0; i < NL; i++)
        if (k + gk[i] < p.K) v[i] = ld8<false>(gp[i] + k, p.K - k - gk[i]);
      __syncthreads();
      step(s + (t & 1) * SH);
    }
  }
  if (full * BK < p.K) {  // the last values of K, zeros past them
    v8h v[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) v[i] = ld8<DMA>(gp[i] + full * BK, p.K - full * BK - gk[i]);
    __syncthreads();
    put(s, v);
    __syncthreads();
    step(s);
  }
  __syncthreads();

  float *xch = (float *)s_raw + wave * 16 * XS;
#pragma unroll
  for (int i = 0; i < TM; i++) {
    const long long rb = r0 + wm + 16 * i;
    if (rb >= p.rows) break;
    const long long row = rb + lr < p.rows ? rb + lr : p.rows - 1;
    if (p.idx) {
      const int id = lora_id(p, bnh_div(row, p.M, p.rM));
      const uint16_t *tp = p.t + row * p.r32 + 8 * q4;
      uint32_t left = (uint32_t)__builtin_amdgcn_ballot_w64(lane < 16 && id >= 0);
      while (left) {  // one adapter of the 16 rows a turn
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
        left &= ~(uint32_t)__builtin_amdgcn_ballot_w64(lane < 16 && id == a);
        v4f u[TN];
#pragma unroll
        for (int j = 0; j < TN; j++) u[j] = (v4f){0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < p.r32; k += 32) {
          const v8h x = *(const v8h *)(tp + k);
#pragma unroll
          for (int j = 0; j < TN; j++) {
            const int n = n0 + wn + 16 * j + lr < p.N ? n0 + wn + 16 * j + lr : p.N - 1;
            u[j] = mma(ld8<VR>(p.b + ((long long)a * p.N + n) * p.r + k + 8 * q4, p.r - k - 8 * q4), x, u[j]);
          }
        }
        if (id == a) {
#pragma unroll
          for (int j = 0; j < TN; j++) acc[j][i] += u[j];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < TN; j++) {
      const int n = n0 + wn + 16 * j + 4 * q4;
      v4f y;
#pragma unroll
      for (int r = 0; r < 4; r++) y[r] = lora_act(acc[j][i][r] + (p.bias && n + r < p.N ? p.bias[n + r] : 0.f), e.act);
      *(v4f *)(xch + lr * XS + 16 * j + 4 * q4) = y;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    constexpr int LPR = 2 * TN, RPP = 64 / LPR;  // lanes to a row, rows a pass
#pragma unroll
    for (int h = 0; h < 16; h += RPP) {
      const int m = h + lane / LPR, c = lane % LPR * 8, n = n0 + wn + c;
      const long long r = rb + m;
      if (m >= 16 || r >= p.rows || n >= p.N) continue;
      const int w = bnh_div(r, p.M, p.rM);
      const long long mr = r - (long long)w * p.M;
      const float *y = xch + m * XS + c;
      uint16_t *o = e.out + w * e.out_ws + mr * e.ldo + n;
      const uint16_t *rs = e.res ? e.res + w * e.res_ws + mr * e.ldr + n : nullptr;
      if (VO) {
        v8h z = {};
        if (rs) z = *(const v8h *)rs;
        v8h t;
#pragma unroll
        for (int k = 0; k < 8; k++) t[k] = (h16)(rs ? y[k] + (float)z[k] : y[k]);
        *(v8h *)o = t;
      } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (n + k < p.N) o[k] = hbits((h16)(rs ? y[k] + (float)hfrom(rs[k]) : y[k]));
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

template <int BM, int BN, int WM, int WN, int BK>
int lora_tiles(const LoraDev &p, const EpiDev &d, bool v, bool vr, bool vo, hipStream_t s) {
  const long long nm = bnh_ceil_div(p.rows, BM), nn = bnh_ceil_div(p.N, BN);
  if (nm * nn >= (1LL << 31)) return bnh_fail("bnh_pw_lora: %lld x %d outputs are too many tiles", p.rows, p.N);
  const dim3 grid((unsigned)(nm * nn)), block(64 * WM * WN);
#define GO(V, VR, VO) \
  hipLaunchKernelGGL((k_lora_gemm<BM, BN, WM, WN, BK, V, VR, VO>), grid, block, 0, s, p, d, (int)nm, (int)nn)
  if (v && vr && vo) GO(true, true, true);
  else if (v && vo) GO(true, false, true);
  else if (v) GO(true, false, false);
  else if (vo) GO(false, false, true);
  else GO(false, false, false);
#undef GO
  BNH_HIP(hipGetLastError());
  return 0;
}
// The largest tile that still gives every compute unit one: a large tile reads its operands from L2 less often
int lora_gemm(const LoraDev &p, const EpiDev &d, bool v, bool vr, bool vo, hipStream_t s) {
  if (bnh_ceil_div(p.rows, 256) * bnh_ceil_div(p.N, 256) >= 256) return lora_tiles<256, 256, 2, 4, 32>(p, d, v, vr, vo, s);
  if (bnh_ceil_div(p.rows, 128) * bnh_ceil_div(p.N, 128) >= 256) return lora_tiles<128, 128, 2, 2, 32>(p, d, v, vr, vo, s);
  return lora_tiles<64, 64, 2, 2, 64>(p, d, v, vr, vo, s);
}

}  // namespace

extern "C" {

size_t bnh_pw_lora_work_bytes(int M, int B, int N, int K, int r) {
  if (M <= 0 || B <= 0 || N <= 0 || K <= 0 || r < 0 || r > 256) {
    bnh_fail("bnh_pw_lora_work_bytes: parameter check failed");
    return 0;
  }
  return (size_t)bnh_round_up((long long)M * B * bnh_round_up(r, 32) * 2, 256);
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
  if (ad) {
    BNH_REQ(on(L->a, 2) && on(L->b, 2) && on(L->scale, 4) && work && on(work, 16));
    BNH_REQ(work_bytes >= bnh_pw_lora_work_bytes(M, B, N, K, L->r));
  }
  LoraDev p = {x, w, ad ? L->a : nullptr, ad ? L->b : nullptr, bias, ad ? L->scale : nullptr, ad ? idx : nullptr,
               (uint16_t *)work, x_ws, lda, ldw, M, N, K, ad ? L->n : 0, ad ? L->r : 0,
               ad ? (int)bnh_round_up(L->r, 32) : 0, (long long)M * B, 1.0 / M};
  EpiDev d = {e->act, e->ldo, e->ldr, e->out, e->res, e->out_ws, e->res_ws};
  hipStream_t s = bnh_stream(stream);
  const bool vx = K % 8 == 0 && lda % 8 == 0 && on(x, 16) && (B == 1 || x_ws % 8 == 0);
  const bool v = vx && ldw % 8 == 0 && on(w, 16), va = ad && vx && on(L->a, 16), vr = ad && L->r % 8 == 0 && on(L->b, 16);
  if (ad) {
    // different adapters among 16 rows in a line: at most the windows that they touch
    const dim3 grid((unsigned)bnh_ceil_div(p.rows, 16), (unsigned)(M >= 15 ? 2 : (14 + M) / M + 1 < 16 ? (14 + M) / M + 1 : 16));
#define GO(RT)                                                                         \
  if (va) hipLaunchKernelGGL((k_lora_down<RT, true>), grid, dim3(256), 0, s, p);       \
  else hipLaunchKernelGGL((k_lora_down<RT, false>), grid, dim3(256), 0, s, p)
    if (p.r32 <= 32) GO(2);
    else if (p.r32 <= 64) GO(4);
    else if (p.r32 <= 128) GO(8);
    else GO(16);
#undef GO
    BNH_HIP(hipGetLastError());
  }
  const bool vo = N % 8 == 0 && e->ldo % 8 == 0 && on(e->out, 16) && (B == 1 || e->out_ws % 8 == 0) &&
                  (!e->res || (e->ldr % 8 == 0 && on(e->res, 16) && (B == 1 || e->res_ws % 8 == 0)));
  return lora_gemm(p, d, v, vr, vo, s);
}

}  // extern "C"
