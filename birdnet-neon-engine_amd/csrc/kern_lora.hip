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

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef h16 v8h __attribute__((ext_vector_type(8)));

// eight halves from p, of which the first n are inside; V: all or none of them are, and p is 16-byte aligned
template <bool V>
__device__ __forceinline__ v8h ld8(const uint16_t *p, int n) {
  v8h r = {};
  if (V) {
    if (n > 0) r = *(const v8h *)p;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
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

// 64 rows x 128 channels a block of four waves, 32 x 64 each, the fragments straight from global memory
template <bool V, bool VR>
__global__ __launch_bounds__(256) void k_lora_gemm(LoraDev p, EpiDev e) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, kc = (lane >> 4) * 8;
  const int nnb = (p.N + 127) / 128;
  const unsigned lb = bnh_xcd_block(blockIdx.x, gridDim.x);
  const long long r0 = (long long)(lb / nnb) * 64 + (wave >> 1) * 32;
  const int n0 = (int)(lb % nnb) * 128 + (wave & 1) * 64;
  if (r0 >= p.rows || n0 >= p.N) return;
  const uint16_t *ap[2], *wp[4];
  int id[2], win[2];
  long long row[2];
#pragma unroll
  for (int t = 0; t < 2; t++) {
    row[t] = r0 + 16 * t + lr < p.rows ? r0 + 16 * t + lr : p.rows - 1;
    win[t] = bnh_div(row[t], p.M, p.rM);
    id[t] = p.idx ? lora_id(p, win[t]) : -1;
    ap[t] = p.x + win[t] * p.x_ws + (long long)(row[t] - (long long)win[t] * p.M) * p.lda + kc;
  }
  int ch[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    ch[j] = n0 + 16 * j + lr < p.N ? n0 + 16 * j + lr : p.N - 1;
    wp[j] = p.w + (long long)ch[j] * p.ldw + kc;
  }
  v4f acc[2][4];
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[t][j] = (v4f){0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < p.K; k += 32) {
    v8h a[2], b[4];
#pragma unroll
    for (int t = 0; t < 2; t++) a[t] = ld8<V>(ap[t] + k, p.K - k - kc);
#pragma unroll
    for (int j = 0; j < 4; j++) b[j] = ld8<V>(wp[j] + k, p.K - k - kc);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int j = 0; j < 4; j++) acc[t][j] = mma(a[t], b[j], acc[t][j]);
  }
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const uint16_t *tp = p.t + row[t] * p.r32 + kc;
    uint32_t left = (uint32_t)__builtin_amdgcn_ballot_w64(lane < 16 && id[t] >= 0);
    while (left) {  // one adapter of the 16 rows a turn
      const int j = __builtin_amdgcn_readlane(id[t], __builtin_ctz(left));
      const uint32_t mine = (uint32_t)__builtin_amdgcn_ballot_w64(lane < 16 && id[t] == j);
      left &= ~mine;
      v4f u[4];
#pragma unroll
      for (int c = 0; c < 4; c++) u[c] = (v4f){0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < p.r32; k += 32) {
        const v8h a = *(const v8h *)(tp + k);
#pragma unroll
        for (int c = 0; c < 4; c++)
          u[c] = mma(a, ld8<VR>(p.b + ((long long)j * p.N + ch[c]) * p.r + k + kc, p.r - k - kc), u[c]);
      }
#pragma unroll
      for (int q = 0; q < 4; q++)
        if (mine >> (4 * (lane >> 4) + q) & 1)
#pragma unroll
          for (int c = 0; c < 4; c++) acc[t][c][q] += u[c][q];
    }
  }
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int m = 4 * (lane >> 4) + q;
      const long long r = r0 + 16 * t + m;
      const int w = __shfl(win[t], m);
      if (r >= p.rows) continue;
      const int mr = (int)(r - (long long)w * p.M);
      uint16_t *o = e.out + w * e.out_ws + (long long)mr * e.ldo;
      const uint16_t *rs = e.res ? e.res + w * e.res_ws + (long long)mr * e.ldr : nullptr;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int n = n0 + 16 * j + lr;
        if (n >= p.N) continue;
        float y = lora_act(acc[t][j][q] + (p.bias ? p.bias[n] : 0.f), e.act);
        if (rs) y += (float)hfrom(rs[n]);
        o[n] = hbits((h16)y);
      }
    }
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
  const long long nb = bnh_ceil_div(p.rows, 64) * bnh_ceil_div(N, 128);
  BNH_REQ(nb < (1LL << 31));
  const dim3 grid((unsigned)nb);
  if (v && vr) hipLaunchKernelGGL((k_lora_gemm<true, true>), grid, dim3(256), 0, s, p, d);
  else if (v) hipLaunchKernelGGL((k_lora_gemm<true, false>), grid, dim3(256), 0, s, p, d);
  else if (vr) hipLaunchKernelGGL((k_lora_gemm<false, true>), grid, dim3(256), 0, s, p, d);
  else hipLaunchKernelGGL((k_lora_gemm<false, false>), grid, dim3(256), 0, s, p, d);
  BNH_HIP(hipGetLastError());
  return 0;
}

}  // extern "C"
