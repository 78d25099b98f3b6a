// Linear attention with a decay for each head (bnh_linattn): per sequence and head, over its rows t
//   S = exp(g_t) S + k_t v_t^T,  o_t = scale q_t^T S,
// S [dk][dv] in fp32.
//
// k_la_step, the recurrence itself, for sequences of few rows: bound by reading and writing the states (8 dk dv bytes a
// sequence and head, against 2 (2 dk + 2 dv) bytes a row). A block owns 4 LANES columns of one state: LANES lanes, four
// columns each (16 bytes), side by side over the 256 / LANES groups that share its rows; a thread keeps its rows' columns
// in registers over all rows of the sequence.
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
  float scale;
};

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
  const int sl = (int)(blockIdx.x % nsl), h = (int)(blockIdx.x / nsl % p.H), b = (int)(blockIdx.x / nsl / p.H);
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
    const float d = expf(p.g[r * p.ldg + h]);
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
int step_run(const LaDev &d, int B, hipStream_t s) {
  constexpr int RG = 256 / LANES;
  const int nsl = (int)bnh_ceil_div(d.dv, 4 * LANES), kr = (int)bnh_ceil_div(d.dk, RG);
  const dim3 grid((unsigned)((long long)nsl * d.H * B)), block(256);
#define GO(KR) hipLaunchKernelGGL((k_la_step<T, LANES, KR, VS>), grid, block, 0, s, d, nsl)
  if (kr <= 256 / RG / 4) GO(256 / RG / 4);
  else if (kr <= 256 / RG / 2) GO(256 / RG / 2);
  else GO(256 / RG);
#undef GO
  BNH_HIP(hipGetLastError());
  return 0;
}

int la_check(const bnh_la *p, int T, int B) {
  BNH_REQ(p && T > 0 && B > 0 && p->H > 0 && p->Hq > 0 && p->Hk > 0 && p->Hv > 0);
  BNH_REQ(p->H % p->Hq == 0 && p->H % p->Hk == 0 && p->H % p->Hv == 0);
  BNH_REQ(p->dk > 0 && p->dk <= 256 && p->dv > 0 && p->dv <= 256 && (p->f16 == 0 || p->f16 == 1));
  BNH_REQ((long long)B * p->H < (1LL << 24) && p->H <= 65536);
  return 0;
}

}  // namespace

extern "C" {

size_t bnh_linattn_work_bytes(const bnh_la *p, int T, int B) {
  if (la_check(p, T, B)) return 0;
  return 0;
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
             p->H, p->H / p->Hq, p->H / p->Hk, p->H / p->Hv, p->dk, p->dv, p->slots, T, rows, p->scale};
  const bool vs = p->dv % 4 == 0 && on(p->s0, 16) && on(p->s1, 16);
  hipStream_t s = bnh_stream(stream);
  if (p->f16) return vs ? step_run<h16, 32, true>(d, B, s) : step_run<h16, 32, false>(d, B, s);
  return vs ? step_run<float, 32, true>(d, B, s) : step_run<float, 32, false>(d, B, s);
}

}  // extern "C"
