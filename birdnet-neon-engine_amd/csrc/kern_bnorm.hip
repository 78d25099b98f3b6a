// The norms around a block, with its gate and residual scale (bnh_block_norm): per row of C values
//   u = post(f);  y = x + rs scale act(gate) u;  n = pre(y),
// post and pre an RMS norm u / sqrt(mean(u^2) + eps) w + b or a layer norm (u - mean) / sqrt(var + eps) w + b.
//
// Bound by HBM: f, gate and x are read once and y and n written once, about 20 operations a value. A row lives in the
// registers of the 16 to 1,024 threads that share it (8 or 16 values each), so that the two statistics and the second pass of the
// variance read nothing again; the layer norm's variance is the sum of squares about the mean already known, not a
// difference of sums. Few values a lane and more waves to a row keep more loads in flight: 17,280 rows of 1,536 in fp16
// take 52.5 us (265 MB, 5.05 TB/s, what a copy reaches) with four waves a row and 8 values a lane, 72 with one wave and 32
// values; 1,200 rows of 1,027 in fp32 10.7 and 20.2. All sums are fp32, lane by lane and then in a fixed tree.
#include "bnh_internal.h"
#include "bnh_f16.h"

namespace {

struct NormDev {
  const void *f, *gate, *x;
  void *y, *n;
  long long f_ws, g_ws, x_ws, y_ws, n_ws;
  int ldf, ldg, ldx, ldy, ldn;
  int post, pre, act;
  float post_eps, pre_eps, rs;
  const float *post_w, *post_b, *pre_w, *pre_b, *scale;
};

// VEC values from p as floats: one load of VEC elements
template <typename T, int VEC>
__device__ __forceinline__ void ld(const T *p, float *v) {
  typedef T V __attribute__((ext_vector_type(VEC)));
  if constexpr (VEC == 1) v[0] = (float)*p;
  else {
    const V t = *(const V *)p;
#pragma unroll
    for (int i = 0; i < VEC; i++) v[i] = (float)t[i];
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void st(T *p, const float *v) {
  typedef T V __attribute__((ext_vector_type(VEC)));
  if constexpr (VEC == 1) *p = (T)v[0];
  else {
    V t;
#pragma unroll
    for (int i = 0; i < VEC; i++) t[i] = (T)v[i];
    *(V *)p = t;
  }
}

// 1 / (1 + e^-z): exp2 of a rounded product, whose relative error only grows where e^-z no longer matters to the sum
// (z >> 0) or where the whole is tiny (z << 0, below 1e-6 relative for |z| < 10)
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

// the sum over the T threads of a row, the same in every one; s: a float of LDS a wave, free on entry
template <int T>
__device__ __forceinline__ float row_sum(float v, float *s) {
#pragma unroll
  for (int d = 1; d < T && d < 64; d *= 2) v += __shfl_xor(v, d);
  if constexpr (T > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
#pragma unroll
    for (int w = 1; w < T / 64; w++) v += s[w];
  }
  return v;
}

// u's norm in place: NV chunks of VEC values a lane, chunk i at column (i T + t) VEC (t the thread within the row), inside
// the row where below C. Values past C are zero on entry and never stored.
template <int T, int VEC, int NV>
__device__ __forceinline__ void norm(float (&u)[NV * VEC], int kind, float eps, const float *w, const float *b, int C,
                                     float rC, int t, float *s) {
  if (kind == 2) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < NV * VEC; i++) a += u[i];
    const float mean = row_sum<T>(a, s) * rC;
#pragma unroll
    for (int i = 0; i < NV; i++)
      if ((i * T + t) * VEC < C)
#pragma unroll
        for (int j = 0; j < VEC; j++) u[i * VEC + j] -= mean;
  }
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < NV * VEC; i++) a = __builtin_fmaf(u[i], u[i], a);
  const float r = rsqrtf(__builtin_fmaf(row_sum<T>(a, s), rC, eps));
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int c = (i * T + t) * VEC;
    if (c >= C) continue;
    float k[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) u[i * VEC + j] *= r;
    if (w) {
      ld<float, VEC>(w + c, k);
#pragma unroll
      for (int j = 0; j < VEC; j++) u[i * VEC + j] *= k[j];
    }
    if (b) {
      ld<float, VEC>(b + c, k);
#pragma unroll
      for (int j = 0; j < VEC; j++) u[i * VEC + j] += k[j];
    }
  }
}

// T threads to a row, a block of 256 or T; rows from row0
template <typename TF, typename TX, int T, int VEC, int NV>
__global__ __launch_bounds__(T > 256 ? T : 256) void k_block_norm(NormDev p, int M, double rM, int C, float rC,
                                                                      unsigned row0, unsigned rows) {
  constexpr int RPB = T < 256 ? 256 / T : 1;  // rows to a block
  __shared__ float s[T > 64 ? T / 64 : 1];
  const int t = threadIdx.x % T;
  const unsigned row = row0 + blockIdx.x * RPB + threadIdx.x / T;
  if (T <= 64 && row >= rows) return;  // all threads of a row, and no barrier in these forms
  const int w = bnh_div(row, M, rM), m = (int)row - w * M;
  float u[NV * VEC], g[NV * VEC], y[NV * VEC];
  const TF *f = p.f ? (const TF *)p.f + w * p.f_ws + (long long)m * p.ldf : nullptr;
  const TF *gate = p.gate ? (const TF *)p.gate + w * p.g_ws + (long long)m * p.ldg : nullptr;
  const TX *x = p.x ? (const TX *)p.x + w * p.x_ws + (long long)m * p.ldx : nullptr;
#pragma unroll
  for (int i = 0; i < NV * VEC; i++) u[i] = y[i] = 0.f, g[i] = 1.f;
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int c = (i * T + t) * VEC;
    if (c >= C) continue;
    if (f) ld<TF, VEC>(f + c, u + i * VEC);
    if (gate) ld<TF, VEC>(gate + c, g + i * VEC);
    if (x) ld<TX, VEC>(x + c, y + i * VEC);
  }
  if (f) {
    if (p.post) norm<T, VEC, NV>(u, p.post, p.post_eps, p.post_w, p.post_b, C, rC, t, s);
    if (gate && p.act) {
#pragma unroll
      for (int i = 0; i < NV * VEC; i++) {
        const float z = g[i];
        g[i] = p.act == 2 ? bnh_relu_f32(z) : p.act == 1 ? z * sigmoid(z) : sigmoid(z);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = (i * T + t) * VEC;
      if (c >= C) continue;
      float k[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j++) k[j] = 1.f;
      if (p.scale) ld<float, VEC>(p.scale + c, k);
#pragma unroll
      for (int j = 0; j < VEC; j++)
        y[i * VEC + j] = __builtin_fmaf(p.rs * k[j], g[i * VEC + j] * u[i * VEC + j], y[i * VEC + j]);
    }
  }
  if (p.y) {
    TX *o = (TX *)p.y + w * p.y_ws + (long long)m * p.ldy;
#pragma unroll
    for (int i = 0; i < NV; i++)
      if ((i * T + t) * VEC < C) st<TX, VEC>(o + (i * T + t) * VEC, y + i * VEC);
  }
  if (p.n) {
    if (p.pre) norm<T, VEC, NV>(y, p.pre, p.pre_eps, p.pre_w, p.pre_b, C, rC, t, s);
    TF *o = (TF *)p.n + w * p.n_ws + (long long)m * p.ldn;
#pragma unroll
    for (int i = 0; i < NV; i++)
      if ((i * T + t) * VEC < C) st<TF, VEC>(o + (i * T + t) * VEC, y + i * VEC);
  }
}

template <typename TF, typename TX, int VEC>
int run(const NormDev &d, int M, int C, int B, hipStream_t s) {
  const unsigned rows = (unsigned)M * B;
  const double rM = 1.0 / M;
  const float rC = 1.f / (float)C;
#define GO(T, E)                                                                                                        \
  do {                                                                                                                  \
    constexpr int NT = T < 256 ? 256 : T, RPB = NT / T;                                                                 \
    const long long most = bnh_most_blocks(NT), blocks = bnh_ceil_div(rows, RPB);                                       \
    for (long long b0 = 0; b0 < blocks; b0 += most) {                                                                   \
      hipLaunchKernelGGL((k_block_norm<TF, TX, T, VEC, (E) / VEC>), dim3((unsigned)(blocks - b0 < most ? blocks - b0 : most)), \
                         dim3(NT), 0, s, d, M, rM, C, rC, (unsigned)(b0 * RPB), rows);                                  \
      BNH_HIP(hipGetLastError());                                                                                       \
    }                                                                                                                   \
    return 0;                                                                                                           \
  } while (0)
  // 20 M values with 8 or 16 a lane: C 64 73 us by 16 threads a row and 212 by 64; C 512 55 by 64 and 100 by 256; C 768 68
  // by 64 (16 values) and 80 by 256 (8); C 1,536 52 by 256 and 72 by 64 (32 values); C 4,096 62 by 256 and 69 by 1,024; C
  // 8,192 58 by 1,024 and 75 by 256 (32 values)
  if (C <= 128) GO(16, 8);
  if (C <= 512) GO(64, 8);
  if (C <= 1024) GO(64, 16);
  if (C <= 2048) GO(256, 8);
  if (C <= 4096) GO(256, 16);
  if (C <= 8192) GO(1024, 8);
  GO(1024, 16);
#undef GO
}

}  // namespace

extern "C" int bnh_block_norm(const bnh_bnorm *p, int M, int C, int B, void *stream) {
  BNH_REQ(p && M > 0 && B > 0 && C > 0 && C <= 16384 && (long long)M * B < (1LL << 31));
  BNH_REQ((p->f16 == 0 || p->f16 == 1) && (p->x16 == 0 || (p->x16 == 1 && p->f16 == 1)));
  BNH_REQ((p->f || p->x) && (p->y || p->n) && (p->f || (!p->gate && !p->scale)));
  BNH_REQ((unsigned)p->post.kind <= 2 && (unsigned)p->pre.kind <= 2 && (unsigned)p->gate_act <= 3);
  BNH_REQ(!p->f || p->ldf >= C);
  BNH_REQ(!p->gate || p->ldg == 0 || p->ldg >= C);
  BNH_REQ(!p->x || p->ldx >= C);
  BNH_REQ(!p->y || (p->ldy >= C && (B == 1 || p->y_ws >= (long long)(M - 1) * p->ldy + C)));
  BNH_REQ(!p->n || (p->ldn >= C && (B == 1 || p->n_ws >= (long long)(M - 1) * p->ldn + C)));
  const size_t ef = p->f16 ? 2 : 4, ex = p->x16 ? 2 : 4;
  bool vec = C % 8 == 0;
  auto see = [&](const void *q, long long ws, int ld, size_t es) {
    if (!q) return true;
    vec = vec && (uintptr_t)q % (8 * es) == 0 && ld % 8 == 0 && (B == 1 || ws % 8 == 0);
    return (uintptr_t)q % es == 0;
  };
  BNH_REQ(see(p->f, p->f_ws, p->ldf, ef) && see(p->gate, p->g_ws, p->ldg, ef) && see(p->x, p->x_ws, p->ldx, ex) &&
          see(p->y, p->y_ws, p->ldy, ex) && see(p->n, p->n_ws, p->ldn, ef));
  for (const float *q : {p->post.w, p->post.b, p->pre.w, p->pre.b, p->scale}) BNH_REQ(see(q, 0, 0, 4));
  NormDev d = {p->f, p->gate, p->x, p->y, p->n, p->f_ws, p->g_ws, p->x_ws, p->y_ws, p->n_ws, p->ldf, p->ldg, p->ldx,
               p->ldy, p->ldn, p->post.kind, p->pre.kind, p->gate_act, p->post.eps, p->pre.eps, p->rs, p->post.w,
               p->post.b, p->pre.w, p->pre.b, p->scale};
  hipStream_t s = bnh_stream(stream);
  if (p->x16) return vec ? run<h16, h16, 8>(d, M, C, B, s) : run<h16, h16, 1>(d, M, C, B, s);
  if (p->f16) return vec ? run<h16, float, 8>(d, M, C, B, s) : run<h16, float, 1>(d, M, C, B, s);
  return vec ? run<float, float, 8>(d, M, C, B, s) : run<float, float, 1>(d, M, C, B, s);
}
