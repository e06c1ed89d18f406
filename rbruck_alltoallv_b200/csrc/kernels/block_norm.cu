// The RMS norms around a transformer block: the norm of the block's output, its gate, the residual scale, the residual sum
// and the norm in front of the next block in one pass over the rows, and the backward pass of the same.
//
//   forward   zhat = z * i1, i1 = rsqrt(mean z^2 + eps);  r2 = r + s g w1 zhat;  xhat = r2 * i2, i2 = rsqrt(mean r2^2 + eps);
//             u = w2 xhat
//   backward  a = w2 du;  D = dr2 + i2 (a - xhat mean(a xhat)) = dr;  b = s g w1 D;  dz = i1 (b - zhat mean(b zhat));
//             dw2 = sum_t du xhat;  dw1 = s sum_t g D zhat;  dg = s w1 D zhat, summed over what g is broadcast over
//
// Bound by HBM: the forward pass reads z and r and writes r2 and u, the backward pass reads z, r, dr2, du and writes dz and
// dr.  A row stays in the registers of the threads that share it, between both norms too, so everything is read once: r2 is
// never read back (the backward pass makes it again from z and r, in 32 bits, at the price of no byte, since it would have to
// read r2 in place of r).  CTAs are persistent and hold the weights of their columns in registers; the rows of the next
// iteration are on the way while one is reduced.  All sums are held in 32 bits and added in a fixed order.
//
// Sums over the tokens: every thread keeps those of its own columns in registers for all rows of its CTA, and the CTAs' sums
// are added by a second, small kernel; no atomics.  With a gate per channel both its gradient and w1's are the same sum
// sum_t D zhat times a factor per channel, so that two sums per column do for three gradients.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "kernels/pdl.cuh"
#include "rbv/norm.h"

namespace rbv {
namespace {

constexpr int kNormWarpRows = 4;          // rows per CTA where a warp has a row to itself

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// VEC consecutive elements as they are in memory; VEC * sizeof(T) is a multiple of 16, or VEC is 1.
template <typename T, int VEC>
struct Raw {
  static constexpr int Q = VEC * (int)sizeof(T) / 16;
  uint4 q[Q];
  __device__ __forceinline__ void load(const T* p) {
    #pragma unroll
    for (int i = 0; i < Q; i++) q[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void store(T* p) const {
    #pragma unroll
    for (int i = 0; i < Q; i++) reinterpret_cast<uint4*>(p)[i] = q[i];
  }
  __device__ __forceinline__ void zero() {
    #pragma unroll
    for (int i = 0; i < Q; i++) q[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ float get(int k) const { return to_f(reinterpret_cast<const T*>(q)[k]); }
  __device__ __forceinline__ void set(int k, float v) { reinterpret_cast<T*>(q)[k] = from_f<T>(v); }
};
template <typename T>
struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ void zero() { v = from_f<T>(0.0f); }
  __device__ __forceinline__ float get(int) const { return to_f(v); }
  __device__ __forceinline__ void set(int, float x) { v = from_f<T>(x); }
};

// Parameters that are fp32 or of the block's type.
template <typename T, int VEC>
__device__ __forceinline__ void params(const void* p, int f32, long long i, float (&v)[VEC]) {
  if (f32) {
    Raw<float, VEC> q;
    q.load(static_cast<const float*>(p) + i);
    #pragma unroll
    for (int k = 0; k < VEC; k++) v[k] = q.get(k);
  } else {
    Raw<T, VEC> q;
    q.load(static_cast<const T*>(p) + i);
    #pragma unroll
    for (int k = 0; k < VEC; k++) v[k] = q.get(k);
  }
}
template <typename T>
__device__ __forceinline__ float param(const void* p, int f32, long long i) {
  return f32 ? static_cast<const float*>(p)[i] : to_f(static_cast<const T*>(p)[i]);
}
template <typename T>
__device__ __forceinline__ void set_param(void* p, int f32, long long i, float v) {
  if (f32) static_cast<float*>(p)[i] = v;
  else static_cast<T*>(p)[i] = from_f<T>(v);
}

// Sum over the threads that share a row: a warp, or the CTA.  `red` alternates between two buffers from call to call, so
// that one barrier per sum is enough (nobody can be two sums ahead).
struct RowSum {
  float (*buf)[32];
  int turn;
  __device__ __forceinline__ float operator()(float v) {
    #pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (blockDim.x == 32) return v;
    float* b = buf[turn];
    turn ^= 1;
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) b[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = lane < warps ? b[lane] : 0.0f;
    #pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  }
};

// scale * w1 (* gate per channel) of VEC columns.
template <typename TZ, int VEC>
__device__ __forceinline__ void post_factors(const rbv_norm_t& a, int col, float (&v)[VEC]) {
  params<TZ>(a.w1, a.w1_f32, col, v);
  #pragma unroll
  for (int k = 0; k < VEC; k++) v[k] *= a.scale;
  if (a.gate_kind == RBV_GATE_CHANNEL) {
    float g[VEC];
    params<TZ>(a.gate, a.gate_f32, col, g);
    #pragma unroll
    for (int k = 0; k < VEC; k++) v[k] *= g[k];
  }
}

// FULL: a gate per element.
template <typename TZ, typename TR, int VEC, int NV, int MAXT, bool FULL>
__global__ void __launch_bounds__(MAXT, 1) block_norm_kernel(const __grid_constant__ rbv_norm_t a) {
  constexpr bool HOLD = NV * VEC <= 8;      // weights and the next rows in registers; beyond that they would spill
  __shared__ float red[2][32];
  RowSum row_sum{red, 0};
  const int H = a.H;
  const float inv_h = 1.0f / (float)H;
  const bool block = a.z != nullptr, norm = a.w2 != nullptr;
  int col[NV];
  bool in[NV];
  #pragma unroll
  for (int i = 0; i < NV; i++) {
    col[i] = (i * (int)blockDim.x + (int)threadIdx.x) * VEC;
    in[i] = col[i] < H;
  }
  pdl_trigger();
  pdl_wait();
  float wg[HOLD ? NV : 1][VEC], w2[HOLD ? NV : 1][VEC];
  if (HOLD) {
    #pragma unroll
    for (int i = 0; i < NV; i++) {
      if (in[i] && block) post_factors<TZ>(a, col[i], wg[HOLD ? i : 0]);
      if (in[i] && norm) params<TZ>(a.w2, a.w2_f32, col[i], w2[HOLD ? i : 0]);
    }
  }
  const long long step = (long long)gridDim.x * blockDim.y;
  long long t = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  Raw<TZ, VEC> z[NV];
  Raw<TR, VEC> r[NV];
  auto fetch = [&](long long row) {
    #pragma unroll
    for (int i = 0; i < NV; i++) {
      z[i].zero(); r[i].zero();
      if (row < a.T && in[i]) {
        if (block) z[i].load(static_cast<const TZ*>(a.z) + row * a.z_ld + col[i]);
        r[i].load(static_cast<const TR*>(a.r) + row * a.r_ld + col[i]);
      }
    }
  };
  if (HOLD) fetch(t);
  for (; t < a.T; t += step) {
    if (!HOLD) fetch(t);
    float x[NV][VEC];                       // r2
    float zf[NV][VEC];
    float s = 0.0f;
    #pragma unroll
    for (int i = 0; i < NV; i++)
      #pragma unroll
      for (int k = 0; k < VEC; k++) {
        zf[i][k] = z[i].get(k);
        x[i][k] = r[i].get(k);
        s = fmaf(zf[i][k], zf[i][k], s);
      }
    if (HOLD) fetch(t + step);
    if (block) {
      const float i1 = rsqrtf(fmaf(row_sum(s), inv_h, a.eps));
      if (a.rstd1 && threadIdx.x == 0) a.rstd1[t] = i1;
      const float f = a.gate_kind == RBV_GATE_TOKEN ? i1 * param<TZ>(a.gate, a.gate_f32, t) : i1;
      #pragma unroll
      for (int i = 0; i < NV; i++) {
        if (!in[i]) continue;
        float w[VEC], g[VEC];
        if (!HOLD) post_factors<TZ>(a, col[i], w);
        if (FULL) params<TZ>(a.gate, a.gate_f32, t * a.gate_ld + col[i], g);
        Raw<TR, VEC> o;
        #pragma unroll
        for (int k = 0; k < VEC; k++) {
          const float v = HOLD ? wg[HOLD ? i : 0][k] : w[k];
          x[i][k] = fmaf(FULL ? v * g[k] : v, zf[i][k] * f, x[i][k]);
          o.set(k, x[i][k]);
        }
        o.store(static_cast<TR*>(a.r2) + t * H + col[i]);
      }
    }
    if (norm) {
      s = 0.0f;
      #pragma unroll
      for (int i = 0; i < NV; i++)
        #pragma unroll
        for (int k = 0; k < VEC; k++) s = fmaf(x[i][k], x[i][k], s);
      const float i2 = rsqrtf(fmaf(row_sum(s), inv_h, a.eps));
      if (a.rstd2 && threadIdx.x == 0) a.rstd2[t] = i2;
      #pragma unroll
      for (int i = 0; i < NV; i++) {
        if (!in[i]) continue;
        float w[VEC];
        if (!HOLD) params<TZ>(a.w2, a.w2_f32, col[i], w);
        Raw<TZ, VEC> o;
        #pragma unroll
        for (int k = 0; k < VEC; k++) o.set(k, x[i][k] * i2 * (HOLD ? w2[HOLD ? i : 0][k] : w[k]));
        o.store(static_cast<TZ*>(a.u) + t * H + col[i]);
      }
    }
  }
}

template <typename TZ, typename TR, int VEC, int NV, int MAXT, bool FULL>
__global__ void __launch_bounds__(MAXT, 1) block_norm_backward_kernel(const __grid_constant__ rbv_norm_t a) {
  constexpr bool HOLD = NV * VEC <= 8;
  __shared__ float red[2][32];
  RowSum row_sum{red, 0};
  const int H = a.H;
  const float inv_h = 1.0f / (float)H;
  const bool block = a.z != nullptr, norm = a.w2 != nullptr && a.du != nullptr;
  int col[NV];
  bool in[NV];
  #pragma unroll
  for (int i = 0; i < NV; i++) {
    col[i] = (i * (int)blockDim.x + (int)threadIdx.x) * VEC;
    in[i] = col[i] < H;
  }
  pdl_trigger();
  pdl_wait();
  float wg[HOLD ? NV : 1][VEC], w2[HOLD ? NV : 1][VEC], s1[NV][VEC], s2[NV][VEC];
  #pragma unroll
  for (int i = 0; i < NV; i++)
    #pragma unroll
    for (int k = 0; k < VEC; k++) {
      s1[i][k] = s2[i][k] = 0.0f;
      if (HOLD) wg[HOLD ? i : 0][k] = w2[HOLD ? i : 0][k] = 0.0f;
    }
  if (HOLD) {
    #pragma unroll
    for (int i = 0; i < NV; i++) {
      if (in[i] && block) post_factors<TZ>(a, col[i], wg[HOLD ? i : 0]);
      if (in[i] && norm) params<TZ>(a.w2, a.w2_f32, col[i], w2[HOLD ? i : 0]);
    }
  }
  const long long step = (long long)gridDim.x * blockDim.y;
  long long t = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  Raw<TZ, VEC> z[NV], du[NV];
  Raw<TR, VEC> r[NV], dr2[NV];
  auto fetch = [&](long long row) {
    #pragma unroll
    for (int i = 0; i < NV; i++) {
      z[i].zero(); du[i].zero(); r[i].zero(); dr2[i].zero();
      if (row < a.T && in[i]) {
        if (block) z[i].load(static_cast<const TZ*>(a.z) + row * a.z_ld + col[i]);
        if (norm) {
          r[i].load(static_cast<const TR*>(a.r) + row * a.r_ld + col[i]);
          du[i].load(static_cast<const TZ*>(a.du) + row * a.du_ld + col[i]);
        }
        if (a.dr2) dr2[i].load(static_cast<const TR*>(a.dr2) + row * a.dr2_ld + col[i]);
      }
    }
  };
  if (HOLD) fetch(t);
  for (; t < a.T; t += step) {
    if (!HOLD) fetch(t);
    const float i1 = block ? a.rstd1[t] : 0.0f, i2 = norm ? a.rstd2[t] : 0.0f;
    const float gt = block && a.gate_kind == RBV_GATE_TOKEN ? param<TZ>(a.gate, a.gate_f32, t) : 1.0f;
    // w(i): scale * w1 (* gate per channel) of vector i; g(i): its gates per token or element
    auto load_w = [&](int i, float (&w)[VEC]) {
      #pragma unroll
      for (int k = 0; k < VEC; k++) w[k] = HOLD ? wg[HOLD ? i : 0][k] : 0.0f;
      if (!HOLD && in[i] && block) post_factors<TZ>(a, col[i], w);
    };
    auto load_g = [&](int i, float (&g)[VEC]) {
      #pragma unroll
      for (int k = 0; k < VEC; k++) g[k] = gt;
      if (FULL && in[i]) params<TZ>(a.gate, a.gate_f32, t * a.gate_ld + col[i], g);
    };
    float zh[NV][VEC], xh[NV][VEC], d[NV][VEC], s = 0.0f;                   // d: a, then D
    Raw<TR, VEC> e[NV];
    #pragma unroll
    for (int i = 0; i < NV; i++) {
      float w[VEC], g[VEC], v2[VEC];
      load_w(i, w);
      load_g(i, g);
      #pragma unroll
      for (int k = 0; k < VEC; k++) v2[k] = HOLD ? w2[HOLD ? i : 0][k] : 0.0f;
      if (!HOLD && in[i] && norm) params<TZ>(a.w2, a.w2_f32, col[i], v2);
      #pragma unroll
      for (int k = 0; k < VEC; k++) {
        zh[i][k] = z[i].get(k) * i1;
        xh[i][k] = fmaf(w[k] * g[k], zh[i][k], r[i].get(k)) * i2;
        const float v = du[i].get(k);
        s2[i][k] = fmaf(v, xh[i][k], s2[i][k]);
        d[i][k] = v * v2[k];
        s = fmaf(d[i][k], xh[i][k], s);
      }
      e[i] = dr2[i];
    }
    if (HOLD) fetch(t + step);
    const float c2 = norm ? row_sum(s) * inv_h : 0.0f;
    s = 0.0f;
    #pragma unroll
    for (int i = 0; i < NV; i++) {
      Raw<TR, VEC> o;
      float w[VEC], g[VEC];
      load_w(i, w);
      load_g(i, g);
      #pragma unroll
      for (int k = 0; k < VEC; k++) {
        d[i][k] = norm ? fmaf(i2, fmaf(-xh[i][k], c2, d[i][k]), e[i].get(k)) : e[i].get(k);
        o.set(k, d[i][k]);
        const float v = d[i][k] * zh[i][k];
        s = fmaf(FULL ? w[k] * g[k] : w[k], v, s);
        s1[i][k] = fmaf(g[k], v, s1[i][k]);
      }
      if (a.dr && in[i]) o.store(static_cast<TR*>(a.dr) + t * H + col[i]);
    }
    if (!block) continue;
    const float q = row_sum(s), c1 = q * gt * inv_h;
    if (a.gate_kind == RBV_GATE_TOKEN && a.dgate && threadIdx.x == 0) set_param<TZ>(a.dgate, a.gate_f32, t, q);
    #pragma unroll
    for (int i = 0; i < NV; i++) {
      if (!in[i]) continue;
      Raw<TZ, VEC> o;
      float w[VEC], g[VEC];
      load_w(i, w);
      load_g(i, g);
      #pragma unroll
      for (int k = 0; k < VEC; k++) {
        o.set(k, i1 * fmaf(-zh[i][k], c1, w[k] * g[k] * d[i][k]));
        if (FULL && a.dgate) set_param<TZ>(a.dgate, a.gate_f32, t * H + col[i] + k, w[k] * zh[i][k] * d[i][k]);
      }
      if (a.dz) o.store(static_cast<TZ*>(a.dz) + t * H + col[i]);
    }
  }
  if (!a.partial) return;
  const long long part = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  #pragma unroll
  for (int i = 0; i < NV; i++)
    #pragma unroll
    for (int k = 0; k < VEC; k++)
      if (in[i]) {
        a.partial[(2 * part) * H + col[i] + k] = s1[i][k];
        a.partial[(2 * part + 1) * H + col[i] + k] = s2[i][k];
      }
}

// Adds the CTAs' sums of 32 columns (x) of one kind (y), eight partial rows at a time.
template <typename TZ>
__global__ void __launch_bounds__(256) block_norm_sums_kernel(const __grid_constant__ rbv_norm_t a, int parts) {
  __shared__ float s_sum[8][32];
  pdl_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, kind = blockIdx.y;
  float s = 0.0f;
  if (c < a.H)
    for (int p = w; p < parts; p += 8) s += a.partial[(2ll * p + kind) * a.H + c];
  s_sum[w][lane] = s;
  __syncthreads();
  if (w || c >= a.H) return;
  #pragma unroll
  for (int i = 1; i < 8; i++) s += s_sum[i][lane];
  if (kind == 1) {
    if (a.dw2) set_param<TZ>(a.dw2, a.w2_f32, c, s);
    return;
  }
  const bool channel = a.gate_kind == RBV_GATE_CHANNEL;
  if (a.dw1) set_param<TZ>(a.dw1, a.w1_f32, c, s * a.scale * (channel ? param<TZ>(a.gate, a.gate_f32, c) : 1.0f));
  if (channel && a.dgate) set_param<TZ>(a.dgate, a.gate_f32, c, s * a.scale * param<TZ>(a.w1, a.w1_f32, c));
}

// ---- host side -------------------------------------------------------------------------------------------------------
struct Shape { int vec, nv, threads, rows, grid, sms; };

int norm_sms() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return sms;
}

// Threads per row: a warp up to 32 vectors, then a warp per 32 vectors up to 512 threads, which take up to 16 elements each;
// 1024 threads beyond.
Shape norm_shape(long long T, int H, int vec, bool backward, int sms) {
  Shape s{};
  s.vec = vec;
  s.sms = sms;
  const int vecs = (H + vec - 1) / vec;
  s.threads = vecs <= 32 ? 32 : vecs <= 512 ? (vecs + 31) / 32 * 32 : vecs <= 512 * 16 / vec ? 512 : 1024;
  s.nv = (vecs + s.threads - 1) / s.threads;
  s.rows = s.threads == 32 ? kNormWarpRows : 1;
  const long long rows = (T + s.rows - 1) / s.rows;
  // the backward pass takes 128 registers a thread; the forward pass asks (launch_shape)
  const long long fill = (long long)sms * (s.threads * s.rows <= 128 ? 4 : s.threads <= 256 ? 2 : 1);
  s.grid = (int)(rows < (backward ? fill : 16ll * sms) ? rows : backward ? fill : 16ll * sms);
  return s;
}

bool aligned(const void* p, long long ld, int vec, int size) {
  return !p || ((reinterpret_cast<uintptr_t>(p) % 16) == 0 && ld % vec == 0 && (vec * size) % 16 == 0);
}

bool valid(const rbv_norm_t& a) {
  if (a.T < 1 || a.H < 1 || a.H > RBV_NORM_MAX_HIDDEN || a.z_type < 0 || a.z_type > 2) return false;
  if (a.r_type != a.z_type && a.r_type != RBV_NORM_FP32) return false;
  if (!a.r || (!a.z && !a.w2) || (a.z && !a.w1)) return false;
  if (a.gate_kind < 0 || a.gate_kind > 3 || (a.gate_kind != RBV_GATE_NONE && !a.gate)) return false;
  return true;
}

template <typename TZ, typename TR, int VEC, int NV, int MAXT, bool BACKWARD>
cudaError_t launch_shape(const rbv_norm_t& a, const Shape& s, cudaStream_t st) {
  void (*kernel)(rbv_norm_t);
  const bool full = a.z && a.gate_kind == RBV_GATE_FULL;
  if constexpr (BACKWARD) kernel = full ? block_norm_backward_kernel<TZ, TR, VEC, NV, MAXT, true> : block_norm_backward_kernel<TZ, TR, VEC, NV, MAXT, false>;
  else kernel = full ? block_norm_kernel<TZ, TR, VEC, NV, MAXT, true> : block_norm_kernel<TZ, TR, VEC, NV, MAXT, false>;
  int grid = s.grid;
  if (!BACKWARD && grid > s.sms) {          // more rows than CTAs that fit at once: as many persistent CTAs as do
    static std::atomic<int> fits[33];       // CTAs per SM by warps per CTA, 0: not asked yet
    std::atomic<int>& known = fits[s.threads * s.rows / 32];
    int n = known.load(std::memory_order_relaxed);
    if (n == 0) {
      const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, s.threads * s.rows, 0);
      if (e != cudaSuccess) return e;
      known.store(n = n < 1 ? 1 : n, std::memory_order_relaxed);
    }
    grid = grid < n * s.sms ? grid : n * s.sms;
  }
  return launch_dependent(kernel, dim3(grid), dim3(s.threads, s.rows), 0, st, a);
}

template <typename TZ, typename TR, bool BACKWARD>
cudaError_t launch(const rbv_norm_t& a, const Shape& s, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(TZ), M = 16 / V;
  if (s.vec == V) {
    if (s.threads > 512) return s.nv <= M ? launch_shape<TZ, TR, V, M, 1024, BACKWARD>(a, s, st) : cudaErrorInvalidValue;
    if (s.nv <= 1) return launch_shape<TZ, TR, V, 1, 512, BACKWARD>(a, s, st);
    if (s.nv <= 2) return launch_shape<TZ, TR, V, 2, 512, BACKWARD>(a, s, st);
    return s.nv <= M ? launch_shape<TZ, TR, V, M, 512, BACKWARD>(a, s, st) : cudaErrorInvalidValue;
  }
  if (s.threads > 512) return s.nv <= 16 ? launch_shape<TZ, TR, 1, 16, 1024, BACKWARD>(a, s, st) : cudaErrorInvalidValue;
  if (s.nv <= 2) return launch_shape<TZ, TR, 1, 2, 512, BACKWARD>(a, s, st);
  if (s.nv <= 8) return launch_shape<TZ, TR, 1, 8, 512, BACKWARD>(a, s, st);
  return s.nv <= 16 ? launch_shape<TZ, TR, 1, 16, 512, BACKWARD>(a, s, st) : cudaErrorInvalidValue;
}

template <bool BACKWARD>
cudaError_t launch_typed(const rbv_norm_t& a, const Shape& s, cudaStream_t st) {
  const bool wide = a.r_type == RBV_NORM_FP32;
  switch (a.z_type) {
    case RBV_NORM_BF16: return wide ? launch<__nv_bfloat16, float, BACKWARD>(a, s, st) : launch<__nv_bfloat16, __nv_bfloat16, BACKWARD>(a, s, st);
    case RBV_NORM_FP16: return wide ? launch<__half, float, BACKWARD>(a, s, st) : launch<__half, __half, BACKWARD>(a, s, st);
    default: return launch<float, float, BACKWARD>(a, s, st);
  }
}

int type_size(int t) { return t == RBV_NORM_FP32 ? 4 : 2; }

// 16-byte vectors of z where every row of every tensor starts at one, single elements otherwise.
int vector_width(const rbv_norm_t& a, bool backward) {
  const int vec = 16 / type_size(a.z_type), zs = type_size(a.z_type), rs = type_size(a.r_type);
  bool ok = a.H % vec == 0 && aligned(a.z, a.z_ld, vec, zs) && aligned(a.r, a.r_ld, vec, rs) && aligned(a.w1, 0, vec, zs) &&
            aligned(a.w2, 0, vec, zs) && (a.gate_kind != RBV_GATE_CHANNEL || aligned(a.gate, 0, vec, zs)) &&
            (a.gate_kind != RBV_GATE_FULL || aligned(a.gate, a.gate_ld, vec, zs));
  if (backward) ok = ok && aligned(a.dr2, a.dr2_ld, vec, rs) && aligned(a.du, a.du_ld, vec, zs) && aligned(a.dz, a.H, vec, zs) && aligned(a.dr, a.H, vec, rs);
  else ok = ok && aligned(a.r2, a.H, vec, rs) && aligned(a.u, a.H, vec, zs);
  return ok ? vec : 1;
}

}  // namespace
}  // namespace rbv

using namespace rbv;

extern "C" int rbv_block_norm_parts(long long T, int H, int z_type) {
  if (T < 1 || H < 1 || H > RBV_NORM_MAX_HIDDEN) return 0;
  const int sms = norm_sms();
  const int vec = H % (16 / type_size(z_type)) == 0 ? 16 / type_size(z_type) : 1;
  const Shape a = norm_shape(T, H, vec, true, sms), b = norm_shape(T, H, 1, true, sms);   // (whichever is taken)
  const int pa = a.grid * a.rows, pb = b.grid * b.rows;
  return pa > pb ? pa : pb;
}

extern "C" int rbv_block_norm(const rbv_norm_t* call, void* stream) {
  if (!call || !valid(*call)) return (int)cudaErrorInvalidValue;
  const rbv_norm_t& a = *call;
  if ((a.z && !a.r2) || (a.w2 && !a.u)) return (int)cudaErrorInvalidValue;
  const int sms = norm_sms();
  if (sms < 1) return (int)cudaErrorUnknown;
  return (int)launch_typed<false>(a, norm_shape(a.T, a.H, vector_width(a, false), false, sms), static_cast<cudaStream_t>(stream));
}

extern "C" int rbv_block_norm_backward(const rbv_norm_t* call, void* stream) {
  if (!call || !valid(*call)) return (int)cudaErrorInvalidValue;
  const rbv_norm_t& a = *call;
  const bool sums = a.dw1 || a.dw2 || (a.gate_kind == RBV_GATE_CHANNEL && a.dgate);
  if ((a.z && !a.rstd1) || (a.w2 && a.du && !a.rstd2) || (sums && !a.partial)) return (int)cudaErrorInvalidValue;
  const int sms = norm_sms();
  if (sms < 1) return (int)cudaErrorUnknown;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  rbv_norm_t b = a;
  if (!sums) b.partial = nullptr;
  const Shape s = norm_shape(a.T, a.H, vector_width(a, true), true, sms);
  const cudaError_t e = launch_typed<true>(b, s, st);
  if (e != cudaSuccess || !sums) return (int)e;
  const int parts = s.grid * s.rows;
  const dim3 grid((a.H + 31) / 32, 2);
  switch (a.z_type) {
    case RBV_NORM_BF16: return (int)launch_dependent(block_norm_sums_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, b, parts);
    case RBV_NORM_FP16: return (int)launch_dependent(block_norm_sums_kernel<__half>, grid, dim3(256), 0, st, b, parts);
    default: return (int)launch_dependent(block_norm_sums_kernel<float>, grid, dim3(256), 0, st, b, parts);
  }
}
