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
// read r2 in place of r).  All sums are held in 32 bits and added in a fixed order.
//
// Two pairs of kernels.  Where there are more rows than SMs, of 2 KB or more, one persistent CTA per SM works on several rows
// at a time, each by a group of warps of its own (block_norm_rows_*): a row passes through four dependent steps, wait, sum,
// sum, store, so what keeps HBM busy is rows in work: four forward and two backward for 4096 elements (there a thread also holds
// the sums over the tokens of its columns), up to eight for shorter rows, 32 and 16 for the shortest, of one warp each.  A group's
// leader fetches its next row into shared memory with one bulk copy per tensor; the weights are in shared memory too.  With one
// row per CTA of 512 threads and the weights in registers 8192 x 4096 in bf16 took 59 us forward, and 4096 x 4096 with the
// residual in fp32 75 us backward; now 47 and 63.
// Short rows, unaligned ones, and few tokens go straight to the registers of one group of threads per row.
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
#include "kernels/sm100_ptx.cuh"
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

__device__ __forceinline__ void lds(uint2& v, uint32_t at) {
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
}

// VEC consecutive elements as they are in memory; VEC * sizeof(T) is a multiple of 16, or VEC is 1.
template <typename T, int VEC>
struct Raw {
  using Word = uint4;
  static constexpr int Q = VEC * (int)sizeof(T) / (int)sizeof(Word);
  Word q[Q];
  __device__ __forceinline__ void load(const T* p) {
    #pragma unroll
    for (int i = 0; i < Q; i++) q[i] = __ldg(reinterpret_cast<const Word*>(p) + i);
  }
  __device__ __forceinline__ void store(T* p) const {
    #pragma unroll
    for (int i = 0; i < Q; i++) reinterpret_cast<Word*>(p)[i] = q[i];
  }
  __device__ __forceinline__ void zero() {
    #pragma unroll
    for (int i = 0; i < Q; i++) q[i] = Word{};
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

// ---- several rows in work per CTA ----------------------------------------------------------------------------------------
constexpr int kNormSlots = 64;

struct NormShared {
  uint64_t full[kNormSlots];
  float red[2][16][32];                     // a sum's parts by turn, group (of several warps: 8 at most) and warp (32 at most)
  int abort;
};

// blockDim.y groups of blockDim.x threads.  The dynamic shared memory holds the weights as 32-bit factors (scale * w1 * gate
// per channel, then w2) and the groups' slots: the tensors of a row, one behind the other.  (Addresses of shared memory as
// numbers: through generic pointers the backward kernel executed twice the instructions, 95 us for the case above.)
template <typename TZ, typename TR, bool BACKWARD, bool FULL>
struct RowGroup {
  const rbv_norm_t& a;
  NormShared& sh;
  uint32_t factors, slots;
  int group, stages, stage = 0, turn = 0;
  uint32_t phase = 0, r_at, du_at, g_at, bytes;
  bool ok = true;
  __device__ __forceinline__ RowGroup(const rbv_norm_t& a_, NormShared& sh_, uint8_t* dyn, int stages_)
      : a(a_), sh(sh_), factors(sm100::smem_u32(dyn)), group(threadIdx.y), stages(stages_) {
    const uint32_t z = a.H * (uint32_t)sizeof(TZ), r = a.H * (uint32_t)sizeof(TR);
    r_at = a.z ? z : 0u;
    du_at = r_at + (BACKWARD && !(a.du && a.w2) ? 0u : r);
    g_at = du_at + (BACKWARD && a.du && a.w2 ? z : 0u);
    bytes = g_at + (FULL ? a.H * (a.gate_f32 ? 4u : (uint32_t)sizeof(TZ)) : 0u);
    slots = factors + 8u * a.H + (uint32_t)(group * stages) * bytes;
  }
  __device__ __forceinline__ uint32_t slot() const { return slots + (uint32_t)stage * bytes; }
  __device__ __forceinline__ uint64_t* bar(int s) const { return &sh.full[group * stages + s]; }
  __device__ __forceinline__ static void copy(uint32_t dst, const void* src, uint32_t n, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(n), "r"(sm100::smem_u32(bar)) : "memory");
  }
  __device__ __forceinline__ void fill(int s, long long t) {       // the group's first thread
    const uint32_t to = slots + (uint32_t)s * bytes;
    uint64_t* b = bar(s);
    sm100::mbar_arrive_expect_tx(b, bytes);
    if (r_at) copy(to, static_cast<const TZ*>(a.z) + t * a.z_ld, r_at, b);
    if (du_at > r_at) copy(to + r_at, static_cast<const TR*>(a.r) + t * a.r_ld, du_at - r_at, b);
    if (g_at > du_at) copy(to + du_at, static_cast<const TZ*>(a.du) + t * a.du_ld, g_at - du_at, b);
    if (FULL) {
      const long long at = t * a.gate_ld;
      copy(to + g_at, a.gate_f32 ? static_cast<const void*>(static_cast<const float*>(a.gate) + at)
                                 : static_cast<const void*>(static_cast<const TZ*>(a.gate) + at), bytes - g_at, b);
    }
  }
  __device__ __forceinline__ void wait() { ok = sm100::mbar_wait(bar(stage), phase, &sh.abort) && ok; }
  __device__ __forceinline__ void next() {
    if (++stage == stages) { stage = 0; phase ^= 1u; }
  }
  __device__ __forceinline__ void sync() {
    if (blockDim.x > 32) asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(blockDim.x) : "memory");
    else __syncwarp();
  }
  // Sum over the group; a barrier of the group lies behind everything that its threads did before.
  __device__ __forceinline__ float sum(float v) {
    #pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (blockDim.x == 32) return v;
    float* r = sh.red[turn][group];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
    sync();
    float s = 0.0f;
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) s += r[w];
    return s;
  }
};

// Two neighbouring elements in one 64-bit register, two operations per instruction: the loops over a row's elements are what a
// CTA with few warps (their registers hold the sums over the tokens) spends its time on.
struct F2 {
  unsigned long long v;
  __device__ __forceinline__ float lo() const { return __uint_as_float((unsigned)v); }
  __device__ __forceinline__ float hi() const { return __uint_as_float((unsigned)(v >> 32)); }
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 f2(float both) { return f2(both, both); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// Four neighbouring elements as they are in memory.
constexpr int kRowsVec = 4;
template <typename T>
struct Four {
  uint2 q;
  __device__ __forceinline__ void load(const T* p) { q = __ldg(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ void load_shared(uint32_t at) { lds(q, at); }
  __device__ __forceinline__ void get(F2 (&v)[2]) const;
  __device__ __forceinline__ static void store(T* p, const F2 (&v)[2]);
};
template <> __device__ __forceinline__ void Four<__nv_bfloat16>::get(F2 (&v)[2]) const {
  v[0] = f2(__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xffff0000u));
  v[1] = f2(__uint_as_float(q.y << 16), __uint_as_float(q.y & 0xffff0000u));
}
template <> __device__ __forceinline__ void Four<__nv_bfloat16>::store(__nv_bfloat16* p, const F2 (&v)[2]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v[0].lo(), v[0].hi()), b = __floats2bfloat162_rn(v[1].lo(), v[1].hi());
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}
template <> __device__ __forceinline__ void Four<__half>::get(F2 (&v)[2]) const {
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&q.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&q.y));
  v[0] = f2(a.x, a.y);
  v[1] = f2(b.x, b.y);
}
template <> __device__ __forceinline__ void Four<__half>::store(__half* p, const F2 (&v)[2]) {
  const __half2 a = __floats2half2_rn(v[0].lo(), v[0].hi()), b = __floats2half2_rn(v[1].lo(), v[1].hi());
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}
template <>
struct Four<float> {
  ulonglong2 q;
  __device__ __forceinline__ void load(const float* p) { q = __ldg(reinterpret_cast<const ulonglong2*>(p)); }
  __device__ __forceinline__ void load_shared(uint32_t at) {
    asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(q.x), "=l"(q.y) : "r"(at) : "memory");
  }
  __device__ __forceinline__ void get(F2 (&v)[2]) const { v[0].v = q.x; v[1].v = q.y; }
  __device__ __forceinline__ static void store(float* p, const F2 (&v)[2]) { *reinterpret_cast<ulonglong2*>(p) = make_ulonglong2(v[0].v, v[1].v); }
};
template <typename T>
__device__ __forceinline__ void shared4(uint32_t at, F2 (&v)[2]) {
  Four<T> q;
  q.load_shared(at);
  q.get(v);
}
// four gates of a slot
template <typename T>
__device__ __forceinline__ void gates4(uint32_t at, int f32, uint32_t c, F2 (&v)[2]) {
  if (f32) shared4<float>(at + c * 4u, v);
  else shared4<T>(at + c * (uint32_t)sizeof(T), v);
}

// Barriers and weights of a CTA; all threads.
template <typename TZ>
__device__ __forceinline__ void rows_begin(const rbv_norm_t& a, NormShared& sh, uint8_t* dyn, int slots, bool norm) {
  const int tid = threadIdx.y * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y;
  if (tid == 0) {
    for (int i = 0; i < slots; i++) sm100::mbar_init(&sh.full[i], 1);
    sh.abort = 0;
    sm100::mbar_fence_init();
  }
  pdl_trigger();
  pdl_wait();
  float* f = reinterpret_cast<float*>(dyn);
  for (int c = tid; c < a.H; c += threads) {
    if (a.z) {
      float w[1];
      post_factors<TZ>(a, c, w);
      f[c] = w[0];
    }
    if (norm) f[a.H + c] = param<TZ>(a.w2, a.w2_f32, c);
  }
  __syncthreads();
}

constexpr int kRowsNV = 4;                // fours of elements per thread

template <typename TZ, typename TR, bool FULL>
__global__ void __launch_bounds__(1024, 1) block_norm_rows_kernel(const __grid_constant__ rbv_norm_t a, int stages) {
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ NormShared sh;
  const int H = a.H;
  const float inv_h = 1.0f / (float)H;
  const bool block = a.z != nullptr, norm = a.w2 != nullptr;
  rows_begin<TZ>(a, sh, dyn, stages * blockDim.y, norm);
  RowGroup<TZ, TR, false, FULL> g(a, sh, dyn, stages);
  const long long step = (long long)gridDim.x * blockDim.y;
  long long t = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (threadIdx.x == 0)
    for (int i = 0; i < stages && t + i * step < a.T; i++) g.fill(i, t + i * step);
  const uint32_t c0 = threadIdx.x * kRowsVec, dc = blockDim.x * kRowsVec;
  for (; t < a.T; t += step) {
    g.wait();
    const uint32_t slot = g.slot();
    F2 x[kRowsNV][2], s = f2(0.0f);
    float f = 0.0f;
    if (block) {
      #pragma unroll
      for (int i = 0; i < kRowsNV; i++) {
        const uint32_t c = c0 + i * dc;
        if (c >= (uint32_t)H) break;
        F2 z[2];
        shared4<TZ>(slot + c * (uint32_t)sizeof(TZ), z);
        s = fma2(z[0], z[0], s);
        s = fma2(z[1], z[1], s);
      }
      f = rsqrtf(fmaf(g.sum(s.lo() + s.hi()), inv_h, a.eps));
      if (!g.ok) f = __int_as_float(0x7fffffff);                   // (a copy that never came: the row is NaN)
      if (a.rstd1 && threadIdx.x == 0) a.rstd1[t] = f;
      if (a.gate_kind == RBV_GATE_TOKEN) f *= param<TZ>(a.gate, a.gate_f32, t);
    }
    s = f2(0.0f);
    const F2 ff = f2(f);
    #pragma unroll
    for (int i = 0; i < kRowsNV; i++) {
      const uint32_t c = c0 + i * dc;
      if (c >= (uint32_t)H) break;
      shared4<TR>(slot + g.r_at + c * (uint32_t)sizeof(TR), x[i]);
      if (block) {
        F2 z[2], w[2];
        shared4<TZ>(slot + c * (uint32_t)sizeof(TZ), z);
        shared4<float>(g.factors + 4u * c, w);
        if (FULL) {
          F2 e[2];
          gates4<TZ>(slot + g.g_at, a.gate_f32, c, e);
          w[0] = mul2(w[0], e[0]);
          w[1] = mul2(w[1], e[1]);
        }
        x[i][0] = fma2(w[0], mul2(z[0], ff), x[i][0]);
        x[i][1] = fma2(w[1], mul2(z[1], ff), x[i][1]);
        Four<TR>::store(static_cast<TR*>(a.r2) + t * H + c, x[i]);
      }
      s = fma2(x[i][0], x[i][0], s);
      s = fma2(x[i][1], x[i][1], s);
    }
    float q = s.lo() + s.hi();
    if (norm) q = g.sum(q);
    else g.sync();
    if (threadIdx.x == 0 && t + stages * step < a.T) g.fill(g.stage, t + stages * step);      // everybody has the row
    g.next();
    if (!norm) continue;
    float i2 = rsqrtf(fmaf(q, inv_h, a.eps));
    if (!g.ok) i2 = __int_as_float(0x7fffffff);
    if (a.rstd2 && threadIdx.x == 0) a.rstd2[t] = i2;
    const F2 ii = f2(i2);
    #pragma unroll
    for (int i = 0; i < kRowsNV; i++) {
      const uint32_t c = c0 + i * dc;
      if (c >= (uint32_t)H) break;
      F2 w[2];
      shared4<float>(g.factors + 4u * (H + c), w);
      w[0] = mul2(mul2(x[i][0], ii), w[0]);
      w[1] = mul2(mul2(x[i][1], ii), w[1]);
      Four<TZ>::store(static_cast<TZ*>(a.u) + t * H + c, w);
    }
  }
}

// With f = i1 * (gate per token), x = r2:  a = du i2 w2;  D = dr2 + a - i2^2 mean(a x) x;  v = D z;  q = i1 sum(w v);
// dz = f w D - i1^2 mean(...) z: the row's factors are taken out of the loops.
template <typename TZ, typename TR, bool FULL>
__global__ void __launch_bounds__(512, 1) block_norm_rows_backward_kernel(const __grid_constant__ rbv_norm_t a, int stages) {
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ NormShared sh;
  const int H = a.H;
  const float inv_h = 1.0f / (float)H;
  const bool block = a.z != nullptr, norm = a.w2 != nullptr && a.du != nullptr;
  rows_begin<TZ>(a, sh, dyn, stages * blockDim.y, norm);
  RowGroup<TZ, TR, true, FULL> g(a, sh, dyn, stages);
  F2 s1[kRowsNV][2], s2[kRowsNV][2];
  #pragma unroll
  for (int i = 0; i < kRowsNV; i++)
    #pragma unroll
    for (int k = 0; k < 2; k++) s1[i][k] = s2[i][k] = f2(0.0f);
  const long long step = (long long)gridDim.x * blockDim.y;
  long long t = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (threadIdx.x == 0)
    for (int i = 0; i < stages && t + i * step < a.T; i++) g.fill(i, t + i * step);
  const uint32_t c0 = threadIdx.x * kRowsVec, dc = blockDim.x * kRowsVec;
  // a row's numbers are fetched while the row before is in work
  float i1_next = 0.0f, i2_next = 0.0f, gt_next = 1.0f;
  auto numbers = [&](long long row) {
    if (row >= a.T) return;
    if (block) i1_next = a.rstd1[row];
    if (norm) i2_next = a.rstd2[row];
    if (block && a.gate_kind == RBV_GATE_TOKEN) gt_next = param<TZ>(a.gate, a.gate_f32, row);
  };
  numbers(t);
  for (; t < a.T; t += step) {
    float i1 = i1_next, i2 = i2_next;
    const float gt = gt_next;
    numbers(t + step);
    Four<TR> dr2[kRowsNV];                                         // wanted in the second step only
    if (a.dr2)
      #pragma unroll
      for (int i = 0; i < kRowsNV; i++) {
        const uint32_t c = c0 + i * dc;
        if (c >= (uint32_t)H) break;
        dr2[i].load(static_cast<const TR*>(a.dr2) + t * a.dr2_ld + c);
      }
    g.wait();
    if (!g.ok) i1 = i2 = __int_as_float(0x7fffffff);               // (a copy that never came: the row is NaN)
    const float f = i1 * gt;
    const F2 ff = f2(f), ii = f2(i2);
    const uint32_t slot = g.slot();
    F2 d[kRowsNV][2], x[kRowsNV][2], s = f2(0.0f);                 // d: a, then D
    Four<TZ> zq[kRowsNV];
    if (block)
      #pragma unroll
      for (int i = 0; i < kRowsNV; i++) {
        const uint32_t c = c0 + i * dc;
        if (c >= (uint32_t)H) break;
        zq[i].load_shared(slot + c * (uint32_t)sizeof(TZ));
      }
    if (norm) {
      #pragma unroll
      for (int i = 0; i < kRowsNV; i++) {
        const uint32_t c = c0 + i * dc;
        if (c >= (uint32_t)H) break;
        F2 du[2], w2[2];
        shared4<TR>(slot + g.r_at + c * (uint32_t)sizeof(TR), x[i]);
        shared4<TZ>(slot + g.du_at + c * (uint32_t)sizeof(TZ), du);
        shared4<float>(g.factors + 4u * (H + c), w2);
        if (block) {
          F2 z[2], w[2], e[2];
          zq[i].get(z);
          shared4<float>(g.factors + 4u * c, w);
          if (FULL) gates4<TZ>(slot + g.g_at, a.gate_f32, c, e);
          #pragma unroll
          for (int k = 0; k < 2; k++) x[i][k] = fma2(FULL ? mul2(w[k], e[k]) : w[k], mul2(z[k], ff), x[i][k]);
        }
        #pragma unroll
        for (int k = 0; k < 2; k++) {
          const F2 v = mul2(du[k], ii);
          s2[i][k] = fma2(v, x[i][k], s2[i][k]);
          d[i][k] = mul2(v, w2[k]);
          s = fma2(d[i][k], x[i][k], s);
        }
      }
    }
    const F2 k2 = f2(norm ? -i2 * i2 * g.sum(s.lo() + s.hi()) * inv_h : 0.0f);
    s = f2(0.0f);
    #pragma unroll
    for (int i = 0; i < kRowsNV; i++) {
      const uint32_t c = c0 + i * dc;
      if (c >= (uint32_t)H) break;
      F2 e2[2] = {f2(0.0f), f2(0.0f)};
      if (a.dr2) dr2[i].get(e2);
      #pragma unroll
      for (int k = 0; k < 2; k++) d[i][k] = norm ? add2(fma2(k2, x[i][k], d[i][k]), e2[k]) : e2[k];
      if (a.dr) Four<TR>::store(static_cast<TR*>(a.dr) + t * H + c, d[i]);
      if (block) {
        F2 z[2], w[2], e[2];
        zq[i].get(z);
        shared4<float>(g.factors + 4u * c, w);
        if (FULL) gates4<TZ>(slot + g.g_at, a.gate_f32, c, e);
        F2 v[2] = {mul2(d[i][0], z[0]), mul2(d[i][1], z[1])};
        if (FULL) {
          if (a.dgate) {
            const F2 i11 = f2(i1);
            const F2 dg[2] = {mul2(mul2(w[0], i11), v[0]), mul2(mul2(w[1], i11), v[1])};
            if (a.gate_f32) Four<float>::store(static_cast<float*>(a.dgate) + t * H + c, dg);
            else Four<TZ>::store(static_cast<TZ*>(a.dgate) + t * H + c, dg);
          }
          v[0] = mul2(v[0], e[0]);
          v[1] = mul2(v[1], e[1]);
        }
        #pragma unroll
        for (int k = 0; k < 2; k++) {
          s1[i][k] = fma2(ff, v[k], s1[i][k]);
          s = fma2(w[k], v[k], s);
        }
      }
    }
    float q = 0.0f;
    if (block) q = i1 * g.sum(s.lo() + s.hi());
    else g.sync();
    // everybody has what it needs of the row, but for a gate per element
    const bool refill = threadIdx.x == 0 && t + stages * step < a.T;
    if (!FULL && refill) g.fill(g.stage, t + stages * step);
    if (block) {
      const F2 k1 = f2(-i1 * i1 * gt * q * inv_h);
      if (a.gate_kind == RBV_GATE_TOKEN && a.dgate && threadIdx.x == 0) set_param<TZ>(a.dgate, a.gate_f32, t, q);
      if (a.dz)
        #pragma unroll
        for (int i = 0; i < kRowsNV; i++) {
          const uint32_t c = c0 + i * dc;
          if (c >= (uint32_t)H) break;
          F2 z[2], w[2], e[2];
          zq[i].get(z);
          shared4<float>(g.factors + 4u * c, w);
          if (FULL) gates4<TZ>(slot + g.g_at, a.gate_f32, c, e);
          #pragma unroll
          for (int k = 0; k < 2; k++) w[k] = fma2(k1, z[k], mul2(mul2(FULL ? mul2(w[k], e[k]) : w[k], ff), d[i][k]));
          Four<TZ>::store(static_cast<TZ*>(a.dz) + t * H + c, w);
        }
    }
    if (FULL) {
      g.sync();
      if (refill) g.fill(g.stage, t + stages * step);
    }
    g.next();
  }
  if (!a.partial) return;
  // the groups' sums over their rows, added in shared memory (every copy into it has been waited for), one pair of rows per CTA
  __syncthreads();
  float* sums = reinterpret_cast<float*>(dyn);
  for (int k = 0; k < (int)blockDim.y; k++) {
    if ((int)threadIdx.y == k)
      #pragma unroll
      for (int i = 0; i < kRowsNV; i++) {
        const uint32_t c = c0 + i * dc;
        if (c >= (uint32_t)H) break;
        #pragma unroll
        for (int kind = 0; kind < 2; kind++) {
          F2 v[2] = {kind ? s2[i][0] : s1[i][0], kind ? s2[i][1] : s1[i][1]}, before[2];
          float* at = sums + kind * H + c;
          if (k) {
            shared4<float>(sm100::smem_u32(at), before);
            v[0] = add2(before[0], v[0]);
            v[1] = add2(before[1], v[1]);
          }
          Four<float>::store(k + 1 < (int)blockDim.y ? at : a.partial + (2ll * blockIdx.x + kind) * H + c, v);
        }
      }
    __syncthreads();
  }
}

// Adds the CTAs' sums of 32 columns (x) of one kind (y): 16 warps take every sixteenth partial row, several at a time.
template <typename TZ>
__global__ void __launch_bounds__(512) block_norm_sums_kernel(const __grid_constant__ rbv_norm_t a, int parts) {
  __shared__ float s_sum[16][32];
  pdl_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, kind = blockIdx.y;
  float s = 0.0f;
  if (c < a.H) {
    const float* from = a.partial + (long long)kind * a.H + c;
    #pragma unroll 5
    for (int p = w; p < parts; p += 16) s += __ldcg(from + 2ll * p * a.H);
  }
  s_sum[w][lane] = s;
  __syncthreads();
  if (w || c >= a.H) return;
  #pragma unroll
  for (int i = 1; i < 16; i++) s += s_sum[i][lane];
  if (kind == 1) {
    if (a.dw2) set_param<TZ>(a.dw2, a.w2_f32, c, s);
    return;
  }
  const bool channel = a.gate_kind == RBV_GATE_CHANNEL;
  if (a.dw1) set_param<TZ>(a.dw1, a.w1_f32, c, s * a.scale * (channel ? param<TZ>(a.gate, a.gate_f32, c) : 1.0f));
  if (channel && a.dgate) set_param<TZ>(a.dgate, a.gate_f32, c, s * a.scale * param<TZ>(a.w1, a.w1_f32, c));
}

// ---- host side -------------------------------------------------------------------------------------------------------
struct Shape { int vec, nv, threads, rows, grid, sms, stages; size_t smem; };      // stages > 0: several rows per CTA

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

// Several rows in work per CTA: 16 elements a thread, in up to 1024 threads forward (64 registers) and 512 backward (128), as
// many groups as threads and slots allow.
Shape rows_shape(long long T, int H, size_t row_bytes, bool backward, int sms) {
  Shape s{};
  s.vec = kRowsVec;
  s.sms = sms;
  const int vecs = H / kRowsVec, most = kRowsNV, threads = backward ? 512 : 1024;
  s.threads = ((vecs + most - 1) / most + 31) / 32 * 32;
  if (s.threads > threads) return s;
  s.nv = (vecs + s.threads - 1) / s.threads;
  const size_t room = 227 * 1024 - sizeof(NormShared) - 512, weights = (size_t)8 * H;
  if (weights + row_bytes > room) return s;
  const size_t slots = (room - weights) / row_bytes;
  s.rows = threads / s.threads;
  if (s.threads > 32 && s.rows > 8) s.rows = 8;              // (barriers)
  if ((size_t)s.rows > slots) s.rows = (int)slots;
  s.stages = (int)(slots / s.rows);
  if (s.stages > kNormSlots / s.rows) s.stages = kNormSlots / s.rows;
  if (s.stages > 4) s.stages = 4;
  s.smem = weights + row_bytes * s.rows * s.stages;
  const long long ctas = (T + s.rows - 1) / s.rows;
  s.grid = (int)(ctas < sms ? ctas : sms);
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
    static std::atomic<int> fits[2][33];    // CTAs per SM by kernel and warps per CTA, 0: not asked yet
    std::atomic<int>& known = fits[full][s.threads * s.rows / 32];
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
cudaError_t launch_rows(const rbv_norm_t& a, const Shape& s, cudaStream_t st) {
  void (*kernel)(rbv_norm_t, int);
  const bool full = a.z && a.gate_kind == RBV_GATE_FULL;
  if constexpr (BACKWARD) kernel = full ? block_norm_rows_backward_kernel<TZ, TR, true> : block_norm_rows_backward_kernel<TZ, TR, false>;
  else kernel = full ? block_norm_rows_kernel<TZ, TR, true> : block_norm_rows_kernel<TZ, TR, false>;
  static std::atomic<unsigned long long> allowed[2];        // by kernel, a bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(allowed[full].load(std::memory_order_relaxed) >> dev & 1)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(227 * 1024 - sizeof(NormShared) - 512));
    if (e != cudaSuccess) return e;
    if (dev < 64) allowed[full].fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  return launch_dependent(kernel, dim3(s.grid), dim3(s.threads, s.rows), s.smem, st, a, s.stages);
}

template <typename TZ, typename TR, bool BACKWARD>
cudaError_t launch(const rbv_norm_t& a, const Shape& s, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(TZ), M = 16 / V;
  if (s.stages) return launch_rows<TZ, TR, BACKWARD>(a, s, st);
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

// Bytes of a row of the tensors that are read.
size_t row_bytes(const rbv_norm_t& a, bool backward) {
  const size_t z = (size_t)a.H * type_size(a.z_type), r = (size_t)a.H * type_size(a.r_type);
  size_t n = a.z ? z : 0;
  if (a.z && a.gate_kind == RBV_GATE_FULL) n += a.gate_f32 ? (size_t)a.H * 4 : z;
  if (!backward) return n + r;
  return n + (a.du && a.w2 ? r + z : 0);      // (dr2 goes to registers)
}

// 16-byte vectors of z where every row of every tensor starts at one, single elements otherwise.
Shape choose_shape(const rbv_norm_t& a, bool backward, int sms) {
  const int zs = type_size(a.z_type), rs = type_size(a.r_type), vec = 16 / zs;
  bool ok = a.H % vec == 0 && aligned(a.z, a.z_ld, vec, zs) && aligned(a.r, a.r_ld, vec, rs) && aligned(a.w1, 0, vec, zs) &&
            aligned(a.w2, 0, vec, zs) && (a.gate_kind != RBV_GATE_CHANNEL || aligned(a.gate, 0, vec, zs)) &&
            (a.gate_kind != RBV_GATE_FULL || aligned(a.gate, a.gate_ld, vec, zs));
  if (backward)
    ok = ok && aligned(a.dr2, a.dr2_ld, vec, rs) && aligned(a.du, a.du_ld, vec, zs) && aligned(a.dz, a.H, vec, zs) && aligned(a.dr, a.H, vec, rs) &&
         (a.gate_kind != RBV_GATE_FULL || aligned(a.dgate, a.H, vec, zs)) && aligned(a.partial, 0, vec, zs);
  else ok = ok && aligned(a.r2, a.H, vec, rs) && aligned(a.u, a.H, vec, zs);
  const size_t bytes = row_bytes(a, backward);
  if (ok && (size_t)a.H * zs >= 2048 && a.T > sms && bytes > 0) {
    const Shape s = rows_shape(a.T, a.H, bytes, backward, sms);
    if (s.stages) return s;
  }
  return norm_shape(a.T, a.H, ok ? vec : 1, backward, sms);
}

}  // namespace
}  // namespace rbv

using namespace rbv;

extern "C" int rbv_block_norm_parts(long long T, int H, int z_type) {
  if (T < 1 || H < 1 || H > RBV_NORM_MAX_HIDDEN) return 0;
  const int sms = norm_sms();
  const int vec = H % (16 / type_size(z_type)) == 0 ? 16 / type_size(z_type) : 1;
  // whichever shape is taken (several rows per CTA: a CTA per SM)
  const Shape a = norm_shape(T, H, vec, true, sms), b = norm_shape(T, H, 1, true, sms);
  const int most = a.grid * a.rows > b.grid * b.rows ? a.grid * a.rows : b.grid * b.rows;
  return most > sms ? most : sms;
}

extern "C" int rbv_block_norm(const rbv_norm_t* call, void* stream) {
  if (!call || !valid(*call)) return (int)cudaErrorInvalidValue;
  const rbv_norm_t& a = *call;
  if ((a.z && !a.r2) || (a.w2 && !a.u)) return (int)cudaErrorInvalidValue;
  const int sms = norm_sms();
  if (sms < 1) return (int)cudaErrorUnknown;
  return (int)launch_typed<false>(a, choose_shape(a, false, sms), static_cast<cudaStream_t>(stream));
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
  const Shape s = choose_shape(a, true, sms);
  const cudaError_t e = launch_typed<true>(b, s, st);
  if (e != cudaSuccess || !sums) return (int)e;
  const int parts = s.stages ? s.grid : s.grid * s.rows;      // (several rows per CTA: it has added them up)
  const dim3 grid((a.H + 31) / 32, 2);
  switch (a.z_type) {
    case RBV_NORM_BF16: return (int)launch_dependent(block_norm_sums_kernel<__nv_bfloat16>, grid, dim3(512), 0, st, b, parts);
    case RBV_NORM_FP16: return (int)launch_dependent(block_norm_sums_kernel<__half>, grid, dim3(512), 0, st, b, parts);
    default: return (int)launch_dependent(block_norm_sums_kernel<float>, grid, dim3(512), 0, st, b, parts);
  }
}
