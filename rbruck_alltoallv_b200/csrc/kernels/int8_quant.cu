// Rows of bf16 -> 8-bit integers with one scale per row:  s = max|x| / 127,  q = round-to-nearest-even(x / s).
//
// Bound by HBM: 2 bytes read and 1 written per element.  A row stays in the registers of the threads that share it between the
// maximum and the quantisation (up to 16384 elements; longer rows are read twice).  The quotient is the correctly rounded
// one, as x / s in 32 bits gives it: x times the reciprocal decides, except next to a half, where the division is done (a
// division for every element would take longer than its bytes).  A row that holds an infinity or a NaN gets the scale NaN, so
// that whatever is made of it is NaN; one whose values are all below 2^-100 counts as zeros (scale 1).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kernels/int8_quant.cuh"
#include "kernels/pdl.cuh"
#include "rbv/moe.h"

namespace rbv {
namespace {

using namespace quant;

struct QuantArgs {
  const __nv_bfloat16* x;
  long long rows, ldx;
  const int* used;            // optional: rows that hold anything
  int K;                      // a multiple of 8
  int8_t* q;                  // [rows, K]
  float* scale;               // [rows]
  int* zero;                  // optional: `zeros` words to set to zero (counters of the kernel behind this one)
  int zeros;
};

// A row per blockDim.x threads (a warp, or the CTA); NV vectors per thread in registers, 0: read the row twice.  CTAS: of 512
// threads per SM.  Three leave 40 registers and spill a few, which pays only where CTAs are so large that with 57 registers no
// more than two fit (4096 rows of 11136: 43.7 us with two, 35.4 with three; 16384 rows of 4096: 47.6 and 48.3; 2000 of 2048: 4.8
// and 6.6).
template <int NV, int CTAS>
__global__ void __launch_bounds__(512, CTAS) quantize_rows_int8_kernel(const __grid_constant__ QuantArgs a) {
  __shared__ float red[2][16];
  pdl_wait();
  pdl_trigger();      // after the wait: the kernel behind may read its weights before it waits for this one
  if (a.zero && blockIdx.x == 0)
    for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < a.zeros; i += blockDim.x * blockDim.y) a.zero[i] = 0;
  const long long rows = a.used ? min((long long)max(*a.used, 0), a.rows) : a.rows;
  const int nvec = a.K / 8;
  int turn = 0;
  for (long long r = (long long)blockIdx.x * blockDim.y + threadIdx.y; r < rows; r += (long long)gridDim.x * blockDim.y) {
    const uint4* x = reinterpret_cast<const uint4*>(a.x + r * a.ldx);
    uint4 v[NV ? NV : 1];
    __nv_bfloat162 both = __float2bfloat162_rn(0.0f);
    if (NV) {
      #pragma unroll
      for (int i = 0; i < NV; i++) {
        const int at = i * (int)blockDim.x + (int)threadIdx.x;
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (at < nvec) v[i] = __ldg(x + at);
      }
      #pragma unroll
      for (int i = 0; i < NV; i++) both = vec_max(v[i], both);
    } else {
      for (int at = threadIdx.x; at < nvec; at += blockDim.x) both = vec_max(__ldg(x + at), both);
    }
    float m = fmaxf(no_nan(__low2float(both)), no_nan(__high2float(both)));       // (a NaN counts as an infinity: both make the row NaN)
    #pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (blockDim.x > 32) {
      const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
      if (lane == 0) red[turn][threadIdx.x >> 5] = m;
      __syncthreads();
      m = lane < warps ? red[turn][lane] : 0.0f;
      turn ^= 1;
      #pragma unroll
      for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      m = __shfl_sync(0xffffffffu, m, 0);
    }
    const RowScale row(m);
    if (threadIdx.x == 0) a.scale[r] = row.scale;
    uint2* q = reinterpret_cast<uint2*>(a.q + r * a.K);
    if (row.zero) {
      for (int at = threadIdx.x; at < nvec; at += blockDim.x) q[at] = make_uint2(0u, 0u);
    } else if (NV) {
      #pragma unroll
      for (int i = 0; i < NV; i++) {
        const int at = i * (int)blockDim.x + (int)threadIdx.x;
        if (at < nvec) q[at] = quantize_vec(v[i], row);
      }
    } else {
      for (int at = threadIdx.x; at < nvec; at += blockDim.x) q[at] = quantize_vec(__ldg(x + at), row);
    }
  }
}

}  // namespace

cudaError_t launch_quantize_rows_int8(const void* x, long long rows, const int* used, int K, long long ldx, void* q, float* scale,
                                      int* zero, int zeros, cudaStream_t st) {
  if (rows < 1 || K < 8 || K % 8 || ldx % 8) return cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(x) & 15) || (reinterpret_cast<uintptr_t>(q) & 7)) return cudaErrorMisalignedAddress;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  const QuantArgs a{static_cast<const __nv_bfloat16*>(x), rows, ldx, used, K, static_cast<int8_t*>(q), scale, zero, zeros};
  const int nvec = K / 8;
  // Few rows: as many threads per row as it has vectors, for latency.  More rows than SMs: four vectors per thread, so that an SM
  // has some eight rows on the way (with 512 threads per row of 4096 it had three: 16384 rows took 95 us, now 48).
  const int want_nv = rows > sms ? 4 : 1, lanes = (nvec + want_nv - 1) / want_nv;
  const int threads = lanes <= 32 ? 32 : lanes <= 512 ? (lanes + 31) / 32 * 32 : 512, per_cta = threads == 32 ? 4 : 1;
  const int nv = (nvec + threads - 1) / threads;
  auto launch = [&](auto* two, auto* three) {
    const bool large = threads > 256;
    const long long want = (rows + per_cta - 1) / per_cta, most = (long long)sms * ((large ? 1536 : 1024) / (threads * per_cta));
    return launch_dependent(large ? three : two, dim3((unsigned)(want < most ? want : most)), dim3(threads, per_cta), 0, st, a);
  };
  if (nv <= 1) return launch(quantize_rows_int8_kernel<1, 2>, quantize_rows_int8_kernel<1, 3>);
  if (nv <= 2) return launch(quantize_rows_int8_kernel<2, 2>, quantize_rows_int8_kernel<2, 3>);
  if (nv <= 4) return launch(quantize_rows_int8_kernel<4, 2>, quantize_rows_int8_kernel<4, 3>);
  return launch(quantize_rows_int8_kernel<0, 2>, quantize_rows_int8_kernel<0, 3>);
}

}  // namespace rbv

extern "C" int rbv_quantize_rows_int8(const void* x_bf16, long long rows, const int* used, int K, long long ldx, void* out_int8,
                                      float* scale, void* cuda_stream) {
  return (int)rbv::launch_quantize_rows_int8(x_bf16, rows, used, K, ldx, out_int8, scale, nullptr, 0, static_cast<cudaStream_t>(cuda_stream));
}
