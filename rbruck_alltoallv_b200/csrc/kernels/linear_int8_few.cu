// 8-bit integer linear for a few rows (1 to 64):  out[r][n] = s_r c_n sum_k q[r][k] W[n][k], sums in 32-bit integers, exact.
//
// Two kernels: the rows are quantised (int8_quant.cu), then the weights stream past them (few_rows.cuh).  Bound by HBM, which
// reads the weights once.  The second kernel starts while the first one runs and has its first weights on the way by then;
// only the quantised rows have to be waited for.  Work is column tiles x chunks of K, cut evenly among the SMs; integer sums of
// a tile that several CTAs share are exact in any order.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "kernels/few_rows.cuh"
#include "kernels/pdl.cuh"
#include "rbv/moe.h"

namespace rbv {

cudaError_t launch_quantize_rows_int8(const void* x, long long rows, const int* used, int K, long long ldx, void* q, float* scale,
                                      int* zero, int zeros, cudaStream_t st);

namespace {

using namespace few;

struct LinearArgs {
  const float *row_scale, *col_scale;
  int M, N, K;
  int* partial;                           // [2 * CTAs][M][tile]
  int* counters;                          // one per column tile
  __nv_bfloat16* out;
  int* error;
  int tile, box, stages, whole;
};

struct LinearPiece { int tile, c0, c1; };

struct LinearWalk {
  Split split;
  unsigned at, end;
  int chunks, tile, c;
  __device__ __forceinline__ explicit LinearWalk(const LinearArgs& a) {
    chunks = (a.K + kChunk - 1) / kChunk;
    const unsigned tiles = (a.N + a.tile - 1) / a.tile;
    split.grain = a.whole ? chunks : 1;
    split.total = a.whole ? tiles : tiles * chunks;
    split.parts = min(gridDim.x, split.total);
    at = end = 0;
    if (blockIdx.x < split.parts) { at = split.begin(blockIdx.x); end = split.begin(blockIdx.x + 1); }
    tile = at / chunks;
    c = at - tile * chunks;
  }
  __device__ __forceinline__ bool next(LinearPiece& p) {
    if (at >= end) return false;
    p.tile = tile++;
    p.c0 = c;
    p.c1 = (int)min((unsigned)chunks, c + (end - at));
    at += p.c1 - p.c0;
    c = 0;
    return true;
  }
};

// NT: tiles of 8 rows of A.
template <int NT>
__global__ void __launch_bounds__(kThreads, 1) linear_int8_few_kernel(const __grid_constant__ WeightMaps maps, const __grid_constant__ WeightMaps q_maps,
                                                                      const __grid_constant__ LinearArgs a) {
  extern __shared__ uint8_t dyn[];
  __shared__ Ring ring;
  __shared__ int flag[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~uintptr_t(1023));
  uint4* red = reinterpret_cast<uint4*>(base);
  if (tid == 0) ring_init(ring, a.stages, 2);
  if (warp >= kWarps) prefetch_maps(warp == kWarps ? maps : q_maps);
  pdl_trigger();
  __syncthreads();
  LinearWalk walk(a);
  LinearPiece p;
  Cursor cur(ring, sm100::smem_u32(base + kRedBytes), a.stages, slot_bytes(a.tile, a.box));
  if (warp >= kWarps) {
    if (lane >= 4) return;
    if (warp == kWarps) {
      while (walk.next(p) && feed<int8_t>(maps, cur, 0, p.tile * a.tile, min(a.tile, a.N - p.tile * a.tile), p.c0, p.c1)) {}
    } else {
      pdl_wait();
      asm volatile("fence.proxy.async;" ::: "memory");
      while (walk.next(p) && feed<int8_t>(q_maps, cur, (uint32_t)a.tile * kChunk, 0, a.box, p.c0, p.c1)) {}
    }
    return;
  }
  pdl_wait();
  int rows_at[NT];
  const int part = warp >> 2, col = warp & 3;
  #pragma unroll
  for (int i = 0; i < NT; i++) rows_at[i] = 8 * i + (lane >> 2) < a.M ? 8 * i + (lane >> 2) : -1;
  auto result = [&](int r, int n, int v0, int v1) {
    const float s = __ldcg(a.row_scale + r);
    const float2 c = *reinterpret_cast<const float2*>(a.col_scale + n);
    *reinterpret_cast<__nv_bfloat162*>(a.out + (long long)r * a.N + n) = __floats2bfloat162_rn((float)v0 * s * c.x, (float)v1 * s * c.y);
  };
  int cut[2] = {-1, -1};                  // tiles shared with the CTA before and the CTA behind
  while (walk.next(p)) {
    const int col0 = p.tile * a.tile, nr = min(a.tile, a.N - col0);
    const Share share(nr, part);
    const Offsets off(nr, share, col);
    int acc[kGroups][NT][4];
    clear(acc);
    auto run = [&](auto tag) {
      constexpr int G = decltype(tag)::value;
      #pragma unroll 1
      for (int c = p.c0; c < p.c1; c++) {
        cur.wait_full();
        __syncwarp();
        Rows<NT> rows;
        rows.load(rows_at, cur.slot + (uint32_t)a.tile * kChunk, a.box, col, lane);
        multiply<G>(acc, cur.slot, off, rows, lane);
        __syncwarp();
        if (lane == 0) cur.release();
        cur.next();
      }
    };
    if (share.count <= 1) run(std::integral_constant<int, 1>());
    else run(std::integral_constant<int, kGroups>());
    const bool starts = p.c0 == 0, whole = starts && p.c1 == walk.chunks;
    int* sums = a.partial + (2ll * blockIdx.x + (starts ? 1 : 0)) * a.M * a.tile;
    add_columns<NT>(acc, red, share, part, col, lane, [&](int r, int n, int v0, int v1) {
      if (r >= a.M || n >= nr) return;
      if (whole) result(r, col0 + n, v0, v1);
      else *reinterpret_cast<int2*>(sums + r * a.tile + n) = make_int2(v0, v1);
    });
    if (!whole) cut[starts ? 1 : 0] = p.tile;
  }
  if (cut[0] >= 0 || cut[1] >= 0) {
    auto owners = [&](int tile, int& c0, int& c1) {
      const unsigned first = tile * walk.chunks;
      c0 = walk.split.owner(first);
      c1 = walk.split.owner(first + walk.chunks - 1);
    };
    __threadfence();
    consumers_sync();
    if (tid < 2) {
      int last = 0;
      if (cut[tid] >= 0) {
        int c0, c1;
        owners(cut[tid], c0, c1);
        last = atomicAdd(a.counters + cut[tid], 1) == c1 - c0;
      }
      flag[tid] = last;
    }
    consumers_sync();
    for (int i = 0; i < 2; i++) {
      if (!flag[i]) continue;
      __threadfence();
      int c0, c1;
      owners(cut[i], c0, c1);
      const int col0 = cut[i] * a.tile, pairs = min(a.tile, a.N - col0) / 2;
      for (int k = tid; k < a.M * pairs; k += kWarps * 32) {
        const int r = k / pairs, n = (k - r * pairs) * 2;
        // only the first one's range may have begun before the tile
        const int* from = a.partial + 2ll * c0 * a.M * a.tile + r * a.tile + n;
        int2 sum = __ldcg(reinterpret_cast<const int2*>(from + a.M * a.tile));
        #pragma unroll 4
        for (int c = 1; c <= c1 - c0; c++) {
          const int2 v = __ldcg(reinterpret_cast<const int2*>(from + 2ll * c * a.M * a.tile));
          sum.x += v.x;
          sum.y += v.y;
        }
        result(r, col0 + n, sum.x, sum.y);
      }
    }
  }
  if (!cur.ok && a.error) atomicExch(a.error, 1);
}

struct LinearPlan { int sms, tile, whole; size_t q_bytes, scale_bytes, partial_bytes, counter_bytes; };

bool linear_plan(int M, int N, int K, LinearPlan* p) {
  if (M < 1 || M > kMaxRows || N < 8 || K < 16 || N % 8 || K % 16 || K > RBV_INT8_MAX_DEPTH) return false;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&p->sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return false;
  if (!split_plan(N, K, 1, p->sms, M, box_rows(M) / 8, false, &p->tile, &p->whole)) return false;
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  p->q_bytes = up((size_t)M * K);
  p->scale_bytes = up((size_t)M * 4);
  p->partial_bytes = up((size_t)2 * p->sms * M * p->tile * 4);
  p->counter_bytes = up((size_t)((N + p->tile - 1) / p->tile) * 4);
  return true;
}

template <int NT>
cudaError_t linear_launch(const LinearArgs& args, const int8_t* q, const void* w, const LinearPlan& p, cudaStream_t st) {
  LinearArgs a = args;
  WeightMaps maps, q_maps;
  if (!weight_maps(&maps, w, (unsigned long long)a.N, (unsigned long long)a.K, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.tile | a.N % p.tile) ||
      !weight_maps(&q_maps, q, (unsigned long long)a.M, (unsigned long long)a.K, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, box_rows(a.M)))
    return cudaErrorUnknown;
  a.tile = p.tile;
  a.whole = p.whole;
  a.box = box_rows(a.M);
  a.stages = ring_stages(a.tile, a.box, sizeof(Ring) + 64);
  const size_t smem = ring_smem(a.tile, a.box, a.stages);
  const cudaError_t e = allow_smem_once<linear_int8_few_kernel<NT>>(sizeof(Ring) + 64);
  return e != cudaSuccess ? e : launch_dependent(linear_int8_few_kernel<NT>, dim3(p.sms), dim3(kThreads), smem, st, maps, q_maps, a);
}

}  // namespace
}  // namespace rbv

using namespace rbv;

extern "C" long long rbv_linear_int8_few_workspace(int M, int N, int K) {
  LinearPlan p;
  return linear_plan(M, N, K, &p) ? (long long)(p.q_bytes + p.scale_bytes + p.partial_bytes + p.counter_bytes) : -1;
}

extern "C" int rbv_linear_int8_few(const void* x, long long ldx, int M, const void* w, const float* w_scale, int N, int K, void* out,
                                   void* workspace, int* error_flag, void* stream) {
  LinearPlan p;
  if (!linear_plan(M, N, K, &p) || !x || !w || !w_scale || !out || !workspace || (M > 1 && ldx < K)) return (int)cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace) |
       reinterpret_cast<uintptr_t>(w_scale)) & 15)
    return (int)cudaErrorMisalignedAddress;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  int8_t* q = reinterpret_cast<int8_t*>(ws);
  float* scale = reinterpret_cast<float*>(ws + p.q_bytes);
  LinearArgs a{};
  a.row_scale = scale; a.col_scale = w_scale;
  a.M = M; a.N = N; a.K = K;
  a.partial = reinterpret_cast<int*>(ws + p.q_bytes + p.scale_bytes);
  a.counters = reinterpret_cast<int*>(ws + p.q_bytes + p.scale_bytes + p.partial_bytes);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.error = error_flag;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = launch_quantize_rows_int8(x, M, nullptr, K, ldx, q, scale, a.counters, (int)(p.counter_bytes / 4), st);
  if (e != cudaSuccess) return (int)e;
  if (M <= 8) return (int)linear_launch<1>(a, q, w, p, st);
  if (M <= 16) return (int)linear_launch<2>(a, q, w, p, st);
  if (M <= 32) return (int)linear_launch<4>(a, q, w, p, st);
  return (int)linear_launch<8>(a, q, w, p, st);
}
