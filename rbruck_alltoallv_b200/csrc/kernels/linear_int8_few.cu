// 8-bit integer linear for a few rows (1 to 64):  out[r][n] = s_r c_n sum_k q[r][k] W[n][k], sums in 32-bit integers, exact.
//
// Two kernels: the rows are quantised (int8_quant.cu), then the weights stream past them (few_rows.cuh).  Bound by HBM, which
// reads the weights once.  The second kernel starts while the first one runs and has its first weights on the way by then;
// only the quantised rows have to be waited for.  Work is column tiles x chunks of K, cut evenly among the SMs; integer sums of
// a tile that several CTAs share are exact in any order.
//
// Up to 4096 elements of A in at most 8 rows, and tiles that are not split: one kernel, in which every CTA quantises the rows for
// itself (they come out of L2) while its first weights are on their way.  4096 x 4096, one row: 7.9 us with two kernels, 6.0 with
// one.  4096 is what two vectors per thread hold, not where the times cross.  Both forms (one kernel with four vectors per thread
// up to 8192 elements, with eight up to 16384), 4096 channels, graph replays: one row of 5120 9.0 us with two kernels, 6.7 with one
// of four vectors, 7.6 of eight; of 8192 11.1, 8.8, 9.9; of 14336 14.9, -, 15.3; four rows of 2048 5.9, 6.6, 7.3; of 4096 7.9, -,
// 11.1; and one row of 4096 itself 5.9, 5.9, 6.7.  Results that are written over the rows take two kernels.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "kernels/few_rows.cuh"
#include "kernels/int8_quant.cuh"
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
  const __nv_bfloat16* x;                 // rows that are quantised here, ldx elements apart
  long long ldx;
  uint32_t row_bytes;                     // room for them, a multiple of 1024
};

constexpr int kOwnElems = 4096, kOwnRows = 8;      // of A at most, where every CTA quantises it for itself

// The rows in shared memory as Rows<1>::load reads them: chunk by chunk, column by column, M rows of 128 bytes with the 16-byte
// units swizzled.  All consumer warps; scales[r] of row r, `largest` zero before.
__device__ __forceinline__ void quantize_own(const LinearArgs& a, uint8_t* rows, unsigned* largest, float* scales) {
  using namespace quant;
  constexpr int kVecs = kOwnElems / 8 / (kWarps * 32);
  const int tid = threadIdx.x, nvec = a.K / 8, total = a.M * nvec;
  uint4 v[kVecs];
  int row[kVecs];
  #pragma unroll
  for (int i = 0; i < kVecs; i++) {
    const int f = i * kWarps * 32 + tid;
    row[i] = f / nvec;
    v[i] = make_uint4(0u, 0u, 0u, 0u);
    if (f < total) v[i] = __ldg(reinterpret_cast<const uint4*>(a.x + row[i] * a.ldx) + f - row[i] * nvec);
  }
  #pragma unroll
  for (int i = 0; i < kVecs; i++) {
    if (i * kWarps * 32 >= total) break;
    const __nv_bfloat162 both = vec_max(v[i], __float2bfloat162_rn(0.0f));
    const unsigned m = __float_as_uint(fmaxf(no_nan(__low2float(both)), no_nan(__high2float(both))));
    const int first = __shfl_sync(0xffffffffu, row[i], 0);
    if (__all_sync(0xffffffffu, row[i] == first)) {        // (magnitudes are in order as unsigned numbers)
      const unsigned most = __reduce_max_sync(0xffffffffu, m);
      if ((tid & 31) == 0 && first < a.M) atomicMax(largest + first, most);
    } else if (row[i] < a.M) {
      atomicMax(largest + row[i], m);
    }
  }
  consumers_sync();
  const int chunk_bytes = a.M * kChunk;
  auto place = [&](int r, int k) {
    const int chunk = k / kChunk, col = k / 128 % kCols, unit = k / 16 % 8;
    return reinterpret_cast<uint2*>(rows + chunk * chunk_bytes + (col * a.M + r) * 128 + ((unit ^ (r & 7)) << 4) + k % 16);
  };
  #pragma unroll
  for (int i = 0; i < kVecs; i++) {
    const int f = i * kWarps * 32 + tid;
    if (f >= total) break;
    const RowScale scale(__uint_as_float(largest[row[i]]));
    const int at = f - row[i] * nvec;
    if (at == 0) scales[row[i]] = scale.scale;
    *place(row[i], at * 8) = scale.zero ? make_uint2(0u, 0u) : quantize_vec(v[i], scale);
  }
  const int behind = (kChunk - a.K % kChunk) % kChunk / 8;       // from the end of a row to the end of its last chunk
  for (int f = tid; f < a.M * behind; f += kWarps * 32) *place(f / behind, a.K + f % behind * 8) = make_uint2(0u, 0u);
  consumers_sync();
}

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

// NT: tiles of 8 rows of A.  OWN: the rows are quantised here.
template <int NT, bool OWN>
__global__ void __launch_bounds__(kThreads, 1) linear_int8_few_kernel(const __grid_constant__ WeightMaps maps, const __grid_constant__ WeightMaps q_maps,
                                                                      const __grid_constant__ LinearArgs a) {
  extern __shared__ uint8_t dyn[];
  __shared__ Ring ring;
  __shared__ int flag[2];
  __shared__ unsigned largest[kOwnRows];
  __shared__ float scales[kOwnRows];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~uintptr_t(1023));
  Red red{reinterpret_cast<uint4*>(base), true};
  if (tid == 0) ring_init(ring, a.stages, OWN ? 1 : 2);
  if (OWN && tid < kOwnRows) largest[tid] = 0u;
  if (warp == kWarps) prefetch_maps(maps);
  if (!OWN && warp == kWarps + 1) prefetch_maps(q_maps);
  pdl_trigger();
  __syncthreads();
  LinearWalk walk(a);
  LinearPiece p;
  uint8_t* own_rows = base + 2 * kRedBytes;
  Cursor cur(ring, sm100::smem_u32(own_rows + (OWN ? a.row_bytes : 0u)), a.stages, slot_bytes(a.tile, OWN ? 0 : a.box));
  if (warp >= kWarps) {
    if (lane >= 4 || (OWN && warp > kWarps)) return;
    if (warp == kWarps) {
      if (OWN) pdl_wait();                // (the kernel before may be one that makes the weights; with two it is the quantiser)
      while (walk.next(p) && feed<int8_t>(maps, cur, 0, p.tile * a.tile, min(a.tile, a.N - p.tile * a.tile), p.c0, p.c1)) {}
    } else {
      pdl_wait();
      asm volatile("fence.proxy.async;" ::: "memory");
      while (walk.next(p) && feed<int8_t>(q_maps, cur, (uint32_t)a.tile * kChunk, 0, a.box, p.c0, p.c1)) {}
    }
    return;
  }
  pdl_wait();
  if (OWN) quantize_own(a, own_rows, largest, scales);
  int rows_at[NT];
  const int part = warp >> 2, col = warp & 3;
  #pragma unroll
  for (int i = 0; i < NT; i++) rows_at[i] = 8 * i + (lane >> 2) < a.M ? 8 * i + (lane >> 2) : -1;
  auto result = [&](int r, int n, int v0, int v1) {
    const float s = OWN ? scales[r] : __ldcg(a.row_scale + r);
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
        if (OWN) rows.load(rows_at, sm100::smem_u32(own_rows) + (uint32_t)(c * a.M * kChunk), a.M, col, lane);
        else rows.load(rows_at, cur.slot + (uint32_t)a.tile * kChunk, a.box, col, lane);
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

struct LinearPlan { int sms, tile, whole, own; size_t q_bytes, scale_bytes, partial_bytes, counter_bytes; };

bool linear_plan(int M, int N, int K, LinearPlan* p) {
  if (M < 1 || M > kMaxRows || N < 8 || K < 16 || N % 8 || K % 16 || K > RBV_INT8_MAX_DEPTH || N > RBV_INT8_MAX_CHANNELS) return false;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&p->sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return false;
  if (!split_plan(N, K, 1, p->sms, M, box_rows(M) / 8, false, &p->tile, &p->whole)) return false;
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  p->own = p->whole && M <= kOwnRows && (long long)M * K <= kOwnElems;
  p->q_bytes = up((size_t)M * K);
  p->scale_bytes = up((size_t)M * 4);
  if (p->own) {                           // one kernel, or two (results over the rows); tiles are whole
    p->partial_bytes = p->counter_bytes = 0;
    return true;
  }
  p->partial_bytes = up((size_t)2 * p->sms * M * p->tile * 4);
  p->counter_bytes = up((size_t)((N + p->tile - 1) / p->tile) * 4);
  return true;
}

template <int NT, bool OWN = false>
cudaError_t linear_launch(const LinearArgs& args, const int8_t* q, const void* w, const LinearPlan& p, cudaStream_t st) {
  LinearArgs a = args;
  WeightMaps maps, q_maps;
  if (!weight_maps(&maps, w, (unsigned long long)a.N, (unsigned long long)a.K, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.tile | a.N % p.tile) ||
      (!OWN && !weight_maps(&q_maps, q, (unsigned long long)a.M, (unsigned long long)a.K, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, box_rows(a.M))))
    return cudaErrorUnknown;
  a.tile = p.tile;
  a.whole = p.whole;
  a.box = OWN ? 0 : box_rows(a.M);
  a.row_bytes = OWN ? ((uint32_t)a.M * (uint32_t)((a.K + kChunk - 1) / kChunk * kChunk) + 1023) / 1024 * 1024 : 0u;
  constexpr size_t kFixed = sizeof(Ring) + 128;
  a.stages = ring_stages(a.tile, a.box, kFixed, 2 * kRedBytes + a.row_bytes);
  const size_t smem = ring_smem(a.tile, a.box, a.stages) + 2 * kRedBytes + a.row_bytes;
  const cudaError_t e = allow_smem_once<linear_int8_few_kernel<NT, OWN>>(kFixed);
  return e != cudaSuccess ? e : launch_dependent(linear_int8_few_kernel<NT, OWN>, dim3(p.sms), dim3(kThreads), smem, st, maps, q_maps, a);
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
  // With one kernel a CTA may read the rows when another one has already stored its results: never over the rows themselves.
  const uintptr_t x_at = reinterpret_cast<uintptr_t>(x), out_at = reinterpret_cast<uintptr_t>(out);
  if (x_at < out_at + 2ull * M * N && out_at < x_at + 2ull * ((M - 1) * ldx + K)) p.own = 0;
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
  if (p.own) {
    if (reinterpret_cast<uintptr_t>(x) & 15 || ldx % 8) return (int)cudaErrorMisalignedAddress;
    a.x = static_cast<const __nv_bfloat16*>(x);
    a.ldx = ldx;
    return (int)linear_launch<1, true>(a, nullptr, w, p, st);
  }
  const cudaError_t e = launch_quantize_rows_int8(x, M, nullptr, K, ldx, q, scale, a.counters, (int)(p.counter_bytes / 4), st);
  if (e != cudaSuccess) return (int)e;
  if (M <= 8) return (int)linear_launch<1>(a, q, w, p, st);
  if (M <= 16) return (int)linear_launch<2>(a, q, w, p, st);
  if (M <= 32) return (int)linear_launch<4>(a, q, w, p, st);
  return (int)linear_launch<8>(a, q, w, p, st);
}
