// Grouped GEMM with 8-bit integer operands, one scale per row of A (token) and one per row of B (output channel):
//
//   C[rows of group g] = epilogue( s_row * c_channel * ( A[rows of group g] (M_g x K) * B_g^T (N x K) ) )
//
// The sums are 32-bit integers in tensor memory, exact up to K = 131072; they are scaled once, in 32-bit floating point, and
// rounded once, to bf16.  No counterpart exists in the reference (it has no compute kernels).
//
// Same plan as the bf16 kernel (grouped_gemm_pair_sm100.cu): clusters of two CTAs on neighbouring SMs, tcgen05 cta_group::2
// with 256 weight rows as M and up to 256 tokens as N, K blocks of 128 bytes in a TMA-fed ring (no multicast), two accumulators
// in TMEM so that the epilogue of one tile overlaps the multiplications of the next.  Differences:
//   * tcgen05.mma.kind::i8 takes 32 bytes of K per instruction and as long as kind::f16 takes for them, so a tile takes half
//     the time and eight warps share the epilogue (a lane holds one channel; warps 2-5 take the even, 6-9 the odd blocks of 32
//     tokens).
//   * Any N and K that are multiples of 8 and 16: a tile that reaches beyond a group's channels reads the next group's (or
//     zeros behind the last) and leaves them out when it stores; K behind the end reads as zero.
//   * Tiles of at most 128 or 64 tokens where those still run all at once.
// All waits are bounded; on expiry both CTAs are told, record an error, release their TMEM and return.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kernels/pdl.cuh"
#include "kernels/sm100_ptx.cuh"
#include "kernels/tok_epilogue.cuh"
#include "rbv/moe.h"

namespace rbv {

using namespace sm100;

namespace {

constexpr int IM = 256;            // weight rows (output channels) per pair tile
constexpr int IH = 128;            // weight rows per CTA
constexpr int IT = 256;            // most tokens per tile
constexpr int IU = 32;             // tokens per unit: a tile's token count is a multiple of this
constexpr int IK = 128;            // bytes of K per stage, one 128-byte swizzle atom
constexpr int IW_BYTES = IH * IK;            // 16 KB of weights
constexpr int IT_BYTES = IT / 2 * IK;        // up to 16 KB of tokens
// Pipeline as in the bf16 kernel: 6 stages with room for a full tile's tokens, 10 with room for 64 where no group has more.
constexpr int ISTAGES = 6, ISTAGE_BYTES = IW_BYTES + IT_BYTES;
constexpr int ISMALL = 64, ISTAGES_SMALL = 10, ISTAGE_BYTES_SMALL = IW_BYTES + ISMALL / 2 * IK;
constexpr int I_THREADS = 320;
constexpr int I_TMEM_COLS = 512;
constexpr size_t I_SMEM = (size_t)ISTAGES_SMALL * ISTAGE_BYTES_SMALL + 1024 /*alignment slack*/;
static_assert(ISTAGES * ISTAGE_BYTES <= ISTAGES_SMALL * ISTAGE_BYTES_SMALL, "shared memory");

// Token boxes of 16, 32, 64 and 128 rows: a CTA's half of a tile (a multiple of 16 rows) is put together from them.
struct I8Maps { CUtensorMap w, tok[4]; };

struct I8Params {
  const int* group_start;            // null: one group of all a_rows rows
  const int* group_rows;
  int G, N, K, ldc, tile_tokens;     // tile_tokens: most tokens per tile
  long long a_rows;
  const float* row_scale;            // [a_rows]
  const float* col_scale;            // [G, N]
  __nv_bfloat16* C;
  int* error;
  int swiglu;
};

struct I8Tile { int tok0, ntok, nt, n0, g; bool valid; };   // first token row, live tokens, columns, first channel, group

// Walks the tile schedule; `at(t)` wants non-decreasing t.
struct I8Walk {
  int g = 0, before = 0;   // tiles of the groups in front of g
  __device__ __forceinline__ I8Tile at(const I8Params& p, int t, const int* s_rows, const int* s_start) {
    I8Tile r; r.valid = false; r.tok0 = r.ntok = r.nt = r.n0 = r.g = 0;
    const int wide = p.tile_tokens / IU;
    for (; g < p.G; g++) {
      const int units = (s_rows[g] + IU - 1) / IU, ntm = (units + wide - 1) / wide;
      const int cnt = ntm * ((p.N + IM - 1) / IM);
      if (t - before < cnt) {
        const int n = (t - before) / ntm, m = (t - before) - n * ntm;
        const int base = units / ntm, extra = units - base * ntm;     // the first `extra` tiles are one unit larger
        const int u0 = m * base + min(m, extra), nu = base + (m < extra ? 1 : 0);
        r.tok0 = s_start[g] + u0 * IU; r.nt = nu * IU; r.ntok = min(s_rows[g] - u0 * IU, r.nt);
        r.n0 = n * IM; r.g = g;
        r.valid = true;
        return r;
      }
      before += cnt;
    }
    return r;
  }
};

// The waits and loads of sm100_ptx.cuh with shared-memory addresses as numbers.
__device__ __forceinline__ bool wait_at(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  for (uint32_t i = 0; i < (1u << 24); i++) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred P;\n\tmbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2;\n\tselp.b32 %0, 1, 0, P;\n\t}"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
    if ((i & 1023u) == 1023u && *abort_flag) return false;
  }
  return false;
}
__device__ __forceinline__ void expect_at(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void load_at(uint32_t dst, const CUtensorMap* m, int x, int y, uint32_t bar_cluster_addr) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(m), "r"(bar_cluster_addr), "r"(x), "r"(y) : "memory");
}

}  // namespace

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I_THREADS, 1)
grouped_gemm_int8_kernel(const __grid_constant__ I8Maps maps, const __grid_constant__ I8Params p) {
  extern __shared__ uint8_t dyn_smem[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full_bar[ISTAGES_SMALL];    // used in the rank-0 CTA: bytes of both CTAs' loads
  __shared__ __align__(8) uint64_t empty_bar[ISTAGES_SMALL];   // in each CTA: its stage has been read by the MMAs
  __shared__ __align__(8) uint64_t tfull_bar[2];         // in each CTA: accumulator b is complete
  __shared__ __align__(8) uint64_t tempty_bar[2];        // used in the rank-0 CTA: both CTAs have drained accumulator b
  __shared__ uint32_t tmem_base_s;
  __shared__ int s_rows[kMoeMaxGroups], s_start[kMoeMaxGroups];
  __shared__ int s_abort, s_most;                        // s_most: rows of the largest group

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

  if (tid == 0) {
    for (int s = 0; s < ISTAGES_SMALL; s++) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int b = 0; b < 2; b++) { mbar_init(&tfull_bar[b], 1); mbar_init(&tempty_bar[b], 16); }
    s_abort = 0;
    s_most = 0;
    mbar_fence_init();
  }
  if (warp == 1) { tmem_alloc_pair(&tmem_base_s, I_TMEM_COLS); tmem_relinquish_pair(); }
  __syncthreads();
  pdl_trigger();
  pdl_wait();
  for (int i = tid; i < p.G; i += blockDim.x) {
    s_start[i] = p.group_start ? p.group_start[i] : 0;
    s_rows[i] = p.group_rows ? rows_inside(s_start[i] < 0 ? 0 : p.group_rows[i], s_start[i], p.a_rows, p.error) : (int)p.a_rows;
    if (s_start[i] < 0 && p.error && blockIdx.x == 0) atomicCAS(p.error, 0, 6);
    atomicMax(&s_most, s_rows[i]);
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();   // barriers of both CTAs are initialised before anything is signalled across
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_base_s;
  const int num_kb = (p.K + IK - 1) / IK;
  const int stages = s_most <= ISMALL ? ISTAGES_SMALL : ISTAGES;
  const int stage_bytes = s_most <= ISMALL ? ISTAGE_BYTES_SMALL : ISTAGE_BYTES;
  volatile int* abort_flag = &s_abort;
  const uint32_t peer_abort = mapa_u32(smem_u32(&s_abort), rank ^ 1u);

  if (warp == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    // One thread feeds the ring, and one issues the MMAs: what they execute per K block (16 to 32 KB) is kept short, with
    // addresses as numbers that are counted up.
    if (elect_one()) {
      tma_prefetch_desc(&maps.w);
      const uint32_t full0 = mapa_u32(smem_u32(&full_bar[0]), 0), my_full = smem_u32(&full_bar[0]), empty0 = smem_u32(&empty_bar[0]);
      const uint32_t base = smem_u32(tiles);
      int stage = 0; uint32_t phase = 1;
      bool ok = true;
      I8Walk walk;
      for (int t = pair; ok; t += npairs) {
        const I8Tile tl = walk.at(p, t, s_rows, s_start);
        if (!tl.valid) break;
        const int half = tl.nt / 2;
        const uint32_t bytes = 2u * (uint32_t)(IW_BYTES + half * IK);
        const int w_row = tl.g * p.N + tl.n0 + (int)rank * IH;
        const int t_row = tl.tok0 + (int)rank * half;
        #pragma unroll 1
        for (int x = 0; x < p.K; x += IK) {
          if (!wait_at(empty0 + 8u * stage, phase, abort_flag)) { ok = false; break; }
          const uint32_t sw = base + (uint32_t)(stage * stage_bytes), bar = full0 + 8u * stage;
          if (leader) expect_at(my_full + 8u * stage, bytes);
          load_at(sw, &maps.w, x, w_row, bar);
          uint32_t to = sw + IW_BYTES;
          int row = t_row;
          #pragma unroll
          for (int b = 3; b >= 0; b--)
            if (half & (16 << b)) {
              load_at(to, &maps.tok[b], x, row, bar);
              to += (16u << b) * IK;
              row += 16 << b;
            }
          if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) { s_abort = 1; st_cluster_u32(peer_abort, 1); if (p.error) atomicExch(p.error, 1); }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (rank-0 CTA only) ----------------
    if (leader && elect_one()) {
      const uint32_t full0 = smem_u32(&full_bar[0]);
      const uint64_t desc0 = umma_desc_sw128(tiles);
      int stage = 0; uint32_t phase = 0;
      bool ok = true;
      int i = 0;
      I8Walk walk;
      for (int t = pair; ok; t += npairs, i++) {
        const I8Tile tl = walk.at(p, t, s_rows, s_start);
        if (!tl.valid) break;
        const uint32_t idesc = umma_idesc_i8(IM, tl.nt);
        const int b = i & 1;
        if (!mbar_wait(&tempty_bar[b], (((uint32_t)i >> 1) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + (uint32_t)b * IT;
        #pragma unroll 1
        for (int kb = 0; kb < num_kb; kb++) {
          if (!wait_at(full0 + 8u * stage, phase, abort_flag)) { ok = false; break; }
          tc_fence_after_sync();
          const uint64_t wdesc = desc0 + (uint64_t)((uint32_t)(stage * stage_bytes) >> 4), tdesc = wdesc + (IW_BYTES >> 4);
          #pragma unroll
          for (int kk = 0; kk < IK / 32; kk++)
            umma_i8_pair(d_tmem, wdesc + 2u * kk, tdesc + 2u * kk, idesc, (uint32_t)((kb | kk) != 0));
          umma_commit_pair(&empty_bar[stage]);   // frees this stage in both CTAs
          if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
        if (ok) umma_commit_pair(&tfull_bar[b]);   // accumulator complete, both CTAs
      }
      if (!ok) { s_abort = 1; st_cluster_u32(peer_abort, 1); if (p.error) atomicExch(p.error, 2); }
    }
  } else {
    // ---------------- epilogue (both CTAs): warps 2..9, TMEM lane quarter = warp % 4 ----------------
    const int q = warp & 3, first = warp < 6 ? 0 : IU;
    bool ok = true;
    int i = 0;
    I8Walk walk;
    for (int t = pair; ok; t += npairs, i++) {
      const I8Tile tl = walk.at(p, t, s_rows, s_start);
      if (!tl.valid) break;
      const int b = i & 1;
      const int nw = tl.n0 + (int)rank * IH + q * 32;   // first of this warp's 32 channels
      const float cs = nw + lane < p.N ? __ldg(p.col_scale + (size_t)tl.g * p.N + nw + lane) : 0.0f;
      float rs[IT / (2 * IU)];                          // scales of this warp's tokens, on their way while the tile is multiplied
      #pragma unroll
      for (int j = 0; j < IT / (2 * IU); j++) {
        const int c = first + j * 2 * IU + lane;
        rs[j] = c < tl.ntok ? __ldg(p.row_scale + tl.tok0 + c) : 0.0f;
      }
      if (!mbar_wait(&tfull_bar[b], ((uint32_t)i >> 1) & 1u, abort_flag)) { ok = false; break; }
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)b * IT;
      const int live_cols = p.N - nw;                   // channels of this warp that exist (a multiple of 8)
      #pragma unroll 1
      for (int c = first; c < tl.nt; c += 2 * IU) {
        uint32_t r[32];
        tmem_ld32(taddr + c, r);
        tmem_ld_wait();
        #pragma unroll
        for (int k = 0; k < 32; k++)
          r[k] = __float_as_uint((float)(int)r[k] * cs * __shfl_sync(0xffffffffu, rs[0], k));
        #pragma unroll
        for (int j = 0; j + 1 < IT / (2 * IU); j++) rs[j] = rs[j + 1];
        __nv_bfloat16* rows = p.C + (size_t)(tl.tok0 + c) * p.ldc;
        // (all lanes take part in the exchanges; tokens or channels that do not exist are not stored)
        if (p.swiglu) tokepi::store_swiglu(r, rows, p.ldc, nw / 2, (lane >> 2) * 4 < live_cols ? tl.ntok - c : 0, lane);
        else tokepi::store_plain(r, [&](int tok) { return rows + (size_t)tok * p.ldc; }, nw, lane < live_cols ? tl.ntok - c : 0, lane);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_u32(smem_u32(&tempty_bar[b]), 0));   // 8 warps x 2 CTAs
    }
    if (!ok && lane == 0) { s_abort = 1; st_cluster_u32(peer_abort, 1); if (p.error) atomicExch(p.error, 3); }
  }

  // ---------------- teardown: nobody leaves while the other CTA may still signal it ----------------
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, I_TMEM_COLS);
  }
}

// ---------------- host side ----------------
namespace {

// [rows, K] bytes row-major, box = box_rows x 128 bytes, 128-byte swizzle
bool i8_make_map(CUtensorMap* m, const void* base, unsigned long long rows, unsigned long long K, unsigned box_rows) {
  typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<Encode>(p) : nullptr;
  }();
  if (!encode) return false;
  const cuuint64_t dims[2] = {K, rows}, strides[1] = {K};
  const cuuint32_t box[2] = {(cuuint32_t)IK, box_rows}, ones[2] = {1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace rbv

extern "C" int rbv_grouped_gemm_int8(const void* A, const float* a_scale, long long a_rows, const void* B, const float* b_scale,
                                     void* C, const int* group_start, const int* group_rows, int G, int N, int K, int ldc,
                                     int epilogue, int* error_flag, int max_ctas, void* cuda_stream) {
  using namespace rbv;
  if (G < 1 || G > kMoeMaxGroups || N < 8 || N % 8 || K < 16 || K % 16 || K > RBV_INT8_MAX_DEPTH || a_rows < 1 || a_rows > RBV_INT8_MAX_ROWS ||
      ldc % 2 || (long long)G * N > RBV_INT8_MAX_CHANNELS || epilogue < 0 || epilogue > 1)
    return (int)cudaErrorInvalidValue;
  if ((!group_start) != (!group_rows) || (!group_start && G != 1)) return (int)cudaErrorInvalidValue;
  if (((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B)) & 15) || (reinterpret_cast<uintptr_t>(C) & 3))
    return (int)cudaErrorMisalignedAddress;
  cudaError_t e = cudaFuncSetAttribute(grouped_gemm_int8_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)I_SMEM);
  if (e != cudaSuccess) return (int)e;
  I8Maps maps;
  if (!i8_make_map(&maps.w, B, (unsigned long long)G * N, (unsigned long long)K, IH)) return (int)cudaErrorUnknown;
  for (int i = 0; i < 4; i++)
    if (!i8_make_map(&maps.tok[i], A, (unsigned long long)a_rows, (unsigned long long)K, 16u << i)) return (int)cudaErrorUnknown;
  int grid = max_ctas;
  if (grid <= 0) {
    int dev = 0;
    if ((e = cudaGetDevice(&dev)) != cudaSuccess || (e = cudaDeviceGetAttribute(&grid, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return (int)e;
  }
  grid &= ~1;   // whole pairs
  if (grid < 2) return (int)cudaErrorInvalidValue;
  I8Params p;
  p.group_start = group_start; p.group_rows = group_rows; p.G = G; p.N = N; p.K = K; p.ldc = ldc;
  p.a_rows = a_rows; p.row_scale = a_scale; p.col_scale = b_scale; p.C = static_cast<__nv_bfloat16*>(C);
  p.error = error_flag; p.swiglu = epilogue;
  // Narrower tiles only while all of them, with the rows shared out evenly among the groups, still run at once: a tile of 32 to 160
  // tokens takes as long as its weights, and a second round as long as the first (72 tiles of 160 tokens: 15.8 us, 144 of 96 and
  // 64: 22.8).
  const long long per_group = (a_rows + G - 1) / G, channels = (N + IM - 1) / IM;
  p.tile_tokens = IT;
  while (p.tile_tokens > 64 && G * channels * ((per_group + p.tile_tokens / 2 - 1) / (p.tile_tokens / 2)) <= grid / 2) p.tile_tokens /= 2;
  return (int)launch_dependent(grouped_gemm_int8_kernel, grid, I_THREADS, I_SMEM, static_cast<cudaStream_t>(cuda_stream), maps, p);
}
