// A whole top-k routed SwiGLU mixture-of-experts layer for a few tokens (1 to 64) in two kernels, all experts on this GPU.
//
//   choice    the top_k largest logits of a token (ties: lower expert), softmax over the chosen ones; -inf is never chosen
//   up        h[t, j] = p_tj silu(W13g x_t) * (W13u x_t), rounded to bf16            (chosen expert j of token t)
//   down      out[t] = sum_j W2 h[t, j]
//
// Bound by HBM: the weights of every chosen expert are read once, 6 H I bytes each; up to 64 rows the multiplications take
// less time than the bytes.  What a chain of router, dispatch, two grouped GEMMs and combine costs on top is launches,
// tiles of 256 weight rows that do not divide evenly among the SMs, and rows that go through memory between the kernels.
// Here every CTA makes the choice itself from the logits (T x E numbers out of L2), nobody waits for a layout, and the
// weights are split among the SMs at multiples of 8 rows (up) or 256 columns of K (down; few_rows.cuh).  The second kernel
// starts as SMs become free and has its first weights on the way before the first one has finished: only h has to be waited
// for.  The gate weight is applied to h, before its rounding, so that the down product can add a token's experts in its
// accumulators: the rounding is relative, and the same as without it.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kernels/few_rows.cuh"
#include "kernels/pdl.cuh"
#include "rbv/moe.h"

namespace rbv {
namespace {

using namespace few;

constexpr int kMaxSlots = kMaxRows * kMoeFewMaxTopK;

struct FewArgs {
  const uint8_t* x;
  long long ldx;                          // bytes
  const float* logits;
  long long ldl;                          // elements
  int T, H, I, E, top_k;
  const uint8_t *w13, *w2;
  __nv_bfloat16* h;                       // [T * top_k, I], in the order of the used experts
  float* partial;                         // [2 * CTAs][T][tile]
  int* counters;                          // one per column tile of the down product
  __nv_bfloat16* out;
  int* error;
  int tile, box, stages;                  // weight rows of a piece and rows of A in a stage, at most; ring stages
};

// The choice, as every CTA makes it.
struct Choice {
  short expert[kMaxSlots];                // of slot t * top_k + j; negative: none
  float weight[kMaxSlots];
  short at[kMaxSlots];                    // row of the slot among its expert's rows
  short list[kMaxSlots];                  // slots by used expert
  short used[kMoeMaxExperts];             // experts that have rows, in order
  short index[kMoeMaxExperts];            // place of an expert in `used`
  short start[kMoeMaxExperts + 1];        // first entry of `list` of a used expert
  short rows[kMoeMaxExperts];             // rows of an expert
  int warp_used[8], warp_rows[8];
  int n_used, n_slots;
};

// Larger keys for larger logits, NaN above all, equal for both zeros; kMasked and below: -inf.
constexpr unsigned kMasked = 0x007fffffu;
__device__ __forceinline__ unsigned logit_key(float v) {
  if (v != v) return 0xffffffffu;
  const unsigned u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ void choose(Choice& c, const FewArgs& a) {   // all threads of the CTA
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
  const int slots = a.T * a.top_k;
  for (int t = warp; t < a.T; t += warps) {
    unsigned key[kMoeMaxExperts / 32];
    float val[kMoeMaxExperts / 32];
    const float* row = a.logits + (long long)t * a.ldl;
    #pragma unroll
    for (int j = 0; j < kMoeMaxExperts / 32; j++) {
      const int e = j * 32 + lane;
      val[j] = e < a.E ? __ldcg(row + e) : 0.0f;
    }
    #pragma unroll
    for (int j = 0; j < kMoeMaxExperts / 32; j++) key[j] = j * 32 + lane < a.E ? logit_key(val[j]) : 0u;
    float first = 0.0f, sum = 0.0f, mine = 0.0f;
    int chosen = -1;
    for (int k = 0; k < a.top_k; k++) {
      unsigned best = 0u;
      #pragma unroll
      for (int j = 0; j < kMoeMaxExperts / 32; j++) best = max(best, key[j]);
      best = __reduce_max_sync(0xffffffffu, best);
      if (best <= kMasked) break;
      int e = 0x7fffffff;
      #pragma unroll
      for (int j = kMoeMaxExperts / 32 - 1; j >= 0; j--)
        if (key[j] == best) e = j * 32 + lane;
      e = __reduce_min_sync(0xffffffffu, e);
      float v = 0.0f;
      #pragma unroll
      for (int j = 0; j < kMoeMaxExperts / 32; j++)
        if (j == (e >> 5)) {
          v = val[j];
          if (lane == (e & 31)) key[j] = 0u;
        }
      v = __shfl_sync(0xffffffffu, v, e & 31);
      if (k == 0) first = v;
      const float p = __expf(v - first);
      sum += p;
      if (lane == k) { chosen = e; mine = p; }
    }
    if (lane < a.top_k) {
      c.expert[t * a.top_k + lane] = (short)chosen;
      c.weight[t * a.top_k + lane] = chosen >= 0 ? mine / sum : 0.0f;
    }
  }
  __syncthreads();
  // rows of every expert, in the order of the slots
  int n = 0;
  if (tid < a.E) {
    for (int s = 0; s < slots; s++)
      if (c.expert[s] == tid) c.at[s] = (short)n++;
  }
  if (tid < kMoeMaxExperts) {
    // place among the used experts and first row: sums over the experts before
    const unsigned has = __ballot_sync(0xffffffffu, n > 0);
    int before = n;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += v;
    }
    if (lane == 31) { c.warp_used[warp] = __popc(has); c.warp_rows[warp] = before; }
    asm volatile("bar.sync 2, 256;" ::: "memory");
    int u = __popc(has & ((1u << lane) - 1u)), r = before - n, all_used = 0, all_rows = 0;
    for (int w = 0; w < 8; w++) {
      if (w < warp) { u += c.warp_used[w]; r += c.warp_rows[w]; }
      all_used += c.warp_used[w];
      all_rows += c.warp_rows[w];
    }
    if (n > 0) {
      c.used[u] = (short)tid;
      c.index[tid] = (short)u;
      c.start[u] = (short)r;
      c.rows[u] = (short)n;
    }
    if (tid == 0) { c.n_used = all_used; c.n_slots = all_rows; }
  }
  __syncthreads();
  for (int s = tid; s < slots; s += blockDim.x)
    if (c.expert[s] >= 0) c.list[c.start[c.index[c.expert[s]]] + c.at[s]] = (short)s;
  __syncthreads();
}

struct Shared {
  Ring ring;
  Choice choice;
  int flag;
};

__device__ __forceinline__ uint8_t* aligned_smem(uint8_t* p) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~uintptr_t(1023));
}

// ---- up: weight rows (gate and up interleaved) of the used experts, 8 at a time, split evenly among the CTAs ------------
struct UpPiece { int u, row0, rows; };    // used expert, first weight row, weight rows

struct UpWalk {
  long long at, end;
  int per_expert, tile;                   // in groups of 8 rows
  __device__ __forceinline__ UpWalk(const FewArgs& a, int n_used) {
    per_expert = 2 * a.I / 8;
    tile = a.tile / 8;
    const long long total = (long long)n_used * per_expert;
    at = total * blockIdx.x / gridDim.x;
    end = total * (blockIdx.x + 1) / gridDim.x;
  }
  __device__ __forceinline__ bool next(UpPiece& p) {
    if (at >= end) return false;
    p.u = (int)(at / per_expert);
    const int g = (int)(at - (long long)p.u * per_expert);
    const int n = (int)min((long long)min(tile, per_expert - g), end - at);
    p.row0 = g * 8;
    p.rows = n * 8;
    at += n;
    return true;
  }
};

template <typename S>
__device__ __forceinline__ bool up_piece(const FewArgs& a, Shared& s, uint4* red, uint32_t slots, Cursor& cur, const UpPiece& p, int warp,
                                         int lane, bool ok) {
  const int R = s.choice.rows[p.u], groups = p.rows / 8, part = warp >> 2, col = warp & 3;
  const int g0 = S::group0(part, groups), mine = S::my_groups(part, groups);
  uint32_t off[S::GROUPS];
  #pragma unroll
  for (int n = 0; n < S::GROUPS; n++) off[n] = group_offset(p.rows, g0 + n, col);
  const short* list = s.choice.list + s.choice.start[p.u];
  const uint8_t* src[S::MT][2];
  #pragma unroll
  for (int m = 0; m < S::MT; m++)
    #pragma unroll
    for (int h = 0; h < 2; h++) {
      const int r = S::row(m, S::set(part), h, lane);
      src[m][h] = r < R ? a.x + (long long)(list[r] / a.top_k) * a.ldx : nullptr;
    }
  float acc[S::MT][S::GROUPS][4];
  clear<S>(acc);
  const int row_bytes = 2 * a.H, chunks = (row_bytes + kChunk - 1) / kChunk;
  Rows<S> ahead[S::AHEAD + 1];             // (beyond the last chunk nothing is read)
  #pragma unroll
  for (int i = 0; i < S::AHEAD; i++) ahead[i].load(src, row_bytes, i, col, lane);
  for (int c = 0; c < chunks; c++) {
    ahead[S::AHEAD].load(src, row_bytes, c + S::AHEAD, col, lane);
    if (ok && !sm100::mbar_wait(&s.ring.full[cur.stage], cur.phase, &s.ring.abort)) { ok = false; s.ring.abort = 1; }
    __syncwarp();
    multiply<S>(acc, slots + (uint32_t)cur.stage * slot_bytes(a.tile, 0), off, mine, ahead[0], lane);
    __syncwarp();
    if (lane == 0) sm100::mbar_arrive(&s.ring.empty[cur.stage]);
    cur.next(a.stages);
    #pragma unroll
    for (int i = 0; i < S::AHEAD; i++) ahead[i] = ahead[i + 1];
  }
  #pragma unroll
  for (int m = 0; m < S::MT; m++) {
    float v[S::SETS][4];
    add_columns<S>(acc[m], red, groups, warp, lane, v);
    if (warp < groups)
      #pragma unroll
      for (int i = 0; i < 2 * S::SETS; i++) {
        const int q = i >> 1, h = i & 1, r = S::row(m, q, h, lane);
        if (r < R) {
          const int slot = list[r];
          const float gate = v[q][2 * h], up = v[q][2 * h + 1];
          const float y = s.choice.weight[slot] * (gate / (1.0f + __expf(-gate)) * up);
          a.h[(long long)(s.choice.start[p.u] + r) * a.I + p.row0 / 2 + warp * 4 + (lane & 3)] = __float2bfloat16_rn(y);
        }
      }
  }
  return ok;
}

// MAX: rows of an expert at most, 16, 32 or 64.
template <int MAX>
__global__ void __launch_bounds__(kThreads, 1) moe_few_up_kernel(const __grid_constant__ WeightMaps maps, const __grid_constant__ FewArgs a) {
  extern __shared__ uint8_t dyn[];
  __shared__ Shared s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* base = aligned_smem(dyn);
  uint4* red = reinterpret_cast<uint4*>(base);
  uint8_t* slots = base + red_bytes(a.tile);
  if (threadIdx.x == 0) ring_init(s.ring, a.stages, 1);
  pdl_wait();
  pdl_trigger();      // after the wait: the down kernel reads the logits before it waits for this one
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < a.H / 8; i += blockDim.x) a.counters[i] = 0;
  choose(s.choice, a);
  UpWalk walk(a, s.choice.n_used);
  UpPiece p;
  Cursor cur;
  if (warp >= kWarps) {
    if (warp != kWarps || lane != 0) return;
    const int chunks = (2 * a.H + kChunk - 1) / kChunk;
    bool ok = true;
    while (ok && walk.next(p)) {
      const int row0 = s.choice.used[p.u] * 2 * a.I + p.row0;
      for (int c = 0; c < chunks; c++) {
        ok = sm100::mbar_wait(&s.ring.empty[cur.stage], cur.phase ^ 1u, &s.ring.abort);
        if (!ok) break;
        fetch<__nv_bfloat16>(maps, slots + (size_t)cur.stage * slot_bytes(a.tile, 0), row0, p.rows, c, &s.ring.full[cur.stage]);
        cur.next(a.stages);
      }
    }
    if (!ok) s.ring.abort = 1;
    return;
  }
  bool ok = true;
  const uint32_t at = sm100::smem_u32(slots);
  while (walk.next(p)) {
    const int R = s.choice.rows[p.u];
    if (MAX == 16 || R <= 16) ok = up_piece<Spread<1, false>>(a, s, red, at, cur, p, warp, lane, ok);
    else if (MAX == 32 || R <= 32) ok = up_piece<Spread<2, false>>(a, s, red, at, cur, p, warp, lane, ok);
    else ok = up_piece<Spread<2, true>>(a, s, red, at, cur, p, warp, lane, ok);
  }
  if (!ok && a.error) atomicExch(a.error, 1);
}

// ---- down: column tiles of the result x used experts x chunks of K, split evenly among the CTAs -------------------------
struct DownWalk {
  Split split;
  long long at, end;
  int chunks, per_tile, n_used;
  int tile, u, c;                         // of step `at`
  __device__ __forceinline__ DownWalk(const FewArgs& a, int n_used_) {
    n_used = n_used_;
    chunks = (2 * a.I + kChunk - 1) / kChunk;
    per_tile = n_used * chunks;
    split.total = (long long)((a.H + a.tile - 1) / a.tile) * per_tile;
    split.parts = (int)min((long long)gridDim.x, split.total);
    at = end = 0;
    if ((int)blockIdx.x < split.parts) { at = split.begin(blockIdx.x); end = split.begin(blockIdx.x + 1); }
    tile = (int)(at / per_tile);
    const int in_tile = (int)(at - (long long)tile * per_tile);
    u = in_tile / chunks;
    c = in_tile - u * chunks;
  }
  __device__ __forceinline__ void step() {
    at++;
    if (++c == chunks) {
      c = 0;
      if (++u == n_used) { u = 0; tile++; }
    }
  }
};

template <typename S>       // by the tokens: 16, 32 or 64 at most
__global__ void __launch_bounds__(kThreads, 1) moe_few_down_kernel(const __grid_constant__ WeightMaps maps, const __grid_constant__ WeightMaps h_maps,
                                                                   const __grid_constant__ FewArgs a) {
  extern __shared__ uint8_t dyn[];
  __shared__ Shared s;
  constexpr int MT = S::MT;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* base = aligned_smem(dyn);
  uint4* red = reinterpret_cast<uint4*>(base);
  uint8_t* slots = base + red_bytes(a.tile);
  if (tid == 0) ring_init(s.ring, a.stages, 2);
  pdl_trigger();
  choose(s.choice, a);
  const int n_used = s.choice.n_used;
  if (n_used == 0) {                      // every token masked
    pdl_wait();
    for (long long i = blockIdx.x * (long long)blockDim.x + tid; i < (long long)a.T * a.H; i += (long long)gridDim.x * blockDim.x)
      a.out[i] = __float2bfloat16_rn(0.0f);
    return;
  }
  DownWalk walk(a, n_used);
  Cursor cur;
  if (warp >= kWarps) {                   // the weights do not wait for the first kernel, the rows of h do
    if (lane != 0) return;
    const bool weights = warp == kWarps;
    bool ok = true;
    if (!weights) {
      pdl_wait();
      asm volatile("fence.proxy.async;" ::: "memory");
    }
    for (; walk.at < walk.end; walk.step()) {
      ok = sm100::mbar_wait(&s.ring.empty[cur.stage], cur.phase ^ 1u, &s.ring.abort);
      if (!ok) break;
      uint8_t* slot = slots + (size_t)cur.stage * slot_bytes(a.tile, a.box);
      uint64_t* bar = &s.ring.full[cur.stage];
      if (weights) {
        const int col0 = walk.tile * a.tile;
        fetch<__nv_bfloat16>(maps, slot, s.choice.used[walk.u] * a.H + col0, min(a.tile, a.H - col0), walk.c, bar);
      } else {
        fetch<__nv_bfloat16>(h_maps, slot + a.tile * kChunk, s.choice.start[walk.u], box_rows(s.choice.rows[walk.u]), walk.c, bar);
      }
      cur.next(a.stages);
    }
    if (!ok) s.ring.abort = 1;
    return;
  }
  pdl_wait();
  bool ok = true;
  const uint32_t slots_at = sm100::smem_u32(slots);
  const int part = warp >> 2, wcol = warp & 3;
  while (walk.at < walk.end) {
    const int tile = walk.tile;
    const long long first = (long long)tile * walk.per_tile, at0 = walk.at, stop = min(walk.end, first + walk.per_tile);
    const int col0 = tile * a.tile, nr = min(a.tile, a.H - col0), groups = nr / 8;
    const int g0 = S::group0(part, groups), mine = S::my_groups(part, groups);
    uint32_t off[S::GROUPS];
    #pragma unroll
    for (int n = 0; n < S::GROUPS; n++) off[n] = group_offset(nr, g0 + n, wcol);
    float acc[MT][S::GROUPS][4];
    clear<S>(acc);
    // where the tokens' rows of h are in a stage of expert u: tokens that did not choose it count as zeros
    int u = -1, box = 0, rows_at[MT][2];
    for (; walk.at < stop; walk.step()) {
      if (walk.u != u) {
        u = walk.u;
        box = box_rows(s.choice.rows[u]);
        const int e = s.choice.used[u];
        #pragma unroll
        for (int m = 0; m < MT; m++)
          #pragma unroll
          for (int h = 0; h < 2; h++) {
            const int t = S::row(m, S::set(part), h, lane);
            rows_at[m][h] = -1;
            if (t < a.T)
              for (int j = 0; j < a.top_k; j++)
                if (s.choice.expert[t * a.top_k + j] == e) rows_at[m][h] = s.choice.at[t * a.top_k + j];
          }
      }
      if (ok && !sm100::mbar_wait(&s.ring.full[cur.stage], cur.phase, &s.ring.abort)) { ok = false; s.ring.abort = 1; }
      __syncwarp();
      const uint32_t slot = slots_at + (uint32_t)cur.stage * slot_bytes(a.tile, a.box);
      Rows<S> rows;
      rows.load(rows_at, slot + (uint32_t)a.tile * kChunk, box, wcol, lane);
      multiply<S>(acc, slot, off, mine, rows, lane);
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&s.ring.empty[cur.stage]);
      cur.next(a.stages);
    }
    const bool whole = at0 == first && stop == first + walk.per_tile;
    // a tile cut by the end of a range: sums to the workspace, the last CTA to arrive adds them up
    float* part = a.partial + (2ll * blockIdx.x + (at0 == first ? 1 : 0)) * a.T * a.tile;
    #pragma unroll
    for (int m = 0; m < MT; m++) {
      float v[S::SETS][4];
      add_columns<S>(acc[m], red, groups, warp, lane, v);
      if (warp < groups)
        #pragma unroll
        for (int i = 0; i < 2 * S::SETS; i++) {
          const int q = i >> 1, h = i & 1, t = S::row(m, q, h, lane), col = warp * 8 + (lane & 3) * 2;
          if (t >= a.T) continue;
          if (whole)
            *reinterpret_cast<__nv_bfloat162*>(a.out + (long long)t * a.H + col0 + col) = __floats2bfloat162_rn(v[q][2 * h], v[q][2 * h + 1]);
          else
            *reinterpret_cast<float2*>(part + (long long)t * a.tile + col) = make_float2(v[q][2 * h], v[q][2 * h + 1]);
        }
    }
    if (!whole) {
      const int c0 = walk.split.owner(first), c1 = walk.split.owner(first + walk.per_tile - 1);
      if (last_to_arrive(a.counters + tile, c1 - c0 + 1, &s.flag)) {
        const int pairs = nr / 2;
        for (int i = tid; i < a.T * pairs; i += kWarps * 32) {
          const int t = i / pairs, col = (i - t * pairs) * 2;
          float2 sum = make_float2(0.0f, 0.0f);
          for (int k = c0; k <= c1; k++) {
            const bool starts = max(walk.split.begin(k), first) == first;
            const float2 v = __ldcg(reinterpret_cast<const float2*>(a.partial + (2ll * k + (starts ? 1 : 0)) * a.T * a.tile +
                                                                    (long long)t * a.tile + col));
            sum.x += v.x;
            sum.y += v.y;
          }
          *reinterpret_cast<__nv_bfloat162*>(a.out + (long long)t * a.H + col0 + col) = __floats2bfloat162_rn(sum.x, sum.y);
        }
      }
    }
  }
  if (!ok && a.error) atomicExch(a.error, 2);
}

// ---- host side -------------------------------------------------------------------------------------------------------
struct FewPlan { int sms, up_tile, down_tile; size_t h_bytes, partial_bytes, counter_bytes; };

size_t round_up(size_t v, size_t to) { return (v + to - 1) / to * to; }

bool few_plan(int T, int H, int I, int E, int top_k, FewPlan* p) {
  if (T < 1 || T > kMaxRows || E < 1 || E > kMoeMaxExperts || top_k < 1 || top_k > kMoeFewMaxTopK || top_k > E) return false;
  if (H < 8 || I < 8 || H % 8 || I % 8 || 2ll * E * I > 0x7fffffffll || (long long)E * H > 0x7fffffffll) return false;
  if (H > (1 << 24) || I > (1 << 24)) return false;      // (row lengths in bytes, and coordinates a box beyond them, fit an int)
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&p->sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return false;
  const int used = E < T * top_k ? E : T * top_k;   // experts in use, at most
  p->up_tile = tile_rows((long long)used * (2 * I / 8), p->sms);
  // columns of the result in a piece: the most, in one box, that leave a CTA eight steps to share the work out evenly
  const long long steps = (long long)used * ((2 * I + kChunk - 1) / kChunk);
  p->down_tile = kMaxTile;
  while (p->down_tile > 8 && (H + p->down_tile - 1) / p->down_tile * steps < 8ll * p->sms) p->down_tile /= 2;
  p->h_bytes = round_up((size_t)T * top_k * I * 2, 256);
  p->partial_bytes = round_up((size_t)2 * p->sms * T * p->down_tile * 4, 256);
  p->counter_bytes = round_up((size_t)(H / 8) * 4, 256);
  return true;
}

template <int MAX, typename S>
cudaError_t few_launch(FewArgs a, const FewPlan& p, cudaStream_t st) {
  const CUtensorMapDataType bf16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  WeightMaps w13, w2, h;
  if (!weight_maps(&w13, a.w13, 2ull * a.E * a.I, 2ull * a.H, bf16, 2) || !weight_maps(&w2, a.w2, (unsigned long long)a.E * a.H, 2ull * a.I, bf16, 2) ||
      !weight_maps(&h, a.h, (unsigned long long)a.T * a.top_k, 2ull * a.I, bf16, 2))
    return cudaErrorUnknown;
  auto launch = [&](auto kernel, int tile, int box, const auto&... maps) {
    a.tile = tile;
    a.box = box;
    a.stages = ring_stages(tile, box, sizeof(Shared));
    const size_t smem = ring_smem(tile, box, a.stages);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    return e != cudaSuccess ? e : launch_dependent(kernel, dim3(p.sms), dim3(kThreads), smem, st, maps..., a);
  };
  const cudaError_t e = launch(moe_few_up_kernel<MAX>, p.up_tile, 0, w13);
  return e != cudaSuccess ? e : launch(moe_few_down_kernel<S>, p.down_tile, box_rows(a.T), w2, h);
}

}  // namespace
}  // namespace rbv

using namespace rbv;

extern "C" long long rbv_moe_few_workspace(int T, int H, int I, int E, int top_k) {
  FewPlan p;
  return few_plan(T, H, I, E, top_k, &p) ? (long long)(p.h_bytes + p.partial_bytes + p.counter_bytes) : -1;
}

extern "C" int rbv_moe_few_tokens(const void* x, long long ldx, const float* logits, long long ldl, int T, int H, int I, int E,
                                  int top_k, const void* w13, const void* w2, void* out, void* workspace, int* error_flag,
                                  void* stream) {
  FewPlan p;
  if (!few_plan(T, H, I, E, top_k, &p) || !x || !logits || !w13 || !w2 || !out || !workspace) return (int)cudaErrorInvalidValue;
  if ((T > 1 && (ldx < H || ldl < E)) || ldx % 8) return (int)cudaErrorInvalidValue;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w13) | reinterpret_cast<uintptr_t>(w2) |
       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return (int)cudaErrorMisalignedAddress;
  FewArgs a{};
  a.x = static_cast<const uint8_t*>(x); a.ldx = ldx * 2; a.logits = logits; a.ldl = ldl;
  a.T = T; a.H = H; a.I = I; a.E = E; a.top_k = top_k;
  a.w13 = static_cast<const uint8_t*>(w13); a.w2 = static_cast<const uint8_t*>(w2);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.h = reinterpret_cast<__nv_bfloat16*>(ws);
  a.partial = reinterpret_cast<float*>(ws + p.h_bytes);
  a.counters = reinterpret_cast<int*>(ws + p.h_bytes + p.partial_bytes);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.error = error_flag;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T <= 16) return (int)few_launch<16, Spread<1, false>>(a, p, st);
  if (T <= 32) return (int)few_launch<32, Spread<2, false>>(a, p, st);
  return (int)few_launch<64, Spread<2, true>>(a, p, st);
}
