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
// accumulators: the rounding is relative, and the same as without it.  h is rounded because the tensor cores take 16 bits: a second
// bf16 term for the rest would double h and the multiplications of the down product, which 32 and 64 tokens are near to being
// bound by.  It costs as much as the rounding of the result: 0.0024 of a result's size (root mean square) against 64 bits, where the
// last rounding alone leaves 0.0017, as in the layer's general path.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "kernels/few_rows.cuh"
#include "kernels/pdl.cuh"
#include "rbv/moe.h"

namespace rbv {
namespace {

using namespace few;

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
  int tile, room, whole;                  // weight rows of a piece at most; bytes of the ring; whole: tiles of the down product are
                                          // not split
  uint32_t red;                           // bytes in which warps add their sums
};

// The choice, as every CTA makes it.
template <int TOKENS>
struct Choice {
  static constexpr int kMaxSlots = TOKENS * RBV_FEW_MAX_TOP_K;
  short expert[kMaxSlots];                // of slot t * top_k + j; negative: none
  float weight[kMaxSlots];
  short at[kMaxSlots];                    // row of the slot among its expert's rows
  short list[kMaxSlots];                  // slots by used expert
  short used[kMoeMaxExperts];             // experts that have rows
  short index[kMoeMaxExperts];            // place of an expert in `used`
  short start[kMoeMaxExperts];            // first entry of `list` of a used expert
  short rows[kMoeMaxExperts];             // rows of a used expert
  int warp_used[8], warp_rows[8], warp_most[8];
  int n_used, most;                       // most: rows of the expert with most
};

// Larger keys for larger logits, NaN above all, equal for both zeros; kMasked and below: -inf.
constexpr unsigned kMasked = 0x007fffffu;
__device__ __forceinline__ unsigned logit_key(float v) {
  if (v != v) return 0xffffffffu;
  const unsigned u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The choice of one token by one warp, for E <= 32 * WORDS; lane j gets the j-th expert (negative: none) and its weight.
template <int WORDS>
__device__ __forceinline__ void choose_token(const float* row, int E, int top_k, int lane, int& expert, float& weight) {
  unsigned key[WORDS];
  float val[WORDS];
  #pragma unroll
  for (int j = 0; j < WORDS; j++) val[j] = j * 32 + lane < E ? __ldcg(row + j * 32 + lane) : 0.0f;
  #pragma unroll
  for (int j = 0; j < WORDS; j++) key[j] = j * 32 + lane < E ? logit_key(val[j]) : 0u;
  float first = 0.0f, sum = 0.0f;
  expert = -1;
  weight = 0.0f;
  for (int k = 0; k < top_k; k++) {
    unsigned best = 0u;
    #pragma unroll
    for (int j = 0; j < WORDS; j++) best = max(best, key[j]);
    best = __reduce_max_sync(0xffffffffu, best);
    if (best <= kMasked) break;
    int e = 0x7fffffff;
    #pragma unroll
    for (int j = WORDS - 1; j >= 0; j--)
      if (key[j] == best) e = j * 32 + lane;
    e = __reduce_min_sync(0xffffffffu, e);
    float v = 0.0f;
    #pragma unroll
    for (int j = 0; j < WORDS; j++)
      if (j == (e >> 5)) {
        v = val[j];
        if (lane == (e & 31)) key[j] = 0u;
      }
    v = __shfl_sync(0xffffffffu, v, e & 31);
    if (k == 0) first = v;
    const float p = __expf(v - first);
    sum += p;
    if (lane == k) { expert = e; weight = p; }
  }
  if (expert >= 0) weight /= sum;
}

template <int TOKENS>
__device__ __forceinline__ void choose(Choice<TOKENS>& c, const FewArgs& a) {   // all threads of the CTA
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
  const int slots = a.T * a.top_k;
  for (int t = warp; t < a.T; t += warps) {
    const float* row = a.logits + (long long)t * a.ldl;
    int expert;
    float weight;
    if (a.E <= 64) choose_token<2>(row, a.E, a.top_k, lane, expert, weight);
    else choose_token<kMoeMaxExperts / 32>(row, a.E, a.top_k, lane, expert, weight);
    if (lane < a.top_k) {
      c.expert[t * a.top_k + lane] = (short)expert;
      c.weight[t * a.top_k + lane] = weight;
    }
  }
  __syncthreads();
  if (slots <= 32) {
    // a warp sees all slots: experts in the order of their first slot
    if (warp == 0) {
      const int e = lane < slots ? c.expert[lane] : -1;
      const unsigned live = __ballot_sync(0xffffffffu, e >= 0), same = __match_any_sync(0xffffffffu, e) & live, below = (1u << lane) - 1u;
      const bool first = e >= 0 && (same & below) == 0;
      const unsigned firsts = __ballot_sync(0xffffffffu, first);
      const int n = __popc(same), u = __popc(firsts & below);
      int start = first ? n : 0;
      #pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, start, o);
        if (lane >= o) start += v;
      }
      start -= first ? n : 0;
      start = __shfl_sync(0xffffffffu, start, same ? __ffs(same) - 1 : 0);
      if (first) {
        c.used[u] = (short)e;
        c.start[u] = (short)start;
        c.rows[u] = (short)n;
      }
      if (e >= 0) {
        const int at = __popc(same & below);
        c.at[lane] = (short)at;
        c.list[start + at] = (short)lane;
      }
      const int most = __reduce_max_sync(0xffffffffu, e >= 0 ? n : 0);
      if (lane == 0) { c.n_used = __popc(firsts); c.most = most; }
    }
    __syncthreads();
    return;
  }
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
    const int warp_most = __reduce_max_sync(0xffffffffu, n);
    if (lane == 31) { c.warp_used[warp] = __popc(has); c.warp_rows[warp] = before; c.warp_most[warp] = warp_most; }
    consumers_sync();
    int u = __popc(has & ((1u << lane) - 1u)), r = before - n, all_used = 0, most = 0;
    for (int w = 0; w < 8; w++) {
      if (w < warp) { u += c.warp_used[w]; r += c.warp_rows[w]; }
      all_used += c.warp_used[w];
      most = max(most, c.warp_most[w]);
    }
    if (n > 0) {
      c.used[u] = (short)tid;
      c.index[tid] = (short)u;
      c.start[u] = (short)r;
      c.rows[u] = (short)n;
    }
    if (tid == 0) { c.n_used = all_used; c.most = most; }
  }
  __syncthreads();
  for (int s = tid; s < slots; s += blockDim.x)
    if (c.expert[s] >= 0) c.list[c.start[c.index[c.expert[s]]] + c.at[s]] = (short)s;
  __syncthreads();
}

template <int TOKENS>
struct Shared {
  Ring ring;
  Choice<TOKENS> choice;
  int flag[2];
};
__device__ __forceinline__ uint8_t* aligned_smem(uint8_t* p) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~uintptr_t(1023));
}

// The ring for stages of a.tile weight rows and `box` rows of A.
__device__ __forceinline__ Cursor ring_cursor(Ring& ring, const FewArgs& a, uint32_t at, int box) {
  const uint32_t slot = slot_bytes(a.tile, box);
  return Cursor(ring, at, min(kMaxStages, (int)((uint32_t)a.room / slot)), slot);
}

// ---- up: weight rows (gate and up interleaved) of the used experts, 8 at a time, split evenly among the CTAs ------------
struct UpPiece { int u, row0, rows; };    // used expert, first weight row, weight rows

struct UpWalk {
  unsigned at, end, per_expert, tile;     // in groups of 8 rows
  unsigned u, g;                          // used expert and group of `at`
  __device__ __forceinline__ UpWalk(const FewArgs& a, int n_used) {
    per_expert = 2 * a.I / 8;
    tile = a.tile / 8;
    const Split split{n_used * per_expert, gridDim.x, 1};
    at = split.begin(blockIdx.x);
    end = split.begin(blockIdx.x + 1);
    u = at / per_expert;
    g = at - u * per_expert;
  }
  __device__ __forceinline__ bool next(UpPiece& p) {
    if (at >= end) return false;
    if (g == per_expert) { g = 0; u++; }
    const unsigned n = min(min(tile, per_expert - g), end - at);
    p.u = u;
    p.row0 = g * 8;
    p.rows = n * 8;
    at += n;
    g += n;
    return true;
  }
};

// The steps along K of a piece: NT tiles of 8 rows of A, at `rows_at` of a box of `box` rows.
template <int NT>
__device__ __forceinline__ void run_steps(float (&acc)[kGroups][NT][4], Cursor& cur, int steps, int tile, int box, const int (&rows_at)[NT],
                                          const Offsets& off, const Share& share, int col, int lane) {
  auto run = [&](auto tag) {
    constexpr int G = decltype(tag)::value;
    #pragma unroll 1
    for (int c = 0; c < steps; c++) {
      cur.wait_full();
      __syncwarp();
      Rows<NT> rows;
      rows.load(rows_at, cur.slot + (uint32_t)tile * kChunk, box, col, lane);
      multiply<G>(acc, cur.slot, off, rows, lane);
      __syncwarp();
      if (lane == 0) cur.release();
      cur.next();
    }
  };
  if (share.count <= 1) run(std::integral_constant<int, 1>());
  else run(std::integral_constant<int, kGroups>());
}

// f(tag of the tiles of 8) for R rows, at most MAX.
template <int MAX, typename F>
__device__ __forceinline__ void by_tiles(int R, F&& f) {
  if (R <= 8) f(std::integral_constant<int, 1>());
  else if (MAX <= 16 || R <= 16) f(std::integral_constant<int, 2>());
  else if (R <= 24) f(std::integral_constant<int, 3>());
  else if (MAX <= 32 || R <= 32) f(std::integral_constant<int, 4>());
  else f(std::integral_constant<int, 8>());
}

// Tokens of an expert with R rows come in one box of all tokens, or gathered four rows at a time.  A box of all is an
// instruction and up to 16 KB (32 tokens) or 32 KB (64), beside 32 KB of weights; gathering takes R instructions of some 90
// cycles each, and a stage's weights 1260.
template <int MAX> __device__ __forceinline__ bool in_one_box(int R) { return MAX == 16 || R > (MAX == 32 ? 4 : 8); }
template <int MAX> __device__ __forceinline__ int token_box(int T, int R) { return box_rows(in_one_box<MAX>(R) ? T : R); }
template <int MAX> struct XMaps { WeightMaps box; CUtensorMap rows; };

template <int NT, int MAX>
__device__ __forceinline__ void up_piece(const FewArgs& a, Shared<MAX>& s, Red& red, Cursor& cur, const UpPiece& p, int warp, int lane) {
  const int R = s.choice.rows[p.u], part = warp >> 2, col = warp & 3;
  const Share share(p.rows, part);
  const Offsets off(p.rows, share, col);
  const short* list = s.choice.list + s.choice.start[p.u];
  int rows_at[NT];
  #pragma unroll
  for (int i = 0; i < NT; i++) {
    const int r = 8 * i + (lane >> 2);
    rows_at[i] = r >= R ? -1 : in_one_box<MAX>(R) ? list[r] / a.top_k : r;
  }
  float acc[kGroups][NT][4];
  clear(acc);
  run_steps<NT>(acc, cur, (2 * a.H + kChunk - 1) / kChunk, a.tile, token_box<MAX>(a.T, R), rows_at, off, share, col, lane);
  add_columns<NT>(acc, red, share, part, col, lane, [&](int r, int row, float gate, float up) {
    if (r >= R || row >= p.rows) return;
    const float y = s.choice.weight[list[r]] * (gate / (1.0f + __expf(-gate)) * up);
    a.h[(long long)(s.choice.start[p.u] + r) * a.I + (p.row0 + row) / 2] = __float2bfloat16_rn(y);
  });
}

// MAX: tokens, and with them rows of an expert, at most: 16, 32 or 64.
template <int MAX>
__global__ void __launch_bounds__(kThreads, 1) moe_few_up_kernel(const __grid_constant__ WeightMaps maps, const __grid_constant__ XMaps<MAX> x_maps,
                                                                 const __grid_constant__ FewArgs a) {
  extern __shared__ uint8_t dyn[];
  __shared__ Shared<MAX> s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* base = aligned_smem(dyn);
  Red red{reinterpret_cast<uint4*>(base), a.red > kRedBytes};
  ring_init_all(s.ring, 2);
  if (warp == kWarps) prefetch_maps(maps);
  if (warp == kWarps + 1) prefetch_maps(x_maps.box);
  pdl_wait();
  pdl_trigger();      // after the wait: the down kernel reads the logits before it waits for this one
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < a.H / 8; i += blockDim.x) a.counters[i] = 0;
  choose(s.choice, a);
  UpWalk walk(a, s.choice.n_used);
  UpPiece p;
  Cursor cur = ring_cursor(s.ring, a, sm100::smem_u32(base + a.red), token_box<MAX>(a.T, s.choice.most));
  const int chunks = (2 * a.H + kChunk - 1) / kChunk;
  if (warp == kWarps) {
    if (lane >= 4) return;
    while (walk.next(p) && feed<__nv_bfloat16>(maps, cur, 0, s.choice.used[p.u] * 2 * a.I + p.row0, p.rows, 0, chunks)) {}
    return;
  }
  if (warp == kWarps + 1) {
    asm volatile("fence.proxy.async;" ::: "memory");
    bool ok = true;
    while (ok && walk.next(p)) {
      const int R = s.choice.rows[p.u];
      const short* list = s.choice.list + s.choice.start[p.u];
      if (in_one_box<MAX>(R)) ok = feed<__nv_bfloat16>(x_maps.box, cur, (uint32_t)a.tile * kChunk, 0, box_rows(a.T), 0, chunks);
      else ok = feed_gathered<__nv_bfloat16>(&x_maps.rows, cur, (uint32_t)a.tile * kChunk, R, 0, chunks, [&](int r) { return list[r] / a.top_k; });
    }
    return;
  }
  while (walk.next(p))
    by_tiles<MAX>(s.choice.rows[p.u], [&](auto tag) { up_piece<decltype(tag)::value>(a, s, red, cur, p, warp, lane); });
  if (!cur.ok && a.error) atomicExch(a.error, 1);
}

// ---- down: column tiles of the result x used experts x chunks of K, split evenly among the CTAs -------------------------
struct DownPiece { int tile, u, c0, c1; };       // column tile, used expert, chunks of K

struct DownWalk {
  Split split;
  unsigned at, end, per_tile;             // in steps
  int chunks, n_used;
  int tile, u, c;                         // of step `at`
  __device__ __forceinline__ DownWalk(const FewArgs& a, int n_used_) {
    n_used = n_used_;
    chunks = (2 * a.I + kChunk - 1) / kChunk;
    per_tile = n_used * chunks;
    const unsigned tiles = (a.H + a.tile - 1) / a.tile;
    split.grain = a.whole ? per_tile : 1;
    split.total = a.whole ? tiles : tiles * per_tile;
    split.parts = min(gridDim.x, split.total);
    at = end = 0;
    if (blockIdx.x < split.parts) { at = split.begin(blockIdx.x); end = split.begin(blockIdx.x + 1); }
    tile = at / per_tile;
    const unsigned in_tile = at - tile * per_tile;
    u = in_tile / chunks;
    c = in_tile - u * chunks;
  }
  __device__ __forceinline__ bool next(DownPiece& p) {
    if (at >= end) return false;
    p.tile = tile;
    p.u = u;
    p.c0 = c;
    p.c1 = (int)min((unsigned)chunks, c + (end - at));
    at += p.c1 - p.c0;
    c = 0;                                // (the next one begins an expert, or there is none)
    if (++u == n_used) { u = 0; tile++; }
    return true;
  }
};

// More than 16 tokens: an expert's rows by themselves, as in the up product; their sums over the expert's K are added to the
// tokens' sums in shared memory, expert by expert.
template <int NT, int MAX>
__device__ __forceinline__ void down_piece(const FewArgs& a, Shared<MAX>& s, Red& red, float* sums, Cursor& cur, const DownPiece& p, int nr,
                                           int warp, int lane) {
  const int R = s.choice.rows[p.u], part = warp >> 2, col = warp & 3;
  const Share share(nr, part);
  const Offsets off(nr, share, col);
  int rows_at[NT];
  #pragma unroll
  for (int i = 0; i < NT; i++) {
    const int r = 8 * i + (lane >> 2);
    rows_at[i] = r < R ? r : -1;
  }
  float acc[kGroups][NT][4];
  clear(acc);
  run_steps<NT>(acc, cur, p.c1 - p.c0, a.tile, box_rows(R), rows_at, off, share, col, lane);
  const short* list = s.choice.list + s.choice.start[p.u];
  add_columns<NT>(acc, red, share, part, col, lane, [&](int r, int n, float v0, float v1) {
    if (r >= R || n >= nr) return;
    float2* at = reinterpret_cast<float2*>(sums + list[r] / a.top_k * kMaxTile + n);
    float2 v = *at;
    v.x += v0;
    v.y += v1;
    *at = v;
  });
  consumers_sync();                       // other warps may have these sums in the next piece
}

template <int MAX>
__global__ void __launch_bounds__(kThreads, 1) moe_few_down_kernel(const __grid_constant__ WeightMaps maps, const __grid_constant__ WeightMaps h_maps,
                                                                   const __grid_constant__ FewArgs a) {
  extern __shared__ uint8_t dyn[];
  __shared__ Shared<MAX> s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* base = aligned_smem(dyn);
  Red red{reinterpret_cast<uint4*>(base), a.red > kRedBytes};
  float* sums = reinterpret_cast<float*>(base + a.red);                // [MAX][kMaxTile] beyond 16 tokens
  constexpr uint32_t kSumBytes = MAX > 16 ? MAX * kMaxTile * 4 : 0;
  ring_init_all(s.ring, 2);
  if (warp >= kWarps) prefetch_maps(warp == kWarps ? maps : h_maps);
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
  DownPiece p;
  Cursor cur = ring_cursor(s.ring, a, sm100::smem_u32(base + a.red + kSumBytes), box_rows(s.choice.most));
  if (warp >= kWarps) {                   // the weights do not wait for the first kernel, the rows of h do
    if (lane >= 4) return;
    if (warp == kWarps) {
      while (walk.next(p)) {
        const int col0 = p.tile * a.tile;
        if (!feed<__nv_bfloat16>(maps, cur, 0, s.choice.used[p.u] * a.H + col0, min(a.tile, a.H - col0), p.c0, p.c1)) break;
      }
    } else {
      pdl_wait();
      asm volatile("fence.proxy.async;" ::: "memory");
      while (walk.next(p) &&
             feed<__nv_bfloat16>(h_maps, cur, (uint32_t)a.tile * kChunk, s.choice.start[p.u], box_rows(s.choice.rows[p.u]), p.c0, p.c1)) {}
    }
    return;
  }
  pdl_wait();
  int cut[2] = {-1, -1};                  // tiles shared with the CTA before and the CTA behind
  const int part = warp >> 2, wcol = warp & 3;
  bool more = walk.next(p);
  while (more) {
    const int tile = p.tile, col0 = tile * a.tile, nr = min(a.tile, a.H - col0);
    const bool starts = p.u == 0 && p.c0 == 0;
    bool ends;
    // a tile cut by the end of a range: the sums go to the workspace, for the last CTA to arrive
    float* part_sums = a.partial + (2ll * blockIdx.x + (starts ? 1 : 0)) * a.T * a.tile;
    auto result = [&](bool whole, int t, int col, float v0, float v1) {
      if (whole) *reinterpret_cast<__nv_bfloat162*>(a.out + (long long)t * a.H + col0 + col) = __floats2bfloat162_rn(v0, v1);
      else *reinterpret_cast<float2*>(part_sums + (long long)t * a.tile + col) = make_float2(v0, v1);
    };
    bool whole;
    if constexpr (MAX == 16) {
      // all tokens at once, those that did not choose an expert as zeros: its sums stay in the accumulators
      const Share share(nr, part);
      const Offsets off(nr, share, wcol);
      auto tokens = [&](auto tag) {
        constexpr int NT = decltype(tag)::value;
        float acc[kGroups][NT][4];
        clear(acc);
        do {
          const int e = s.choice.used[p.u];
          int rows_at[NT];
          #pragma unroll
          for (int i = 0; i < NT; i++) {
            const int t = 8 * i + (lane >> 2);
            rows_at[i] = -1;
            if (t < a.T)
              for (int j = 0; j < a.top_k; j++)
                if (s.choice.expert[t * a.top_k + j] == e) rows_at[i] = s.choice.at[t * a.top_k + j];
          }
          run_steps<NT>(acc, cur, p.c1 - p.c0, a.tile, box_rows(s.choice.rows[p.u]), rows_at, off, share, wcol, lane);
          ends = p.u == n_used - 1 && p.c1 == walk.chunks;
          more = walk.next(p);
        } while (more && p.tile == tile);
        whole = starts && ends;
        add_columns<NT>(acc, red, share, part, wcol, lane, [&](int t, int col, float v0, float v1) {
          if (t < a.T && col < nr) result(whole, t, col, v0, v1);
        });
      };
      if (a.T <= 8) tokens(std::integral_constant<int, 1>());
      else tokens(std::integral_constant<int, 2>());
    } else {
      for (int i = tid; i < a.T * kMaxTile; i += kWarps * 32) sums[i] = 0.0f;
      consumers_sync();
      do {
        by_tiles<MAX>(s.choice.rows[p.u], [&](auto tag) { down_piece<decltype(tag)::value>(a, s, red, sums, cur, p, nr, warp, lane); });
        ends = p.u == n_used - 1 && p.c1 == walk.chunks;
        more = walk.next(p);
      } while (more && p.tile == tile);
      whole = starts && ends;
      for (int i = tid; i < a.T * (nr / 2); i += kWarps * 32) {
        const int t = i / (nr / 2), col = (i - t * (nr / 2)) * 2;
        const float2 v = *reinterpret_cast<const float2*>(sums + t * kMaxTile + col);
        result(whole, t, col, v.x, v.y);
      }
      consumers_sync();                   // the sums are free for the next tile
    }
    if (!whole) cut[starts ? 1 : 0] = tile;
  }
  // the (at most two) tiles that this CTA shares with others
  if (cut[0] >= 0 || cut[1] >= 0) {
    auto owners = [&](int tile, int& c0, int& c1) {
      const unsigned first = tile * walk.per_tile;
      c0 = walk.split.owner(first);
      c1 = walk.split.owner(first + walk.per_tile - 1);
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
      s.flag[tid] = last;
    }
    consumers_sync();
    for (int i = 0; i < 2; i++) {
      if (!s.flag[i]) continue;
      __threadfence();
      int c0, c1;
      owners(cut[i], c0, c1);
      const int col0 = cut[i] * a.tile, pairs = min(a.tile, a.H - col0) / 2;
      for (int k = tid; k < a.T * pairs; k += kWarps * 32) {
        const int t = k / pairs, col = (k - t * pairs) * 2;
        // only the first one's range may have begun before the tile
        const float* from = a.partial + 2ll * c0 * a.T * a.tile + (long long)t * a.tile + col;
        float2 sum = __ldcg(reinterpret_cast<const float2*>(from + a.T * a.tile));
        #pragma unroll 4
        for (int c = 1; c <= c1 - c0; c++) {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(from + 2ll * c * a.T * a.tile));
          sum.x += v.x;
          sum.y += v.y;
        }
        *reinterpret_cast<__nv_bfloat162*>(a.out + (long long)t * a.H + col0 + col) = __floats2bfloat162_rn(sum.x, sum.y);
      }
    }
  }
  if (!cur.ok && a.error) atomicExch(a.error, 2);
}

// ---- host side -------------------------------------------------------------------------------------------------------
struct FewPlan { int sms, up_tile, down_tile, whole; size_t h_bytes, partial_bytes, counter_bytes; };

size_t round_up(size_t v, size_t to) { return (v + to - 1) / to * to; }

bool few_plan(int T, int H, int I, int E, int top_k, FewPlan* p) {
  if (T < 1 || T > kMaxRows || E < 1 || E > kMoeMaxExperts || top_k < 1 || top_k > RBV_FEW_MAX_TOP_K || top_k > E) return false;
  if (H < 8 || I < 8 || H % 8 || I % 8 || 2ll * E * I > 0x7fffffffll || (long long)E * H > 0x7fffffffll) return false;
  if (H > (1 << 24) || I > (1 << 24)) return false;      // (row lengths in bytes, and coordinates a box beyond them, fit an int)
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&p->sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return false;
  const int used = E < T * top_k ? E : T * top_k;   // experts in use, at most
  p->up_tile = tile_rows((long long)used * (2 * I / 8), p->sms);
  const bool each = T > 16;                         // the down product goes expert by expert
  const int row_tiles = each ? (T * top_k + 8 * used - 1) / (8 * used) : (T + 7) / 8;
  if (!split_plan(H, 2ll * I, used, p->sms, T, row_tiles, each, &p->down_tile, &p->whole) || (long long)used * (2 * I / 8) * p->sms > 0xffffffffll) return false;
  p->h_bytes = round_up((size_t)T * top_k * I * 2, 256);
  p->partial_bytes = round_up((size_t)2 * p->sms * T * p->down_tile * 4, 256);
  p->counter_bytes = round_up((size_t)(H / 8) * 4, 256);
  return true;
}

template <int MAX, auto* Kernel, typename... Maps>
cudaError_t launch_ring(FewArgs a, int tile, size_t row_bytes, size_t sums, int sms, cudaStream_t st, const Maps&... maps) {
  const size_t smem = ring_room(sizeof(Shared<MAX>));
  a.tile = tile;
  // A second buffer for the sums saves a barrier at the end of every piece and costs half a stage.  Up to 16 tokens and pieces of at
  // most 8 steps gain (31 tokens of 128 experts, 512 / 1024: 98.5 -> 91.5 us; 16 tokens of 8, 4096 / 14336: 421 -> 411), long pieces
  // with more tokens lose (64 tokens: 468 -> 512).
  a.red = MAX == 16 || row_bytes <= 8 * kChunk ? 2 * kRedBytes : kRedBytes;
  a.room = (int)(smem - 1024 /*alignment*/ - a.red - sums);
  const cudaError_t e = allow_smem_once<Kernel>(sizeof(Shared<MAX>));
  return e != cudaSuccess ? e : launch_dependent(Kernel, dim3(sms), dim3(kThreads), smem, st, maps..., a);
}

template <int MAX>
cudaError_t few_launch(FewArgs a, const FewPlan& p, cudaStream_t st) {
  const CUtensorMapDataType bf16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const unsigned long long T = a.T, E = a.E, h_row = 2ull * a.I, x_row = 2ull * a.H, x_step = (unsigned long long)a.ldx;
  WeightMaps w13, w2, h;
  XMaps<MAX> x;
  if (!weight_maps(&w13, a.w13, 2ull * E * a.I, x_row, bf16, 2, heights_up_to(p.up_tile)) ||
      !weight_maps(&w2, a.w2, E * a.H, h_row, bf16, 2, p.down_tile | a.H % p.down_tile) ||
      !weight_maps(&h, a.h, T * a.top_k, h_row, bf16, 2, heights_up_to(box_rows(a.T))) ||
      !weight_maps(&x.box, a.x, T, x_row, bf16, 2, box_rows(a.T), x_step) || (MAX > 16 && !gather_map(&x.rows, a.x, T, x_row, x_step, bf16, 2)))
    return cudaErrorUnknown;
  a.whole = p.whole;
  const cudaError_t e = launch_ring<MAX, moe_few_up_kernel<MAX>>(a, p.up_tile, x_row, 0, p.sms, st, w13, x);
  return e != cudaSuccess ? e : launch_ring<MAX, moe_few_down_kernel<MAX>>(a, p.down_tile, h_row, MAX > 16 ? (size_t)MAX * kMaxTile * 4 : 0, p.sms, st, w2, h);
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
  if (T <= 16) return (int)few_launch<16>(a, p, st);
  if (T <= 32) return (int)few_launch<32>(a, p, st);
  return (int)few_launch<64>(a, p, st);
}
