// Matrix products of a few rows (1 to 64) with large weights, bound by reading the weights once: the parts that the
// few-token MoE layer (bf16) and the 8-bit integer linear share.
//
//   D[row][n] = sum_k A[row][k] W[n][k]
//
// A CTA streams pieces of W through a ring in shared memory.  One producer warp fetches, for `nr` weight rows (a multiple
// of 8, at most 64) and a chunk of 512 bytes along K, four columns of 128 bytes with TMA, all four in one box of 64, 32, 16
// or 8 rows (K beyond the end reads as zero).  Each of eight consumer warps takes a column and half of the weight rows; the
// sums of the four columns are added when the K range of a piece is done.  The rows of A come through the ring too, fetched
// by a second producer warp, in one box where they lie one behind the other and four at a time where they do not: under load
// L2 takes longer than a stage, and registers do not reach far enough ahead.
//
// Weight rows are the M (16) of mma.sync and rows of A its N (8).  On this GPU mma.sync is slow, a 16 x 8 x 16 product in some 32
// cycles of a quarter of an SM: with the rows of A as M (and weights as N) up to 16 rows took as many products as 16, and 32
// tokens of 8 experts were bound by them.  (tcgen05 is not, but its M are tiles of 64 or more weight rows: for one token and two
// of 64 experts that is 44 tiles of 128 rows for 148 SMs.  Here a CTA's share of the weights can be cut at any multiple of 8
// rows.)  The order of K is free as long as A and W agree: lane t of a row has bytes 32 t to 32 t + 31 of its column, in two
// halves of 16 consecutive bytes, each of which feeds two multiplications, so every operand is one 16-byte load.  Half s of
// all rows lies in the 16-byte units 2 t + s, which the 128-byte swizzle (unit ^ row % 8) puts into different banks for the
// two rows that a quarter of a warp reads at a time.
//
// One bulk copy per weight row and chunk in place of the boxes reached a quarter of the bandwidth: 401 us against 115 for one
// token of a layer that reads 704 MB.
#pragma once
#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "kernels/sm100_ptx.cuh"
#include "rbv/moe.h"

namespace rbv {
namespace few {

constexpr int kChunk = 512;               // bytes of a row per stage
constexpr int kCols = 4;                  // columns of 128 bytes in it
constexpr int kWarps = 2 * kCols;         // consumer warps
constexpr int kThreads = (kWarps + 2) * 32;         // and two producers, one for the weights and one for the rows of A
constexpr int kMaxRows = RBV_FEW_ROWS;    // rows of A
constexpr int kMaxTile = 64;              // weight rows of a piece
constexpr int kMaxStages = 32;

// Boxes of 8, 16, 32 and 64 rows: `all` of four columns (the row seen as columns of 128 bytes, as many as it has whole ones),
// `one` of a single column.
struct WeightMaps {
  CUtensorMap all[4], one[4];
  int heights;                             // 8, 16, 32, 64 in the bits of a mask: the boxes there are
  int whole;                               // chunks that `all` covers; the rest of a row that does not end with a column: `one`
};

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void part_sync(int part) { asm volatile("bar.sync %0, 128;" ::"r"(2 + part) : "memory"); }

// bf16 x bf16 -> fp32 (K 16) and s8 x s8 -> s32 (K 32): the same bytes per register.
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct Ring {
  uint64_t full[kMaxStages], empty[kMaxStages];
  int abort;
};

__device__ __forceinline__ void ring_init(Ring& ring, int stages, int producers) {      // one thread
  for (int s = 0; s < stages; s++) { sm100::mbar_init(&ring.full[s], producers); sm100::mbar_init(&ring.empty[s], kWarps); }
  ring.abort = 0;
  sm100::mbar_fence_init();
}

// The same for all stages there may be, by the first threads of a CTA that learns later how many fit.
__device__ __forceinline__ void ring_init_all(Ring& ring, int producers) {
  const int s = threadIdx.x;
  if (s >= kMaxStages) return;
  sm100::mbar_init(&ring.full[s], producers);
  sm100::mbar_init(&ring.empty[s], kWarps);
  if (s == 0) ring.abort = 0;
  sm100::mbar_fence_init();
}

// A warp's place in the ring, as addresses in shared memory: a warp that works alone pays for every instruction between two
// loads or multiplications, a stage of a small piece with as many cycles as its bytes take.
struct Cursor {
  uint32_t full, empty, slot;             // barriers and start of the current stage
  uint32_t phase = 0;
  int left, stages;                        // stages until the ring begins again
  uint32_t slot_bytes;
  Ring* ring;
  bool ok = true;
  __device__ __forceinline__ Cursor(Ring& r, uint32_t slots, int n, uint32_t bytes)
      : full(sm100::smem_u32(r.full)), empty(sm100::smem_u32(r.empty)), slot(slots), left(n), stages(n), slot_bytes(bytes), ring(&r) {}
  __device__ __forceinline__ void next() {
    full += 8; empty += 8; slot += slot_bytes;
    if (--left == 0) {
      left = stages;
      full -= 8u * stages; empty -= 8u * stages; slot -= slot_bytes * stages;
      phase ^= 1u;
    }
  }
  __device__ __forceinline__ static bool try_wait(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred P;\n\tmbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2;\n\tselp.b32 %0, 1, 0, P;\n\t}"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
  }
  // Bounded; once a wait of this CTA has run out, nobody waits any more (results are garbage, and reported).
  __device__ __forceinline__ void wait(uint32_t bar, uint32_t parity) {
    if (try_wait(bar, parity) || !ok) return;
    volatile int* abort = &ring->abort;
    for (uint32_t i = 0; i < (1u << 24); i++) {
      if (try_wait(bar, parity)) return;
      if ((i & 1023u) == 1023u && *abort) break;
    }
    ok = false;
    *abort = 1;
  }
  __device__ __forceinline__ void wait_full() { wait(full, phase); }
  __device__ __forceinline__ void wait_empty() { wait(empty, phase ^ 1u); }
  __device__ __forceinline__ void release() {          // one lane per consumer warp
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(empty) : "memory");
  }
};

// Shared memory of a CTA: the buffer, or two, in which warps add their sums, then the stages, 1024-byte aligned.
constexpr uint32_t kRedBytes = 2 * 4 * kCols * 32 * 16;       // four tiles at a time per part
// A stage: `tile` weight rows and `rows` of A.
__host__ __device__ inline uint32_t slot_bytes(int tile, int rows) { return (uint32_t)(tile + rows) * kChunk; }
// Rows of the box that holds r rows of A.
__host__ __device__ inline int box_rows(int r) { return r <= 8 ? 8 : r <= 16 ? 16 : r <= 32 ? 32 : 64; }

__device__ __forceinline__ void expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* m, int row, int column, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(dst), "l"(m), "r"(bar), "r"(0), "r"(row), "r"(column) : "memory");
}
__device__ __forceinline__ void load_column(uint32_t dst, const CUtensorMap* m, int x, int row, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(m), "r"(bar), "r"(x), "r"(row) : "memory");
}

// Fetches chunks c0 to c1 - 1 of `rows` rows (a multiple of 8) from `row0` on, one per stage, `off` bytes into it: box by box, in
// a box column by column.  Four lanes of a warp (others may come along), one for each height of a box: a lane gets a box on its way in 150 cycles or
// more whatever its size, so there is one box per height and stage (with a box per column the producer set the pace, 205 us
// against 119 for one token of a layer that reads 704 MB).  False: a wait ran out, stop.
template <typename E>                      // element: its size turns bytes along K into coordinates
__device__ __forceinline__ bool feed(const WeightMaps& maps, Cursor& cur, uint32_t off, int row0, int rows, int c0, int c1) {
  const int lane = threadIdx.x & 31, size = min(lane, 3), height = 8 << size;
  const bool mine = lane < 4 && (rows & height) != 0;
  const int before = rows & ~(2 * height - 1);           // rows in larger boxes
  const uint32_t bytes = (uint32_t)rows * kChunk, to = off + (uint32_t)before * kChunk;
  const CUtensorMap *all = &maps.all[size], *one = &maps.one[size];
  int c = c0;
  #pragma unroll 1
  for (; c < c1 && c < maps.whole; c++) {
    cur.wait_empty();
    if (!cur.ok) return false;
    if (lane == 0) expect(cur.full, bytes);
    if (mine) load_box(cur.slot + to, all, row0 + before, c * kCols, cur.full);
    cur.next();
  }
  #pragma unroll 1
  for (; c < c1; c++) {
    cur.wait_empty();
    if (!cur.ok) return false;
    if (lane == 0) expect(cur.full, bytes);
    if (mine)
      #pragma unroll 1
      for (int j = 0; j < kCols; j++)
        load_column(cur.slot + to + (uint32_t)(j * 128 * height), one, (c * kChunk + j * 128) / (int)sizeof(E), row0 + before, cur.full);
    cur.next();
  }
  return true;
}

// The same for rows of A that lie anywhere in a matrix: `rows` of them, row i at at(i), into a box of box_rows(rows).  A whole warp;
// an instruction fetches 128 bytes of four rows (`map`: boxes of one row).
template <typename E, typename At>
__device__ __forceinline__ bool feed_gathered(const CUtensorMap* map, Cursor& cur, uint32_t off, int rows, int c0, int c1, At&& at) {
  const int lane = threadIdx.x & 31, fours = (rows + 3) / 4, items = fours * kCols;
  const uint32_t col_bytes = (uint32_t)box_rows(rows) * 128u;
  int row[2][4], x[2];
  uint32_t to[2];
  #pragma unroll
  for (int k = 0; k < 2; k++) {            // (kMaxRows / 4 * kCols = 64 of them at most)
    const int item = lane + 32 * k, col = item & 3, q = item >> 2;
    #pragma unroll
    for (int i = 0; i < 4; i++) row[k][i] = item < items ? at(min(4 * q + i, rows - 1)) : 0;
    x[k] = col * 128 / (int)sizeof(E);
    to[k] = off + (uint32_t)col * col_bytes + (uint32_t)q * 512u;
  }
  #pragma unroll 1
  for (int c = c0; c < c1; c++) {
    cur.wait_empty();
    if (!cur.ok) return false;
    if (lane == 0) expect(cur.full, (uint32_t)items * 512u);
    #pragma unroll
    for (int k = 0; k < 2; k++)
      if (lane + 32 * k < items)
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
                     ::"r"(cur.slot + to[k]), "l"(map), "r"(cur.full), "r"(x[k] + c * (kChunk / (int)sizeof(E))), "r"(row[k][0]), "r"(row[k][1]),
                       "r"(row[k][2]), "r"(row[k][3]) : "memory");
    cur.next();
  }
  return true;
}

__device__ __forceinline__ void prefetch_maps(const WeightMaps& maps) {      // a warp
  const int lane = threadIdx.x & 31;
  if (lane < 4 && maps.whole && (maps.heights & (8 << lane))) sm100::tma_prefetch_desc(&maps.all[lane]);
}

// Where in a stage of `rows` weight rows the 8 rows of group g are, column j.
__device__ __forceinline__ uint32_t group_offset(int rows, int g, int j) {
  int at = 0, n = 0;
  #pragma unroll
  for (int b = 3; b >= 0; b--) {
    if (g * 8 < at + n) break;             // (n: rows of the box that ends at `at + n`)
    at += n;
    n = rows & (8 << b);
  }
  return (uint32_t)(at * kChunk + j * n * 128 + (g * 8 - at) * 128);
}

// A warp's rows of A are NT tiles of 8, its weight rows up to two groups of 16.
constexpr int kGroups = kMaxTile / 32;
// The groups of 16 of `rows` weight rows that a part (0 or 1) takes.
struct Share {
  int first, count;                        // groups of 16
  __device__ __forceinline__ Share(int rows, int part) {
    const int all = (rows + 15) / 16, half = (all + 1) / 2;
    first = part ? half : 0;
    count = part ? all - half : half;
  }
};
// Where the halves of its groups are in a stage of `rows` weight rows, column j; negative: there is none.
struct Offsets {
  int at[kGroups][2];
  __device__ __forceinline__ Offsets(int rows, const Share& share, int j) {
    #pragma unroll
    for (int n = 0; n < kGroups; n++)
      #pragma unroll
      for (int h = 0; h < 2; h++) {
        const int g = 2 * (share.first + n) + h;
        at[n][h] = n < share.count && g * 8 < rows ? (int)group_offset(rows, g, j) : -1;
      }
  }
};

// A lane's part of the rows of A for one chunk: 32 bytes of row 8 i + lane / 4 of each tile i, zeros for rows that do not exist.
template <int NT>
struct Rows {
  uint4 v[NT][2];                          // tile, half of the 32 bytes
  // from a box of a stage; `at`: rows of it, negative for those that do not exist
  __device__ __forceinline__ void load(const int (&at)[NT], uint32_t box, int rows, int col, int lane) {
    const uint32_t base = box + (uint32_t)(col * rows * 128), t = (uint32_t)lane & 3;
    #pragma unroll
    for (int i = 0; i < NT; i++)
      #pragma unroll
      for (int s = 0; s < 2; s++) {
        v[i][s] = make_uint4(0u, 0u, 0u, 0u);
        if (at[i] >= 0) v[i][s] = lds16(base + (uint32_t)at[i] * 128u + (((2u * t + s) ^ ((uint32_t)at[i] & 7u)) << 4));
      }
  }
};

template <typename Acc, int NT>
__device__ __forceinline__ void clear(Acc (&acc)[kGroups][NT][4]) {
  #pragma unroll
  for (int n = 0; n < kGroups; n++)
    #pragma unroll
    for (int i = 0; i < NT; i++)
      #pragma unroll
      for (int k = 0; k < 4; k++) acc[n][i][k] = 0;
}

// One stage's part of a warp: G of its groups, at w + off.  Halves that do not exist are multiplied as zeros: without branches
// all loads are on their way before the first multiplication and the chains of different tiles overlap.
template <int G, int NT, typename Acc>
__device__ __forceinline__ void multiply(Acc (&acc)[kGroups][NT][4], uint32_t w, const Offsets& off, const Rows<NT>& a, int lane) {
  const uint32_t row = (uint32_t)lane >> 2, t = (uint32_t)lane & 3;
  const uint32_t wl = w + row * 128u;
  #pragma unroll
  for (int s = 0; s < 2; s++) {
    uint4 b[G][2];
    #pragma unroll
    for (int n = 0; n < G; n++)
      #pragma unroll
      for (int h = 0; h < 2; h++) {
        b[n][h] = make_uint4(0u, 0u, 0u, 0u);
        if (off.at[n][h] >= 0) b[n][h] = lds16(wl + (uint32_t)off.at[n][h] + (((2u * t + s) ^ row) << 4));
      }
    #pragma unroll
    for (int half = 0; half < 2; half++)
      #pragma unroll
      for (int i = 0; i < NT; i++)
        #pragma unroll
        for (int n = 0; n < G; n++) {
          if (half == 0) mma(acc[n][i], b[n][0].x, b[n][1].x, b[n][0].y, b[n][1].y, a.v[i][s].x, a.v[i][s].y);
          else mma(acc[n][i], b[n][0].z, b[n][1].z, b[n][0].w, b[n][1].w, a.v[i][s].z, a.v[i][s].w);
        }
  }
}

// Adds the sums of a part's four columns and hands them out: put(row of A, weight row of the piece, sums of that weight row and
// the next one; even weight rows).  Four tiles of 16 x 8 at a time, one per warp.  The parts do not wait for one another.  With two
// buffers in turn, from call to call too, one barrier is enough: who writes into one has passed the barrier behind which everybody
// has left it.
struct Red { uint4* at; bool two; int turn = 0; };
template <int NT, typename Acc, typename Put>
__device__ __forceinline__ void add_columns(const Acc (&acc)[kGroups][NT][4], Red& red, const Share& share, int part, int col, int lane,
                                            Put&& put) {
  const int g = lane >> 2, t = lane & 3;
  const bool odd = (g & 1) != 0;
  const int tiles = share.count * NT;
  #pragma unroll
  for (int first = 0; first < kGroups * NT; first += 4) {
    if (first >= tiles) break;
    uint4* mine = red.at + (2 * red.turn + part) * (4 * kCols * 32);
    if (red.two) red.turn ^= 1;
    #pragma unroll
    for (int k = 0; k < 4; k++)            // (tile first + k: group / NT, tile of rows % NT)
      if (first + k < kGroups * NT)
        mine[(k * kCols + col) * 32 + lane] = *reinterpret_cast<const uint4*>(acc[(first + k) / NT][(first + k) % NT]);
    part_sync(part);
    const int tile = first + col;
    if (tile < tiles) {
      Acc v[4] = {0, 0, 0, 0};             // weight rows g, g and g + 8, g + 8; rows of A 2 t, 2 t + 1 and again
      #pragma unroll
      for (int j = 0; j < kCols; j++) {
        const uint4 u = mine[(col * kCols + j) * 32 + lane];
        v[0] += *reinterpret_cast<const Acc*>(&u.x);
        v[1] += *reinterpret_cast<const Acc*>(&u.y);
        v[2] += *reinterpret_cast<const Acc*>(&u.z);
        v[3] += *reinterpret_cast<const Acc*>(&u.w);
      }
      #pragma unroll
      for (int h = 0; h < 2; h++) {        // neighbouring weight rows are in lanes 4 apart: each lane gets both for one row of A
        const Acc got = __shfl_xor_sync(0xffffffffu, odd ? v[2 * h] : v[2 * h + 1], 4);
        put(8 * (tile % NT) + 2 * t + (odd ? 1 : 0), 16 * (share.first + tile / NT) + 8 * h + (g & ~1), odd ? got : v[2 * h], odd ? v[2 * h + 1] : got);
      }
    }
    if (!red.two) part_sync(part);
  }
}

// ---- work split along K over CTAs ------------------------------------------------------------------------------------
// `total` steps (tile by tile, each of `per_tile` steps along K) are cut into `parts` contiguous ranges of equal length, within
// one step, or within one tile where that costs less than to put tiles together again.  A tile whose steps lie in several
// ranges is finished by the last of their CTAs to arrive, which adds the others' sums in the order of the ranges: the result
// does not depend on who that is.  (total * parts fits 32 bits.)
struct Split {
  unsigned total, parts, grain;           // in units of `grain` steps, of which there are at least `parts`
  __device__ __forceinline__ unsigned begin(unsigned part) const { return part * total / parts * grain; }
  __device__ __forceinline__ unsigned owner(unsigned step) const { return ((step / grain + 1) * parts - 1) / total; }
};

// ---- host side -------------------------------------------------------------------------------------------------------
// Weight rows of a piece: an even share of `groups` groups of 8 among `parts`, at most 64 rows.
inline int tile_rows(long long groups, int parts) {
  const long long n = (groups + parts - 1) / parts;
  return (int)(n < 1 ? 8 : n > kMaxTile / 8 ? kMaxTile : n * 8);
}

// How `n` weight rows (or columns of the result) of row_bytes each, `experts` times, are cut for `rows` rows of A: rows of a
// piece, and whether pieces stay whole, by the nanoseconds that the CTA with most of the work takes.  Measured: a step of t
// weight rows takes as long as its 512 t bytes at an SM's share of the memory's rate (twice that where half the SMs have
// nothing to do), as its multiplications (2.8 ns per weight row and tile of 8 rows of A) or as its waits (0.25 us); the end
// of a piece 1.1 us, once per expert where every expert's sums are put away (`each`); putting a tile together that several
// CTAs share 3.2 us, and 0.2 us for every 512 sums of every one of them.  8-bit weights of 4096 columns, 3 rows of A, a call:
// 28672 weight rows in whole tiles of 64 / 32 / 8 26.5 / 29.6 / 62.5 us; 4096 in whole tiles of 64 / 32 / 8 8.1 / 7.9 / 13.4
// us, split among the SMs in 64 11.8 us.  A layer of 12 experts, 1024 / 2816: whole 50 us, split 36.5 us.
// False: too much for 32-bit step numbers.
inline bool split_plan(long long n, long long row_bytes, long long experts, int sms, int rows, int row_tiles, bool each, int* tile, int* whole) {
  const long long chunks = (row_bytes + kChunk - 1) / kChunk, steps = experts * chunks;
  double best = 1e300;
  for (int t = kMaxTile; t >= 8; t /= 2) {
    const long long tiles = (n + t - 1) / t, total = tiles * steps;
    for (int w = 1; w >= 0; w--) {
      const long long parts = w ? tiles : total, busy = parts < sms ? parts : sms;
      const long long most = w ? (tiles + sms - 1) / sms * steps : (total + busy - 1) / busy;       // steps of a CTA
      const double share = busy * 2 > sms ? (double)busy / sms : 0.5;
      const double step = std::max({11.6 * t * share, 2.8 * t * row_tiles, 209.0 + 35.0 * row_tiles});
      const double ends = each ? (double)most / chunks + 1 - w : (double)most / steps + 1 - w;
      const double join = w ? 0.0 : 3200.0 + 205.0 * ((steps + most - 1) / most + 1) * ((rows * t + 511) / 512);
      const double ns = most * step + ends * (1000.0 + 125.0 * row_tiles) + join;
      if (ns < best) { best = ns; *tile = t; *whole = w; }
    }
  }
  return (n + *tile - 1) / *tile * steps * sms <= 0xffffffffll;
}

// Dynamic shared memory that a CTA can have beside `fixed` bytes of static variables (which the compiler may round up).
inline size_t ring_room(size_t fixed) { return 227 * 1024 - (fixed + 511) / 256 * 256; }

// Stages that fit beside `other` bytes of dynamic shared memory.
inline int ring_stages(int tile, int rows, size_t fixed, size_t other) {
  const size_t room = ring_room(fixed) - 1024 /*alignment*/ - other, n = room / slot_bytes(tile, rows);
  return n > (size_t)kMaxStages ? kMaxStages : (int)n;
}
// Once per kernel and device: as much dynamic shared memory as there is beside `fixed` bytes.  (A call on one token takes less
// time on the GPU than a handful of runtime calls.)
template <auto* Kernel>
inline cudaError_t allow_smem_once(size_t fixed) {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1))) return e;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ring_room(fixed));
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return e;
}
inline size_t ring_smem(int tile, int rows, int stages) { return 1024 + (size_t)slot_bytes(tile, rows) * stages; }

typedef CUresult (*TensorMapEncoder)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                     const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                     CUtensorMapFloatOOBfill);
inline TensorMapEncoder tensor_map_encoder() {       // null: the driver has none
  static const TensorMapEncoder encode = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<TensorMapEncoder>(p) : nullptr;
  }();
  return encode;
}

// Boxes for pieces of at most `rows` rows, all multiples of 8 among them.
inline int heights_up_to(int rows) {
  int all = 0;
  for (int h = 8; h <= rows; h *= 2) all |= h;
  return all;
}

// Rows for feed_gathered: `rows` of `len` bytes, `row_bytes` apart (multiples of 16).
inline bool gather_map(CUtensorMap* m, const void* base, unsigned long long rows, unsigned long long len, unsigned long long row_bytes,
                       CUtensorMapDataType type, int size) {
  const cuuint64_t dims[2] = {len / size, rows}, strides[1] = {row_bytes};
  const cuuint32_t box[2] = {128u / (unsigned)size, 1}, ones[2] = {1, 1};
  return tensor_map_encoder() && tensor_map_encoder()(m, type, 2, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Weights of `rows` rows of row_bytes (a multiple of 16) each, `step` bytes apart, elements of `size` bytes; 128-byte swizzle.  Bits 3 to 6 of
// `heights`: the boxes that pieces are made of (a map takes a third of a microsecond to make).
inline bool weight_maps(WeightMaps* m, const void* base, unsigned long long rows, unsigned long long row_bytes, CUtensorMapDataType type,
                        int size, int heights, unsigned long long step = 0) {
  if (!step) step = row_bytes;
  const TensorMapEncoder encode = tensor_map_encoder();
  if (!encode) return false;
  const unsigned per_col = 128u / (unsigned)size;
  m->heights = heights;
  const cuuint64_t cols = row_bytes / 128;                 // whole columns
  const bool even = row_bytes % 128 == 0;
  m->whole = (int)(even ? (cols + kCols - 1) / kCols : cols / kCols);      // (columns behind the last one read as zeros)
  const cuuint64_t dims3[3] = {per_col, rows, cols}, strides3[2] = {step, 128};
  const cuuint64_t dims2[2] = {row_bytes / size, rows}, strides2[1] = {step};
  const cuuint32_t ones[3] = {1, 1, 1};
  for (int b = 0; b < 4; b++) {
    if (!(heights & (8 << b))) continue;
    const cuuint32_t box3[3] = {per_col, 8u << b, (cuuint32_t)kCols}, box2[2] = {per_col, 8u << b};
    if (m->whole > 0 && encode(&m->all[b], type, 3, const_cast<void*>(base), dims3, strides3, box3, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
    if (!even && encode(&m->one[b], type, 2, const_cast<void*>(base), dims2, strides2, box2, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
  }
  return true;
}

}  // namespace few
}  // namespace rbv
