// Decode attention over a paged cache whose sequences may share their first rows, on the
// 5th-generation tensor cores (tcgen05):
//
//   out[b, h] = sum_j softmax_j(scale q[b, h] . K_j) V_j   over the rows j < lens[b].
//
// The rows below `shared` are the same for every sequence that has them all: for one kv head
// they are one key / value matrix against the query rows of the whole batch, 128 query rows
// to a tile (prefix work).  Each sequence's rows from there on (all of a shorter sequence's)
// meet its own few query rows only (own work).  Both are the same computation on a tile of up
// to 128 query rows and a run of 128-key chunks, so one kernel does both, at once: the prefix
// part is bound by the tensor cores and the exponentials, the own part by memory, and they
// run on different SMs side by side.
//
// The work is a line of chunks, each with a cost, cut into one piece of equal cost per CTA
// (PagedLine): the cut is arithmetic on the lengths, made on the device, so a captured launch
// follows the lengths and results do not depend on scheduling.  A CTA writes the partial
// result (O, running maximum, sum) of every unit it meets; sink_paged_combine_kernel joins a
// row's partials.
//
// Inside a CTA two softmax warpgroups each own a stream of steps (a tile of scores S = Q K^T
// for one chunk, its probabilities P, and O += P V); step n is on stream n & 1.  With two query
// tiles (a pair) every chunk is a step on both streams, one per tile, and K and V are read from
// shared memory for 256 query rows; with one tile chunks alternate between the streams.  While
// one warpgroup takes exponentials the tensor cores work for the other.  A thread owns a query
// row (a TMEM lane): no reduction across threads.  P goes back to TMEM over its own scores,
// 16-bit, and is the MMA's A operand from there (one rounding to the cache's type: the tensor
// cores take 16-bit operands; the sum of probabilities is of the unrounded ones).  The reference maximum only moves when a score
// passes it by 2^8 (then O is rescaled in TMEM), so the usual chunk touches O in the MMA only.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "sink_chunk.cuh"
#include "sink_tcgen05.cuh"

namespace sinkb200 {

constexpr int kPgKeys = 128;      // keys per chunk
constexpr int kPgTile = 128;      // query rows per tile
constexpr int kPgThreads = 320;   // two softmax warpgroups, the MMA warp, the load warp
constexpr int kPgNarrow = 8;      // query rows of a tile up to which four warps share its keys
constexpr int kPgMmaWarp = 8, kPgLoadWarp = 9;
constexpr float kPgRescale = 8.f; // log2
constexpr int kPgP = 64;          // P's first column within its scores' 128
constexpr int kPgTmemCols = 512;  // S of the streams at 0 and 128, O at 256 and 384

template <int D>
struct PgGeom {
  static constexpr int kTileBytes = kPgKeys * D * 2;  // a K, V or Q tile: D / 64 boxes of 128 rows
  static constexpr int kBoxBytes = kPgKeys * 128;
  static constexpr int kRing = D == 128 ? 5 : 12;     // K and V tiles in flight
  static constexpr int kBarBytes = 1024;
  static constexpr int kSmem = 1024 + (2 + kRing) * kTileBytes + kBarBytes;
};

struct PagedArgs {
  CUtensorMap kmap, vmap;  // [pages, Hkv, page_size, D], box {64, page_size, 1, 1}
  CUtensorMap qtile;       // [B, Hq, D], box {64, G, 128 / G}: a tile's query rows
  CUtensorMap qgroup;      // box {64, G, 1}: one sequence's
  const int32_t* table;
  const int32_t* lens;
  int* status;
  char* out;
  int64_t table_sb, o_sb, o_sh;
  float* o_prefix;   // [prefix slots][2][128][D]
  float2* ml_prefix; // [prefix slots][2][128] (maximum, sum)
  float* o_own;      // [own slots][2][G][D]
  float2* ml_own;
  int* offsets;      // [B] chunks of the sequences before, [B]: of all, [B + 1]: prefix in use
  int batch, heads_kv, group, page_size, pages, table_width, shared;
  int per_tile, tiles;  // sequences per query tile, tiles per kv head
  int ctas;
  float scale_log2;  // of |scale|
  uint32_t negate;   // scale < 0: the MMA negates Q
};

// ------------------------------------------------------------------ the line of work

// Costs of a chunk in clocks of one SM, by measurement: one tile or a pair of tiles on it, and
// an own chunk, at least kOwnMin and, where memory bounds the own work, its share of the time
// that memory takes for all of it (kOwnMem when every SM streams).
template <int D>
struct PgCost {
  static constexpr int kPair = D == 128 ? 2400 : 2200;
  static constexpr int kOne = D == 128 ? 1400 : 1200;
  static constexpr int kOwnMin = D == 128 ? 1400 : 1200;
  static constexpr int kOwnMem = D == 128 ? 2750 : 1375;
};

struct PagedLine {
  int chunks;            // prefix chunks (0: nothing shared, or no sequence that has it all)
  int units;             // prefix units: kv heads x groups of up to two tiles
  int groups, pairs;     // groups per head, the first `pairs` of them of two tiles
  int own_cost;
  long long head_cost;   // prefix cost of one head
  long long prefix_cost, total;
};

template <int D>
__device__ __forceinline__ PagedLine paged_line(const PagedArgs& A, int own_chunks, bool prefix) {
  PagedLine L;
  L.chunks = prefix ? (A.shared + kPgKeys - 1) / kPgKeys : 0;
  L.pairs = A.tiles / 2;
  L.groups = (A.tiles + 1) / 2;
  L.units = L.chunks > 0 ? A.heads_kv * L.groups : 0;
  L.head_cost = (long long)L.chunks * (L.pairs * PgCost<D>::kPair + (L.groups - L.pairs) * PgCost<D>::kOne);
  L.prefix_cost = L.units > 0 ? L.head_cost * A.heads_kv : 0;
  const long long own = (long long)own_chunks * A.heads_kv;
  long long c = PgCost<D>::kOwnMem - (own > 0 ? L.prefix_cost / own : 0);
  L.own_cost = int(c < PgCost<D>::kOwnMin ? PgCost<D>::kOwnMin : c);
  L.total = L.prefix_cost + own * L.own_cost;
  return L;
}

__device__ __forceinline__ long long paged_cut(const PagedLine& L, int ctas, int c) { return L.total * c / ctas; }

// The CTA whose piece holds position x of the line (x < total).
__device__ __forceinline__ int paged_cta_of(const PagedLine& L, int ctas, long long x) {
  int c = int(x * ctas / L.total);
  while (c > 0 && paged_cut(L, ctas, c) > x) --c;
  while (c + 1 < ctas && paged_cut(L, ctas, c + 1) <= x) ++c;
  return c;
}

__device__ __forceinline__ int paged_len(const PagedArgs& A, int b) {
  const int n = A.lens[b];
  return imax(0, imin(n, A.table_width * A.page_size));
}
// First row of a sequence's own work, and its chunks.
__device__ __forceinline__ int paged_own_row(const PagedArgs& A, int len) { return len >= A.shared ? A.shared : 0; }
__device__ __forceinline__ int paged_own_chunks(const PagedArgs& A, int len) {
  return (len - paged_own_row(A, len) + kPgKeys - 1) / kPgKeys;
}

// Chunks [j0, j1) of the unit at `base` of n chunks of cost w that lie in [lo, hi).
__device__ __forceinline__ void paged_span(long long lo, long long hi, long long base, int n, int w, int& j0, int& j1) {
  const long long a = lo <= base ? 0 : (lo - base + w - 1) / w;
  const long long e = hi <= base ? 0 : (hi - base + w - 1) / w;
  j0 = int(a < n ? a : n);
  j1 = int(e < n ? e : n);
}

struct PagedPiece {
  int unit;    // of the prefix, or b * heads_kv + h
  int h;
  int which;   // prefix: first tile; own: the sequence
  int j0, j1;  // chunks
  int len;     // own: the sequence's length
  bool own, pair;
};

// Walks the pieces of one CTA in line order.  Every role of the CTA runs its own copy.
struct PagedWalk {
  long long lo, hi, base;
  int unit, h, at, len;  // at: group of the head, or sequence
  bool own;

  __device__ __forceinline__ bool next(const PagedArgs& A, const PagedLine& L, PagedPiece& p) {
    while (base < hi) {
      int n, w;
      if (!own) {
        if (unit >= L.units) {
          own = true;
          unit = h = at = 0;
          len = -1;
          continue;
        }
        p.which = 2 * at;
        p.pair = at < L.pairs;
        n = L.chunks;
        // cost of the unit's chunks
        w = p.pair ? cost_pair : cost_one;
      } else {
        if (at >= A.batch) return false;
        if (len < 0) len = paged_len(A, at);
        n = paged_own_chunks(A, len);
        w = L.own_cost;
        p.which = at;
        p.pair = false;
      }
      p.unit = unit;
      p.h = h;
      p.own = own;
      p.len = len;
      if (own && n == 0) {
        unit += A.heads_kv - h;
        h = 0;
        ++at;
        len = -1;
        continue;
      }
      paged_span(lo, hi, base, n, w, p.j0, p.j1);
      base += (long long)n * w;
      ++unit;
      if (own) {
        if (++h == A.heads_kv) {
          h = 0;
          ++at;
          len = -1;
        }
      } else if (++at == L.groups) {
        at = 0;
        ++h;
      }
      if (p.j0 < p.j1) return true;
    }
    return false;
  }
  int cost_pair, cost_one;
};

// ------------------------------------------------------------------ helpers

__host__ __device__ constexpr uint32_t pg_idesc(uint32_t fmt, int n, bool b_mn_major) {
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (uint32_t(b_mn_major) << 16) | (uint32_t(n >> 3) << 17) |
         (uint32_t(kPgTile >> 4) << 24);
}
constexpr uint32_t kPgNegateA = 1u << 13;

__device__ __forceinline__ float pg_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A bounded wait whose answer the whole warp shares.
__device__ __forceinline__ bool pg_warp_wait(uint32_t bar, uint32_t parity) {
  return __all_sync(kFull, mbar_wait_bounded(bar, parity));
}

template <typename T>
__device__ __forceinline__ uint32_t pg_pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pg_pack<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pg_pack<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// exp2 arithmetic two elements at a time.
__device__ __forceinline__ uint64_t pg_pair(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ uint64_t pg_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t pg_add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ float2 pg_two(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}

// 32 scores of a query row (fp32 bits), keys from `limit` on left out: -infinity.
__device__ __forceinline__ void pg_mask(uint32_t (&r)[32], int limit) {
  if (limit < 32) {
#pragma unroll
    for (int x = 0; x < 32; ++x)
      if (x >= limit) r[x] = __float_as_uint(kNegInf);
  }
}

__device__ __forceinline__ float pg_max(const uint32_t (&r)[32], float mx) {
#pragma unroll
  for (int x = 0; x < 32; ++x) mx = fmaxf(mx, __uint_as_float(r[x]));
  return mx;
}

// Moves the row's reference maximum up to `mx` (log2 units) when that passes it by kPgRescale:
// the sum and, if `has_o`, the row's O in TMEM are rescaled.  Rows that are no query (`valid`
// false) compute along.
template <int D>
__device__ __forceinline__ void pg_reference(float mx, bool valid, bool has_o, uint32_t t_o, float& mref, float& l) {
  const bool need = valid && mx > mref + kPgRescale;
  if (!__any_sync(kFull, need)) return;
  float alpha = 1.f;
  if (need) {
    alpha = pg_exp2(mref - mx);
    mref = mx;
    l *= alpha;
  }
  if (has_o) {  // (the last MMA on it is complete)
#pragma unroll 1
    for (int x = 0; x < D; x += 32) {
      uint32_t o[32];
      tc_ld32(t_o + x, o);
      tc_wait_ld();
#pragma unroll
      for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * alpha);
      tc_st32(t_o + x, o);
    }
  }
}

// Probabilities 2^(scale s - m) of 32 scores, their sum added to `sum` (two accumulators),
// rounded to T and packed.
template <typename T>
__device__ __forceinline__ void pg_probs(const uint32_t (&r)[32], uint64_t scale2, uint64_t m2, uint64_t (&sum)[2],
                                         uint32_t (&pk)[16]) {
#pragma unroll
  for (int x = 0; x < 16; ++x) {
    const float2 e = pg_two(pg_fma2(pg_pair(__uint_as_float(r[2 * x]), __uint_as_float(r[2 * x + 1])), scale2, m2));
    const float p0 = pg_exp2(e.x), p1 = pg_exp2(e.y);
    sum[x & 1] = pg_add2(sum[x & 1], pg_pair(p0, p1));
    pk[x] = pg_pack<T>(p0, p1);
  }
}

// ------------------------------------------------------------------ kernel

template <typename T, int D>
__global__ void __launch_bounds__(kPgThreads, 1) sink_paged_kernel(const __grid_constant__ PagedArgs A) {
  using G_ = PgGeom<D>;
  constexpr int kRing = G_::kRing, kTB = G_::kTileBytes, kBox = G_::kBoxBytes, kBoxes = D / 64;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;  // swizzled tiles want 1024-byte alignment
  unsigned char* gbase = smem_raw + (base - raw);
  const uint32_t s_q = base, s_ring = base + 2 * kTB, s_bar = s_ring + kRing * kTB;
  const uint32_t b_full = s_bar, b_empty = b_full + 8 * kRing, b_qfull = b_empty + 8 * kRing, b_qempty = b_qfull + 16;
  const uint32_t b_s = b_qempty + 16, b_p = b_s + 16, b_o = b_p + 16, b_wg = b_o + 16, b_merge = b_wg + 16, b_done = b_merge + 32;
  unsigned char* g_bar = gbase + (s_bar - base);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(g_bar + 336);
  int* flag = reinterpret_cast<int*>(g_bar + 340);
  int* scan = reinterpret_cast<int*>(g_bar + 344);          // [12] warp sums
  int* start = reinterpret_cast<int*>(g_bar + 392);         // first own sequence, chunks before it
  int* any = reinterpret_cast<int*>(g_bar + 400);
  float2* g_ml = reinterpret_cast<float2*>(g_bar + 512);    // [2 streams][4 warps][8 rows] of narrow tiles
  static_assert(2 * 8 * kRing + 16 * 8 + 8 <= 336 && 512 + 2 * 4 * kPgNarrow * 8 <= G_::kBarBytes, "barriers");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(b_full + 8 * i, 1);
      mbar_init(b_empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(b_qfull + 8 * i, 1);
      mbar_init(b_qempty + 8 * i, 1);
      mbar_init(b_merge + 8 * i, 1);
      mbar_init(b_merge + 16 + 8 * i, 1);
      mbar_init(b_s + 8 * i, 1);
      mbar_init(b_p + 8 * i, 128);
      mbar_init(b_o + 8 * i, 1);
      mbar_init(b_wg + 8 * i, 128);
    }
    mbar_init(b_done, 1);
    *flag = 0;
    *any = 0;
    start[0] = A.batch;
    start[1] = 0;
    fence_mbar_init();
  }
  __syncwarp();
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "n"(kPgTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  grid_dependency_wait();  // lengths, table, query and cache rows are written
  __syncthreads();

  // ---- the line: own chunks before each thread's run of sequences
  const int per = (A.batch + kPgThreads - 1) / kPgThreads;
  const int b_lo = imin(tid * per, A.batch), b_hi = imin(b_lo + per, A.batch);
  int mine = 0;
  bool full = false;
  for (int b = b_lo; b < b_hi; ++b) {
    const int n = paged_len(A, b);
    mine += paged_own_chunks(A, n);
    full |= n >= A.shared;
    if (blockIdx.x == 0 && A.lens[b] > A.table_width * A.page_size) atomicOr(A.status, 2);
  }
  if (full && A.shared > 0) *any = 1;
  int before = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int x = __shfl_up_sync(kFull, before, off);
    if (lane >= off) before += x;
  }
  if (lane == 31) scan[warp] = before;
  __syncthreads();
  int own_chunks = 0;
#pragma unroll
  for (int w = 0; w < kPgThreads / 32; ++w) {
    if (w < warp) before += scan[w];
    own_chunks += scan[w];
  }
  before -= mine;
  const PagedLine L = paged_line<D>(A, own_chunks, *any != 0);
  PagedWalk walk0;
  walk0.lo = paged_cut(L, A.ctas, int(blockIdx.x));
  walk0.hi = paged_cut(L, A.ctas, int(blockIdx.x) + 1);
  walk0.cost_pair = PgCost<D>::kPair;
  walk0.cost_one = PgCost<D>::kOne;
  const long long own_unit = (long long)L.own_cost * A.heads_kv;
  {
    int c = before;
    const long long want = walk0.lo - L.prefix_cost;  // the first sequence whose work reaches past lo
    for (int b = b_lo; b < b_hi; ++b) {
      const int n = paged_own_chunks(A, paged_len(A, b));
      if (blockIdx.x == 0) A.offsets[b] = c;
      if (n > 0 && want >= own_unit * c && want < own_unit * (c + n)) {
        start[0] = b;
        start[1] = c;
      }
      c += n;
    }
    if (blockIdx.x == 0 && tid == 0) {
      A.offsets[A.batch] = own_chunks;
      A.offsets[A.batch + 1] = L.chunks > 0;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (walk0.lo < L.prefix_cost) {
    walk0.own = false;
    walk0.len = 0;
    walk0.h = int(walk0.lo / L.head_cost);
    const long long r = walk0.lo - walk0.h * L.head_cost;
    const long long pair_cost = (long long)L.chunks * PgCost<D>::kPair;
    walk0.at = imin(int(r / pair_cost), L.pairs);
    if (walk0.at >= L.groups) walk0.at = L.groups - 1;
    walk0.unit = walk0.h * L.groups + walk0.at;
    walk0.base = walk0.h * L.head_cost + walk0.at * pair_cost;
  } else {
    walk0.own = true;
    walk0.at = start[0];
    walk0.base = L.prefix_cost + own_unit * start[1];
    walk0.len = -1;
    walk0.h = 0;
    if (walk0.at < A.batch) {
      walk0.len = paged_len(A, walk0.at);
      const long long unit_cost = (long long)L.own_cost * paged_own_chunks(A, walk0.len);
      walk0.h = int((walk0.lo - walk0.base) / unit_cost);
      walk0.base += walk0.h * unit_cost;
    }
    walk0.unit = walk0.at * A.heads_kv + walk0.h;
  }

  bool failed = false;
  PagedWalk walk = walk0;
  PagedPiece pc;
  const bool narrow_prefix = A.tiles == 1 && A.batch * A.group <= kPgNarrow;
  if (warp == kPgLoadWarp) {
    // ================================================================ loads (the warp's lanes share a tile's pages)
    const int npg = kPgKeys / A.page_size;
    const int qrow_bytes = A.group * 128 * kBoxes;
    int tile = 0, qseq = 0, step = 0;  // ring tiles, Q tiles and steps issued
    // Per stream s and Q slot, at bit 2 s + slot: whether s merges in the slot's present tile
    // (then the slot is free only after b_merge), and, 4 bits up, that barrier's parity.
    uint32_t merges = 0;
    auto ring_slot = [&](int i) -> bool {  // waits until tile i's slot is free
      return i < kRing || pg_warp_wait(b_empty + 8 * (i % kRing), ((i / kRing) - 1) & 1);
    };
    while (!failed && walk.next(A, L, pc)) {
      const int nq = pc.pair ? 2 : 1;
      for (int s = 0; s < nq && !failed; ++s, ++qseq) {
        const int slot = qseq & 1;
        if (qseq >= 2 && !pg_warp_wait(b_qempty + 8 * slot, ((qseq >> 1) - 1) & 1)) {
          failed = true;
          break;
        }
        for (int x = slot; x < 4; x += 2) {
          if (!((merges >> x) & 1u)) continue;
          if (!pg_warp_wait(b_merge + 8 * x, (merges >> (4 + x)) & 1u)) failed = true;
          merges ^= 0x11u << x;
        }
        if (failed) break;
        if (pc.own || narrow_prefix) {
          const int n = pc.j1 - pc.j0;
          merges |= 1u << (2 * (step & 1) + slot);            // the stream of the first chunk
          if (n > 1) merges |= 1u << (2 * (~step & 1) + slot);
        }
        if (lane == 0) {
          const uint32_t bar = b_qfull + 8 * slot, dst = s_q + slot * kTB;
          // a narrow tile's rows once for each warp of the warpgroup, 32 TMEM lanes apart
          const int copies = pc.own || narrow_prefix ? 4 : 1;
          const CUtensorMap* map = pc.own ? &A.qgroup : &A.qtile;
          const int seq = pc.own ? pc.which : (pc.which + s) * A.per_tile;
          mbar_arrive_expect_tx(bar, (pc.own ? qrow_bytes : qrow_bytes * A.per_tile) * copies);
          for (int x = 0; x < kBoxes; ++x)
            for (int c = 0; c < copies; ++c)
              tma_load_3d(dst + x * kBox + c * 32 * 128, map, 64 * x, pc.h * A.group, seq, bar);
        }
      }
      step += (pc.j1 - pc.j0) * nq;
      // rows [row0, end) of the sequence (of the shared part) through one row of the table
      const int row0 = pc.own ? paged_own_row(A, pc.len) : 0;
      const int end = pc.own ? pc.len : A.shared;
      const int32_t* trow = A.table + (pc.own && row0 == A.shared ? pc.which * A.table_sb : 0);
      auto page_of = [&](int j) -> int {  // this lane's page of chunk j; A.pages reads as zeros
        const int row = row0 + j * kPgKeys + lane * A.page_size;
        if (lane >= npg || j >= pc.j1 || row >= end) return A.pages;
        const int p = trow[row / A.page_size];
        if (p >= 0 && p < A.pages) return p;
        atomicOr(A.status, 2);
        return A.pages;
      };
      int page = page_of(pc.j0);
      for (int j = pc.j0; j < pc.j1 && !failed; ++j) {
        const int next_page = page_of(j + 1);
        for (int v = 0; v < 2; ++v, ++tile) {
          if (!ring_slot(tile)) {
            failed = true;
            break;
          }
          const uint32_t bar = b_full + 8 * (tile % kRing), dst = s_ring + (tile % kRing) * kTB;
          if (lane == 0) mbar_arrive_expect_tx(bar, kTB);
          __syncwarp();
          if (lane < npg) {
            const CUtensorMap* map = v ? &A.vmap : &A.kmap;
            for (int x = 0; x < kBoxes; ++x)
              tma_load_4d(dst + x * kBox + lane * A.page_size * 128, map, 64 * x, 0, pc.h, page, bar);
          }
        }
        page = next_page;
      }
    }
    if (failed) {  // let the copies in flight land before the CTA can exit (bounded waits)
      for (int i = tile - 1; i >= 0 && i >= tile - kRing; --i)
        pg_warp_wait(b_full + 8 * (i % kRing), (i / kRing) & 1);
      for (int i = qseq - 1; i >= 0 && i >= qseq - 2; --i) pg_warp_wait(b_qfull + 8 * (i & 1), (i >> 1) & 1);
    }
  } else if (warp == kPgMmaWarp) {
    // ================================================================ MMA issue (one lane)
    if (lane == 0) {
      constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      const uint32_t idesc_s = pg_idesc(kFmt, kPgKeys, false) | (A.negate ? kPgNegateA : 0u);
      constexpr uint32_t idesc_o = pg_idesc(kFmt, D, true);
      // A cursor over the steps: chunk j of a piece, sub-step t of its tiles
      struct Cursor {
        PagedWalk walk;
        PagedPiece pc;
        int j, t, chunk, step, q0;  // chunk: chunks before it; q0: Q tiles before this piece
        bool live;
      };
      auto open = [&](Cursor& c) {
        c.live = c.walk.next(A, L, c.pc);
        c.j = c.pc.j0;
        c.t = 0;
      };
      auto advance = [&](Cursor& c) {
        ++c.step;
        if (c.pc.pair && c.t == 0) {
          c.t = 1;
          return;
        }
        c.t = 0;
        ++c.chunk;
        if (++c.j == c.pc.j1) {
          c.q0 += c.pc.pair ? 2 : 1;
          open(c);
        }
      };
      Cursor a;
      a.walk = walk;
      a.chunk = a.step = a.q0 = 0;
      open(a);
      Cursor b = a;
      auto qk = [&](Cursor& c) -> bool {
        const int s = c.step & 1, q = c.q0 + c.t;
        const int i = 2 * c.chunk;
        if (c.j == c.pc.j0 && !mbar_wait_bounded(b_qfull + 8 * (q & 1), (q >> 1) & 1)) return false;
        if (!mbar_wait_bounded(b_full + 8 * (i % kRing), (i / kRing) & 1)) return false;
        tc_fence_after();
        const uint32_t kb = s_ring + (i % kRing) * kTB, qb = s_q + (q & 1) * kTB;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * kBox + (kk & 3) * 32;
          tc_mma(tmem + s * kPgKeys, tc_desc(qb + off, 16), tc_desc(kb + off, 16), idesc_s, kk > 0);
        }
        tc_commit(b_s + 8 * s);
        if (!c.pc.pair || c.t == 1) tc_commit(b_empty + 8 * (i % kRing));
        if (c.j + 1 == c.pc.j1) tc_commit(b_qempty + 8 * (q & 1));
        return true;
      };
      auto pv = [&](Cursor& c) -> bool {
        const int s = c.step & 1, i = 2 * c.chunk + 1;
        if (!mbar_wait_bounded(b_p + 8 * s, (c.step >> 1) & 1)) return false;
        if (!mbar_wait_bounded(b_full + 8 * (i % kRing), (i / kRing) & 1)) return false;
        tc_fence_after();
        const uint32_t vb = s_ring + (i % kRing) * kTB;
        const bool first = c.pc.pair ? c.j == c.pc.j0 : c.j - c.pc.j0 < 2;
#pragma unroll
        for (int kk = 0; kk < kPgKeys / 16; ++kk)
          tc_mma_ta(tmem + 256 + s * 128, tmem + s * kPgKeys + kPgP + kk * 8, tc_desc(vb + kk * 2048, kBox), idesc_o,
                    !(first && kk == 0));
        if (!c.pc.pair || c.t == 1) tc_commit(b_empty + 8 * (i % kRing));
        if (c.pc.pair ? c.j + 1 == c.pc.j1 : c.j + 2 >= c.pc.j1) tc_commit(b_o + 8 * s);
        return true;
      };
      for (int n = 0; n < 2 && a.live && !failed; ++n) {
        if (!qk(a)) failed = true;
        advance(a);
      }
      while (b.live && !failed) {
        if (!pv(b)) {
          failed = true;
          break;
        }
        advance(b);
        if (a.live) {
          if (!qk(a)) failed = true;
          advance(a);
        }
      }
      tc_commit(b_done);  // TMEM is freed only after every MMA has completed
      mbar_wait_bounded(b_done, 0);
    }
  } else {
    // ================================================================ softmax: warpgroup s, a thread per query row
    const int s = warp >> 2, row = tid & 127, wq = warp & 3;
    const uint32_t lanes = uint32_t(wq * 32) << 16;
    const uint32_t t_s = tmem + s * kPgKeys + lanes, t_o = tmem + 256 + s * 128 + lanes;
    int step = 0, chunk = 0, qseq = 0;  // steps, chunks and Q tiles before this piece
    int items = 0, syncs = 0;           // pieces this stream had steps of; barriers of the warpgroup
    auto wg_sync = [&]() -> bool {      // the warpgroup's threads, bounded
      mbar_arrive(b_wg + 8 * s);
      return pg_warp_wait(b_wg + 8 * s, (syncs++) & 1);
    };
    // whether prefix row r of tile `tile` belongs to a sequence that has the whole prefix
    auto takes_part = [&](int tile, int r) { return paged_len(A, tile * A.per_tile + r / A.group) >= A.shared; };
    while (!failed && walk.next(A, L, pc)) {
      const int n = pc.j1 - pc.j0;
      const int t = (step & 1) ^ s;  // the tile, or the first of the piece's chunks, of this stream
      const int inc = pc.pair ? 1 : 2;
      const int row0 = pc.own ? paged_own_row(A, pc.len) : 0;
      const int end = (pc.own ? pc.len : A.shared) - row0;
      int rows;  // query rows of the tile
      if (pc.own)
        rows = A.group;
      else
        rows = imin(A.per_tile, A.batch - (pc.which + (pc.pair ? t : 0)) * A.per_tile) * A.group;
      const bool narrow = pc.own || narrow_prefix;  // warp wq of the warpgroup takes keys 32 wq .. 32 wq + 31
      const bool idle = !narrow && wq * 32 >= rows;  // no row of this warp holds a query
      float mref = kNegInf, l = 0.f;
      for (int c = pc.pair ? 0 : t; c < n && !failed; c += inc) {
        const int st = pc.pair ? step + 2 * c + t : step + c;
        const int limit = end - (pc.j0 + c) * kPgKeys;  // keys of this chunk that count
        if (!pg_warp_wait(b_s + 8 * s, (st >> 1) & 1)) {
          failed = true;
          break;
        }
        if (limit < kPgKeys && limit % A.page_size != 0) {
          // The last page's rows past the end hold anything: zeros instead, so that their
          // probability of 0 gives 0.
          const int i = 2 * (chunk + c) + 1;
          if (!pg_warp_wait(b_full + 8 * (i % kRing), (i / kRing) & 1)) {
            failed = true;
            break;
          }
          const int stop = (limit / A.page_size + 1) * A.page_size;
          unsigned char* vt = gbase + (s_ring - base) + (i % kRing) * kTB;
          for (int x = row; x < (stop - limit) * kBoxes * 8; x += 128) {
            const int box = x / ((stop - limit) * 8), r = x - box * (stop - limit) * 8;
            *reinterpret_cast<uint4*>(vt + box * kBox + limit * 128 + r * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tc_fence_after();
        const uint64_t scale2 = pg_pair(A.scale_log2, A.scale_log2);
        uint64_t sum[2] = {0, 0};
        if (narrow) {
          uint32_t r[32], pk[16], none[16];
          tc_ld32(t_s + 32 * wq, r);
          tc_wait_ld();
          pg_mask(r, limit - 32 * wq);
          pg_reference<D>(pg_max(r, kNegInf) * A.scale_log2, lane < rows, c >= inc, t_o, mref, l);
          const float m = mref == kNegInf ? 0.f : -mref;
          pg_probs<T>(r, scale2, pg_pair(m, m), sum, pk);
#pragma unroll
          for (int x = 0; x < 16; ++x) none[x] = 0u;
#pragma unroll
          for (int x = 0; x < 4; ++x) {  // no probability for the other warps' keys
            if (x == wq)
              tc_st16(t_s + kPgP + 16 * x, pk);
            else
              tc_st16(t_s + kPgP + 16 * x, none);
          }
        } else if (!idle) {
          // Once for the maximum, then again 32 at a time (the row's 128 scores would not fit
          // the registers).  P takes the place of the last 64 scores, held in registers by then.
          uint32_t x0[32], x1[32], pk[16];
          tc_ld32(t_s, x0);
          tc_ld32(t_s + 32, x1);
          tc_wait_ld();
          pg_mask(x0, limit);
          pg_mask(x1, limit - 32);
          float mx = pg_max(x1, pg_max(x0, kNegInf));
          tc_ld32(t_s + 64, x0);
          tc_ld32(t_s + 96, x1);
          tc_wait_ld();
          pg_mask(x0, limit - 64);
          pg_mask(x1, limit - 96);
          mx = pg_max(x1, pg_max(x0, mx));
          pg_reference<D>(mx * A.scale_log2, row < rows, c >= inc, t_o, mref, l);
          const float m = mref == kNegInf ? 0.f : -mref;
          const uint64_t m2 = pg_pair(m, m);
          pg_probs<T>(x0, scale2, m2, sum, pk);
          tc_st16(t_s + kPgP + 32, pk);
          tc_ld32(t_s, x0);
          pg_probs<T>(x1, scale2, m2, sum, pk);
          tc_st16(t_s + kPgP + 48, pk);
          tc_wait_ld();
          tc_ld32(t_s + 32, x1);
          pg_mask(x0, limit);
          pg_probs<T>(x0, scale2, m2, sum, pk);
          tc_st16(t_s + kPgP, pk);
          tc_wait_ld();
          pg_mask(x1, limit - 32);
          pg_probs<T>(x1, scale2, m2, sum, pk);
          tc_st16(t_s + kPgP + 16, pk);
        }
        const float2 add = pg_two(pg_add2(sum[0], sum[1]));
        l += add.x + add.y;
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(b_p + 8 * s);
      }
      if (!failed && (pc.pair || t < n)) {
        // ---- this stream's partial result of the piece
        if (!pg_warp_wait(b_o + 8 * s, items & 1)) failed = true;
        ++items;
        tc_fence_after();
        const size_t slot = size_t(int(blockIdx.x) + pc.unit) * 2 + t;
        const int tile = pc.which + (pc.pair ? t : 0);
        float* o_to = pc.own ? A.o_own + slot * A.group * D : A.o_prefix + slot * kPgTile * D;
        float2* ml_to = pc.own ? A.ml_own + slot * A.group : A.ml_prefix + slot * kPgTile;
        if (narrow) {
          // The four warps' results over their keys, joined in shared memory: this stream's half
          // of the piece's Q tile, which no MMA reads any more.
          float* part = reinterpret_cast<float*>(gbase + (qseq & 1) * kTB + s * (kTB / 2));  // [4][8][D]
          float2* ml = g_ml + s * 4 * kPgNarrow;
          if (lane < rows) ml[wq * kPgNarrow + lane] = make_float2(mref, l);
#pragma unroll
          for (int x = 0; x < D; x += 32) {
            uint32_t o[32];
            tc_ld32(t_o + x, o);
            tc_wait_ld();
            if (lane < rows) {  // 16-byte words of a row turned by the row, against bank conflicts
#pragma unroll
              for (int y = 0; y < 32; y += 4)
                *reinterpret_cast<uint4*>(part + (wq * kPgNarrow + lane) * D + (((x + y) >> 2) ^ lane) * 4) =
                    make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]);
            }
          }
          if (!wg_sync()) failed = true;
          for (int i = row; i < rows * D; i += 128) {
            const int g = i / D, d = i % D;
            float m = kNegInf;
#pragma unroll
            for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[w * kPgNarrow + g].x);
            float o = 0.f, sum = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const float2 v = ml[w * kPgNarrow + g];
              if (v.x == kNegInf) continue;
              const float f = pg_exp2(v.x - m);
              o = fmaf(f, part[(w * kPgNarrow + g) * D + (((d >> 2) ^ g) << 2) + (d & 3)], o);
              sum = fmaf(f, v.y, sum);
            }
            if (failed) break;
            if (!pc.own && !takes_part(tile, g)) m = kNegInf;
            o_to[i] = o;
            if (d == 0) ml_to[g] = make_float2(m, sum);
          }
          fence_proxy_async_smem();  // the next Q tile there is written by TMA
          if (!wg_sync()) failed = true;
          if (row == 0) mbar_arrive(b_merge + 16 * s + 8 * (qseq & 1));  // done with its half of the Q tile
        } else if (!idle && !failed) {
          const bool counts = row < rows;
#pragma unroll
          for (int x = 0; x < D; x += 32) {
            uint32_t o[32];
            tc_ld32(t_o + x, o);
            tc_wait_ld();
            if (counts) {
#pragma unroll
              for (int y = 0; y < 32; y += 4)
                *reinterpret_cast<uint4*>(o_to + row * D + x + y) = make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]);
            }
          }
          // a sequence without the whole prefix does not take part
          if (counts) ml_to[row] = takes_part(tile, row) ? make_float2(mref, l) : make_float2(kNegInf, 0.f);
        }
        tc_fence_before();
      }
      qseq += pc.pair ? 2 : 1;
      step += pc.pair ? 2 * n : n;
      chunk += n;
    }
  }
  if (failed) atomicOr(flag, 1);
  allow_dependents();
  tc_fence_before();
  __syncthreads();
  if (*flag != 0 && tid == 0) atomicOr(A.status, 1);
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kPgTmemCols) : "memory");
  }
}

// Joins the partials of one query row per CTA of D threads: weights 2^(m - max m) of its
// partials (prefix pieces, then own pieces, in line order), then thread d sums output d.
constexpr int kPgMaxParts = 4 * 512;  // two streams x (prefix, own) x CTAs

template <typename T, int D>
__global__ void __launch_bounds__(D) sink_paged_combine_kernel(const __grid_constant__ PagedArgs A) {
  __shared__ float w[kPgMaxParts];
  __shared__ int src[kPgMaxParts];
  __shared__ float red[D / 32], red2[D / 32];
  grid_dependency_wait();
  allow_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hq = A.heads_kv * A.group;
  const int b = int(blockIdx.x) / hq, q = int(blockIdx.x) - b * hq, h = q / A.group, g = q - h * A.group;
  const PagedLine L = paged_line<D>(A, A.offsets[A.batch], A.offsets[A.batch + 1] != 0);
  const int len = paged_len(A, b);
  T* out = reinterpret_cast<T*>(A.out) + b * A.o_sb + q * A.o_sh;
  if (len == 0) {
    out[tid] = Elem<T>::from_f(0.f);
    return;
  }
  // ---- where the partials are: CTAs [c0, c0 + np) of the prefix unit, [c1, c1 + no) of the own unit
  int c0 = 0, np = 0, c1 = 0, no = 0, sub0 = 0, subs = 0, prow = 0, unit_p = 0;
  long long base_p = 0, base_o = 0;
  int cost_p = 1;
  if (L.chunks > 0 && len >= A.shared) {
    const int tile = b / A.per_tile, grp = tile >> 1;
    const bool pair = grp < L.pairs;
    unit_p = h * L.groups + grp;
    cost_p = pair ? PgCost<D>::kPair : PgCost<D>::kOne;
    base_p = h * L.head_cost + (long long)grp * L.chunks * PgCost<D>::kPair;
    c0 = paged_cta_of(L, A.ctas, base_p);
    np = paged_cta_of(L, A.ctas, base_p + (long long)(L.chunks - 1) * cost_p) - c0 + 1;
    sub0 = pair ? tile & 1 : 0;
    subs = pair ? 1 : 2;
    prow = (b - tile * A.per_tile) * A.group + g;
  }
  const int n_own = paged_own_chunks(A, len);
  if (n_own > 0) {
    base_o = L.prefix_cost + (long long)L.own_cost * ((long long)A.offsets[b] * A.heads_kv + (long long)h * n_own);
    c1 = paged_cta_of(L, A.ctas, base_o);
    no = paged_cta_of(L, A.ctas, base_o + (long long)(n_own - 1) * L.own_cost) - c1 + 1;
  }
  const int n = np * 2 + no * 2;
  float mx = kNegInf;
  for (int i = tid; i < n; i += D) {
    const bool own = i >= 2 * np;
    const int k = own ? i - 2 * np : i;
    const int c = (own ? c1 : c0) + (k >> 1), sub = k & 1;
    int j0, j1;
    paged_span(paged_cut(L, A.ctas, c), paged_cut(L, A.ctas, c + 1), own ? base_o : base_p, own ? n_own : L.chunks,
               own ? L.own_cost : cost_p, j0, j1);
    float2 ml = make_float2(kNegInf, 0.f);
    int at = 0;
    if (own) {
      if (sub < j1 - j0) {
        at = ((c + b * A.heads_kv + h) * 2 + sub) * A.group + g;
        ml = A.ml_own[at];
      }
    } else if (j1 > j0 && (subs == 1 ? sub == sub0 : sub < j1 - j0)) {
      at = ((c + unit_p) * 2 + sub) * kPgTile + prow;
      ml = A.ml_prefix[at];
    }
    w[i] = ml.x;
    src[i] = at;
    mx = fmaxf(mx, ml.x);
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, off));
  __syncthreads();
  if (lane == 0) red[warp] = mx;
  __syncthreads();
  for (int i = 0; i < D / 32; ++i) mx = fmaxf(mx, red[i]);
  float sum = 0.f;
  for (int i = tid; i < n; i += D) {
    const float m = w[i];
    float x = 0.f;
    if (m != kNegInf) {
      const bool own = i >= 2 * np;
      x = pg_exp2(m - mx);
      sum = fmaf(x, (own ? A.ml_own : A.ml_prefix)[src[i]].y, sum);
    } else {
      src[i] = -1;
    }
    w[i] = x;
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(kFull, sum, off);
  if (lane == 0) red2[warp] = sum;
  __syncthreads();
  sum = 0.f;
  for (int i = 0; i < D / 32; ++i) sum += red2[i];
  float o = 0.f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const int at = src[i];
    if (at >= 0) o = fmaf(w[i], (i >= 2 * np ? A.o_own : A.o_prefix)[size_t(at) * D + tid], o);
  }
  out[tid] = Elem<T>::from_f(sum == 0.f ? 0.f : o / sum);
}

}  // namespace sinkb200
