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
// Inside a CTA two softmax warpgroups each own a stream of steps; a step is one tile of query
// rows against one chunk: scores S = Q K^T, probabilities P, O += P V.  Step n is on stream
// n & 1.  With two query tiles (a pair) every chunk is a step on both streams, one per tile, and
// K and V are read from shared memory for 256 query rows; with one tile chunks alternate
// between the streams.  A step's scores come in two halves of 64 keys with a TMEM buffer each:
// while a warpgroup takes the exponentials of one half, the tensor cores fill the other.  A
// thread owns a query row (a TMEM lane): no reduction across threads.  P goes back to TMEM over
// its own scores, 16-bit, and is the MMA's A operand from there (one rounding to the cache's
// type: the tensor cores take 16-bit operands; the sum of probabilities is of the unrounded
// ones).  The reference maximum only moves when a score passes it by 2^8 (then O is rescaled in
// TMEM), so the usual half touches O in the MMA only.
//
// A tile of at most 8 query rows (own work, a prefix for a tiny batch) would leave all but one
// warp idle.  Such a narrow tile holds its rows four times, 32 lanes apart, and warp w of the
// warpgroup takes the w-th quarter of the keys, probability 0 elsewhere; the four partial
// results are joined at the end of the piece.
//
// Measured, against the rate of a plain copy (6.5 TB/s) and of a library product (1672 TFLOP/s):
// 64 sequences of 16K own rows, 8 kv heads, D = 64: 333 us, 6.4 TB/s; of 1K to 16K rows, D = 128:
// 374 to 432 us, 5.4 to 6.3 TB/s.  A prefix of 32K rows for 64 sequences of 4 query heads per kv
// head, D = 128: 49 us, 700 TFLOP/s; for 256, D = 64: 131 us, 520 TFLOP/s, bound by the
// exponentials (53 % of the special-function rate) and the wait for the products between them.
// 4K shared and 16 to 1020 own rows, 64 sequences: 43 us for 23 us of bytes, 8 us of it start
// and join.
#pragma once

#include <cuda.h>
#include <limits.h>

#include <type_traits>

#include "sink_chunk.cuh"
#include "sink_tcgen05.cuh"

namespace sinkb200 {

constexpr int kPgKeys = 128;      // keys per chunk
constexpr int kPgHalf = 64;       // keys per half step
constexpr int kPgTile = 128;      // query rows per tile
constexpr int kPgThreads = 352;   // two softmax warpgroups, the load warp, two MMA warps
constexpr int kPgLoadWarp = 8, kPgQkWarp = 9, kPgPvWarp = 10;
constexpr int kPgNarrow = 8;      // query rows of a tile up to which four warps share its keys
constexpr float kPgRescale = 8.f; // log2
constexpr int kPgO = 256;         // TMEM: S of stream s, half h at 128 s + 64 h; O at 256 + 128 s
constexpr int kPgTmemCols = 512;
constexpr int kPgSteps = 16;      // step records in flight between the load warp and the MMA warps

// Shared memory: two wide Q tiles, or in the place of the first four narrow ones, their 8-row
// blocks interleaved, and in that of the second the narrow tiles' merge area, half per stream |
// the ring of K and V tiles | barriers and records.
template <int D>
struct PgGeom {
  static constexpr int kTileBytes = kPgKeys * D * 2;  // a K, V or Q tile: D / 64 boxes of 128 rows
  static constexpr int kBoxBytes = kPgKeys * 128;
  static constexpr int kMergeBytes = 2 * 4 * kPgNarrow * D * 4;
  static constexpr int kRing = D == 128 ? 5 : 12;     // K and V tiles in flight
  static constexpr int kBarBytes = 1152;
  static constexpr int kSmem = 1024 + (2 + kRing) * kTileBytes + kBarBytes;
  static_assert(kMergeBytes <= kTileBytes && kSmem <= 232448, "227 KB of shared memory");
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
  float* o_prefix;   // [prefix slots][2][D / 4][128][4]
  float2* ml_prefix; // [prefix slots][2][128] (maximum, sum)
  float* o_own;      // [own slots][2][G][D]
  float2* ml_own;
  const char* v;     // the V pool, for the combine's look at values that are not finite
  int64_t v_sp, v_sh;
  int2* bounds;      // first and last CTA with a piece of the unit: prefix units, then own units
  int units;         // prefix units that `bounds` has room for
  int batch, heads_kv, group, page_size, pages, table_width, shared;
  int per_tile, tiles;  // sequences per query tile, tiles per kv head
  int ctas;
  float scale_log2;  // of |scale|
  uint32_t negate;   // scale < 0: the MMA negates Q
  int wait_polls;    // of each bounded wait (kWaitPolls unless a failure-detection test shortens it)
  int skip_tile;     // failure-detection test hook, -1 when off: the K or V tile from which on no CTA loads
};

// ------------------------------------------------------------------ the line of work

// Costs of a chunk in units of 64 clocks of one SM, by measurement (only their ratios count): one
// tile or a pair of tiles on it, and an own chunk, at least kOwnMin and, where memory bounds the own
// work, its share of the time that memory takes for all of it (kOwnMem when every SM streams); kUnit
// for each own unit, its query and the join of its result.  (Without kUnit the CTAs of short units
// finish last: 64 sequences with 4K shared and 16 to 1020 own rows 44.5 us without, 43.2 with 14,
// 44.4 with 30, 45.5 with 40; 64 sequences of 512 own rows, units all alike, 46.0 without and 46.7
// with 14.  A pair at 70 and 58 (D = 128, 64): 43.2 us, 42.0 at 80 and 62, 42.0 at 90 and 68, the
// same with 16K shared and 512 own rows 56.5, 57.5, 61.3.)
template <int D>
struct PgCost {
  static constexpr int kPair = D == 128 ? 80 : 62;
  static constexpr int kOne = D == 128 ? 43 : 34;
  static constexpr int kOwnMin = D == 128 ? 34 : 25;
  static constexpr int kOwnMem = D == 128 ? 43 : 26;
  static constexpr int kUnit = 14;
};

// a / b for b > 0, in 32 bits where they suffice (a 64-bit division takes several hundred clocks).
__device__ __forceinline__ long long pg_div(long long a, long long b) {
  if (((a | b) >> 32) == 0) return (long long)(unsigned(a) / unsigned(b));
  return a / b;
}

struct PagedLine {
  int chunks;            // prefix chunks (0: nothing shared, or no sequence that has it all)
  int units;             // prefix units: kv heads x groups of up to two tiles
  int groups, pairs;     // groups per head, the first `pairs` of them of two tiles
  int own_cost;
  long long head_cost;   // prefix cost of one head
  long long prefix_cost, total;
  long long per_cta;     // cost of a CTA's piece: at least one chunk starts in every one
};

template <int D>
__device__ __forceinline__ PagedLine paged_line(const PagedArgs& A, int own_chunks, int own_seqs, bool prefix) {
  using C = PgCost<D>;
  PagedLine L;
  L.chunks = prefix ? (A.shared + kPgKeys - 1) / kPgKeys : 0;
  L.pairs = A.tiles / 2;
  L.groups = (A.tiles + 1) / 2;
  L.units = L.chunks > 0 ? A.heads_kv * L.groups : 0;
  L.head_cost = (long long)L.chunks * (L.pairs * C::kPair + (L.groups - L.pairs) * C::kOne);
  L.prefix_cost = L.head_cost * A.heads_kv;
  const long long own = (long long)own_chunks * A.heads_kv;
  const float share = own > 0 ? float(L.prefix_cost) / float(own) : 0.f;
  L.own_cost = imax(C::kOwnMin, C::kOwnMem - int(fminf(share, float(C::kOwnMem))));
  L.total = L.prefix_cost + own * L.own_cost + (long long)own_seqs * A.heads_kv * C::kUnit;
  const int most = imax(own > 0 ? C::kUnit + L.own_cost : 0, L.chunks == 0 ? 0 : L.pairs > 0 ? C::kPair : C::kOne);
  L.per_cta = pg_div(L.total + A.ctas - 1, A.ctas);
  if (L.per_cta < most) L.per_cta = most;
  return L;
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

// Chunks [j0, j1) of the unit at `base`, n chunks of cost w after a cost u (u + n * w < 2^31), that
// start in [0, span).  The first starts at the base, the others behind u and those before them.
__device__ __forceinline__ void paged_span(int span, int base, int n, int w, int u, int& j0, int& j1) {
  auto started = [&](int x) -> int {  // chunks that start before x
    if (x <= base) return 0;
    const unsigned d = unsigned(x) - unsigned(base);
    if (d >= unsigned(u) + unsigned(n) * unsigned(w)) return n;
    return d <= unsigned(u + w) ? 1 : int((d - unsigned(u) + unsigned(w) - 1) / unsigned(w));
  };
  j0 = started(0);
  j1 = started(span);
}

struct PagedPiece {
  int unit;    // of the prefix, or b * heads_kv + h
  int h;
  int which;   // prefix: first tile; own: the sequence
  int j0, j1;  // chunks
  int n;       // chunks of the whole unit
  int len;     // own: the sequence's length
  bool own, pair;
};

// Walks the pieces of one CTA in line order, positions counted from the start of its part (the host
// keeps a part below 2^29).  Every role of the CTA runs its own copy.
struct PagedWalk {
  int span, base;        // length of the part; where the next unit starts
  int unit, h, at, len;  // at: group of the head, or sequence
  bool own;

  __device__ __forceinline__ bool next(const PagedArgs& A, const PagedLine& L, PagedPiece& p) {
    while (base < span) {
      int n, w, u = 0;
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
        u = unit_cost;
        p.which = at;
        p.pair = false;
      }
      p.unit = unit;
      p.h = h;
      p.own = own;
      p.len = len;
      p.n = n;
      if (own && n == 0) {
        unit += A.heads_kv - h;
        h = 0;
        ++at;
        len = -1;
        continue;
      }
      paged_span(span, base, n, w, u, p.j0, p.j1);
      base += u + n * w;
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
  int cost_pair, cost_one, unit_cost;
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

// True in one lane of the warp.
__device__ __forceinline__ bool pg_elect() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// A wait of at most `polls` polls (one at least), and one whose answer the whole warp shares.
__device__ __forceinline__ bool pg_wait(uint32_t bar, uint32_t parity, int polls) {
#pragma unroll 1
  for (int i = 0;;) {
    if (mbar_try_wait(bar, parity)) return true;
    if (i >= 64) __nanosleep(256);
    if (++i >= polls) return false;
  }
}
__device__ __forceinline__ bool pg_warp_wait(uint32_t bar, uint32_t parity, int polls) {
  return __all_sync(kFull, pg_wait(bar, parity, polls));
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

// N scores of a query row (fp32 bits), keys from `limit` on left out: -infinity.
template <int N>
__device__ __forceinline__ void pg_mask(uint32_t (&r)[N], int limit) {
  if (limit < N) {
#pragma unroll
    for (int x = 0; x < N; ++x)
      if (x >= limit) r[x] = __float_as_uint(kNegInf);
  }
}

template <int N>
__device__ __forceinline__ float pg_max(const uint32_t (&r)[N]) {
  float m[4] = {kNegInf, kNegInf, kNegInf, kNegInf};  // four chains: latency, not rate, bounds a step
#pragma unroll
  for (int x = 0; x < N; x += 8) {
#pragma unroll
    for (int y = 0; y < 4; ++y)
      m[y] = fmaxf(m[y], fmaxf(__uint_as_float(r[x + y]), __uint_as_float(r[x + 4 + y])));
  }
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// Moves the row's reference maximum up to `mx` (log2 units) when that passes it by kPgRescale:
// the sum and, if `has_o`, the row's O in TMEM are rescaled, once the last MMA on it is
// complete (phase parity `parity` of b_pv).  Rows that are no query (`valid` false) compute along.
// False when a wait ran out.
template <int D>
__device__ __forceinline__ bool pg_reference(float mx, bool valid, bool has_o, uint32_t t_o, uint32_t b_pv,
                                             uint32_t parity, int polls, float& mref, float& l) {
  const bool need = valid && mx > mref + kPgRescale;
  if (!__any_sync(kFull, need)) return true;
  float alpha = 1.f;
  if (need) {
    alpha = pg_exp2(mref - mx);
    mref = mx;
    l *= alpha;
  }
  if (has_o) {
    if (!pg_warp_wait(b_pv, parity, polls)) return false;
    tc_fence_after();
#pragma unroll 1
    for (int x = 0; x < D; x += 32) {
      uint32_t o[32];
      tc_ld_raw(t_o + x, o);
      tc_wait_ld();
#pragma unroll
      for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * alpha);
      tc_st_raw(t_o + x, o);
    }
  }
  return true;
}

// Probabilities 2^(scale s - m) of N scores, their sum added to `sum` (two accumulators),
// rounded to T and packed.  (Half, a quarter or an eighth of the powers in FMA arithmetic beside
// the special-function unit changed nothing: 256 query rows x 32K keys 141 us each way.)
template <typename T, int N>
__device__ __forceinline__ void pg_probs(const uint32_t (&r)[N], uint64_t scale2, float m, uint64_t (&sum)[2],
                                         uint32_t* pk) {
  const uint64_t m2 = pg_pair(-m, -m);
#pragma unroll
  for (int x = 0; x < N / 2; ++x) {
    const uint64_t e = pg_fma2(pg_pair(__uint_as_float(r[2 * x]), __uint_as_float(r[2 * x + 1])), scale2, m2);
    const float2 v = pg_two(e);
    const float p0 = pg_exp2(v.x), p1 = pg_exp2(v.y);
    sum[x & 1] = pg_add2(sum[x & 1], pg_pair(p0, p1));
    pk[x] = pg_pack<T>(p0, p1);
  }
}

// The softmax of a half step on N scores of the thread's row: packed probabilities, and l, mref
// and O moved on.  The probabilities are taken against the reference maximum as it stands while
// the scores' own maximum is still being found, so that neither waits for the other, and
// taken again in the rare half step that moves the reference; a piece's first half step
// (`fresh`) knows no reference yet and looks first.  False when a wait ran out.
template <typename T, int D, int N>
__device__ __forceinline__ bool pg_half_step(uint32_t (&r)[N], int keys, bool valid, bool fresh, float scale,
                                             uint64_t scale2, uint32_t t_o, uint32_t b_pv, uint32_t parity,
                                             int polls, float& mref, float& l, uint32_t* pk) {
  pg_mask(r, keys);
  uint64_t sum[2] = {0, 0};
  if (!fresh) pg_probs<T>(r, scale2, mref == kNegInf ? 0.f : mref, sum, pk);
  const float mx = pg_max(r) * scale;
  if (__any_sync(kFull, valid && mx > mref + kPgRescale) || fresh) {
    if (!pg_reference<D>(mx, valid, !fresh, t_o, b_pv, parity, polls, mref, l)) return false;
    sum[0] = sum[1] = 0;
    pg_probs<T>(r, scale2, mref == kNegInf ? 0.f : mref, sum, pk);
  }
  const float2 add = pg_two(pg_add2(sum[0], sum[1]));
  l += add.x + add.y;
  return true;
}

// A partial result's (maximum, sum).  A maximum of -infinity says that nothing is there, and is
// what NaN scores leave too (fmaxf passes over them): their sum is NaN, so they count as a
// partial with a maximum of 0, and the row's result is NaN.
__device__ __forceinline__ float2 pg_partial(float mref, float l) {
  return make_float2(mref == kNegInf && l != 0.f ? 0.f : mref, l);
}

// What the MMA warps have to know of a step, written by the load warp.
struct PgStep {
  static constexpr uint32_t kFirst = 1u;                   // the piece's first step on its stream
  static constexpr uint32_t kQWait = 2u, kQRelease = 4u;   // first, last chunk of the Q tile
  static constexpr uint32_t kMore = 8u;                    // the chunk has a second step
  static constexpr uint32_t kStop = 16u;                   // no step: the end
  // bits 8..11: Q slot (0, 1 wide; 2.. narrow), bit 12: the slot's phase parity, bits 16..: the
  // tile's shared-memory address in 16-byte words
};

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
  // mbarriers: full, empty [kRing]; qfull, qempty [6]; s, p, pv [stream * 2 + half]; rec [4]; wg [stream]; done
  const uint32_t b_full = s_bar, b_empty = b_full + 8 * kRing, b_qfull = b_empty + 8 * kRing, b_qempty = b_qfull + 48;
  const uint32_t b_s = b_qempty + 48, b_p = b_s + 32, b_pv = b_p + 32, b_rec = b_pv + 32;
  const uint32_t b_wg = b_rec + 32, b_done = b_wg + 16;
  unsigned char* g_bar = gbase + (s_bar - base);
  static_assert(16 * kRing + 96 + 128 + 16 + 8 <= 464, "barriers");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(g_bar + 464);
  int* flag = reinterpret_cast<int*>(g_bar + 468);
  int* start = reinterpret_cast<int*>(g_bar + 472);             // first own sequence, its length, cost before (64-bit)
  long long* scan = reinterpret_cast<long long*>(g_bar + 488);  // [11] warp sums
  float2* g_ml = reinterpret_cast<float2*>(g_bar + 576);        // [2 streams][4 warps][8 rows] of narrow tiles
  uint32_t* steps = reinterpret_cast<uint32_t*>(g_bar + 576 + 2 * 4 * kPgNarrow * 8);  // [kPgSteps]
  static_assert(576 + 2 * 4 * kPgNarrow * 8 + 4 * kPgSteps <= G_::kBarBytes, "records");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(b_full + 8 * i, 1);
      mbar_init(b_empty + 8 * i, 1);
    }
    for (int i = 0; i < 6; ++i) {
      mbar_init(b_qfull + 8 * i, 1);
      mbar_init(b_qempty + 8 * i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(b_s + 8 * i, 1);
      mbar_init(b_p + 8 * i, 4);
      mbar_init(b_pv + 8 * i, 1);
      mbar_init(b_rec + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(b_wg + 8 * i, 4);
    mbar_init(b_done, 2);
    *flag = 0;
    start[0] = A.batch;
    start[1] = start[2] = start[3] = 0;
    fence_mbar_init();
  }
  if (tid == 32 * kPgLoadWarp) {
    tma_prefetch_map(&A.qtile);
    tma_prefetch_map(&A.qgroup);
    tma_prefetch_map(&A.kmap);
    tma_prefetch_map(&A.vmap);
  }
  __syncwarp();
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "n"(kPgTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  grid_dependency_wait();  // lengths, table, query and cache rows are written

  // ---- the line: own chunks before each thread's run of sequences
  const int per = (A.batch + kPgThreads - 1) / kPgThreads;
  const int b_lo = imin(tid * per, A.batch), b_hi = imin(b_lo + per, A.batch);
  long long mine = 0;  // chunks, and in the upper half sequences that have any
  bool full = false;
  for (int b = b_lo; b < b_hi; ++b) {
    const int len = paged_len(A, b), n = paged_own_chunks(A, len);
    mine += n > 0 ? (1ll << 32) + n : 0;
    full |= len >= A.shared;
    if (blockIdx.x == 0 && A.lens[b] > A.table_width * A.page_size) atomicOr(A.status, 2);
  }
  long long before = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long x = __shfl_up_sync(kFull, before, off);
    if (lane >= off) before += x;
  }
  if (lane == 31) scan[warp] = before;
  const bool prefix = __syncthreads_or(full) != 0 && A.shared > 0;
  long long all = 0;
#pragma unroll
  for (int w = 0; w < kPgThreads / 32; ++w) {
    if (w < warp) before += scan[w];
    all += scan[w];
  }
  before -= mine;
  const PagedLine L = paged_line<D>(A, int(all), int(all >> 32), prefix);
  PagedWalk walk;
  const long long lo = L.per_cta * blockIdx.x, rest = L.total - lo;
  walk.span = int(rest < 0 ? 0 : rest < L.per_cta ? rest : L.per_cta);
  walk.cost_pair = PgCost<D>::kPair;
  walk.cost_one = PgCost<D>::kOne;
  walk.unit_cost = PgCost<D>::kUnit;
  // cost of the own work of `n` (chunks, sequences) of all heads
  auto own_cost = [&](long long n) {
    return ((n & 0xffffffffll) * L.own_cost + (n >> 32) * PgCost<D>::kUnit) * A.heads_kv;
  };
  if (mine > 0) {  // the sequence whose work holds position lo
    const long long want = lo - L.prefix_cost;
    if (want >= own_cost(before) && want < own_cost(before + mine)) {
      long long c = before;
      for (int b = b_lo; b < b_hi; ++b) {
        const int len = paged_len(A, b), n = paged_own_chunks(A, len);
        const long long next = c + (n > 0 ? (1ll << 32) + n : 0);
        if (want < own_cost(next)) {
          start[0] = b;
          start[1] = len;
          *reinterpret_cast<long long*>(start + 2) = own_cost(c);
          break;
        }
        c = next;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // the CTA holds all 512 columns
  const uint32_t tmem_held = *tmem_slot;
  if (lo < L.prefix_cost) {
    walk.own = false;
    walk.len = 0;
    walk.h = int(pg_div(lo, L.head_cost));
    const long long r = lo - walk.h * L.head_cost;
    const long long pair_cost = (long long)L.chunks * PgCost<D>::kPair;
    walk.at = imin(int(pg_div(r, pair_cost)), L.groups - 1);  // the groups before the last are pairs
    walk.unit = walk.h * L.groups + walk.at;
    walk.base = int(walk.at * pair_cost - r);
  } else {
    walk.own = true;
    walk.at = start[0];
    const long long into = lo - L.prefix_cost - *reinterpret_cast<const long long*>(start + 2);
    walk.base = 0;
    walk.len = -1;
    walk.h = 0;
    if (walk.at < A.batch) {
      walk.len = start[1];
      const long long unit_cost = (long long)L.own_cost * paged_own_chunks(A, walk.len) + PgCost<D>::kUnit;
      walk.h = int(pg_div(into, unit_cost));
      walk.base = int(walk.h * unit_cost - into);
    }
    walk.unit = walk.at * A.heads_kv + walk.h;
  }

  bool failed = false;
  const int polls = A.wait_polls;
  const bool narrow_prefix = A.tiles == 1 && A.batch * A.group <= kPgNarrow;
  if (warp == kPgLoadWarp) {
    // ================================================================ loads (a lane per page of a tile)
    // The warp's own instructions bound a chunk that is in L2: with divisions by the ring's and the
    // pages' sizes and a wait per tile 0.99 us at D = 64, without 0.87 (0.74 is memory's rate), and
    // 1.16 in place of 1.27 at D = 128.  A second warp for V made 64 sequences with 4K shared rows
    // 45.2 us in place of 43.4.  Where the ring holds whole chunks one vote waits for both tiles;
    // an odd ring keeps K and V apart, not to leave its last slot empty.
    constexpr bool kBoth = kRing % 2 == 0;
    const int npg = kPgKeys / A.page_size, page_bits = 31 - __clz(A.page_size);
    const int qrow_bytes = A.group * 128 * kBoxes;
    const uint32_t box_rows = lane * A.page_size * 128;  // this lane's page within a box
    int slot_k = 0, slot_v = 1;                // ring slots of the next K and V,
    uint32_t phase_k = 1, phase_v = 1;         // and the parity of their release
    int tile = 0, step = 0;            // ring tiles and steps issued
    int wide = 0, thin = 0;            // wide and narrow Q tiles issued
    int bare = 0;                      // 1: the slot after the last tile's has a phase without a copy
    // An own piece reads its rows through its own row of the table, the shared ones (the prefix's,
    // or a shorter sequence's) through row 0.  `row0`, `limit`: this lane's first row of chunk 0,
    // and where the rows end.
    struct Rows {
      const int32_t* table;
      int row0, limit;
    };
    auto rows_of = [&](const PagedPiece& p) {
      const int own_row = p.own ? paged_own_row(A, p.len) : 0;
      return Rows{A.table + (p.own && own_row == A.shared ? p.which * A.table_sb : 0), own_row + lane * A.page_size,
                  lane >= npg ? 0 : p.own ? p.len : A.shared};
    };
    // This lane's page of chunk j, -1 where its rows are past the end.
    auto page_of = [&](const Rows& w, int j) -> int {
      const int row = w.row0 + j * kPgKeys;
      return unsigned(row) < unsigned(w.limit) ? w.table[row >> page_bits] : -1;
    };
    PagedPiece pc, ahead;
    bool live = walk.next(A, L, pc), more = false;
    Rows rows{A.table, 0, 0}, rows_ahead = rows;
    if (live) rows = rows_of(pc);
    int page = live ? page_of(rows, pc.j0) : -1;
    for (; live && !failed; live = more, pc = ahead, rows = rows_ahead) {
      uint32_t q_bits[2] = {0, 0};
      const bool narrow = pc.own || narrow_prefix;
      if (lane == 0) {
        int* bound = reinterpret_cast<int*>(A.bounds + (pc.own ? A.units : 0) + pc.unit);
        if (pc.j0 == 0) bound[0] = int(blockIdx.x);
        if (pc.j1 == pc.n) bound[1] = int(blockIdx.x);
      }
      if (narrow && wide > 0) {  // the narrow tiles take the wide ones' place
        for (int i = wide > 1 ? wide - 2 : 0; i < wide && !failed; ++i)
          failed = !pg_warp_wait(b_qempty + 8 * (i & 1), (i >> 1) & 1, polls);
        if (failed) break;
        wide = 0;
      }
      for (int t = 0; t < (pc.pair ? 2 : 1) && !failed; ++t) {
        const int slot = narrow ? 2 + (thin & 3) : wide & 1, use = narrow ? thin >> 2 : wide >> 1;
        if (use > 0 && !pg_warp_wait(b_qempty + 8 * slot, (use - 1) & 1, polls)) {
          failed = true;
          break;
        }
        // a narrow tile's rows once for each warp of the warpgroup, 32 TMEM lanes apart
        const int copies = narrow ? 4 : 1;
        const uint32_t bar = b_qfull + 8 * slot, dst = s_q + (narrow ? (slot - 2) * 1024 : slot * kTB);
        if (lane == 0) mbar_arrive_expect_tx(bar, (pc.own ? qrow_bytes : qrow_bytes * A.per_tile) * copies);
        __syncwarp();
        if (lane < copies * kBoxes) {  // a lane per copy
          const int x = lane / copies, c = lane - x * copies;
          tma_load_3d(dst + x * kBox + c * 32 * 128, pc.own ? &A.qgroup : &A.qtile, 64 * x, pc.h * A.group,
                      pc.own ? pc.which : (pc.which + t) * A.per_tile, bar);
        }
        q_bits[t] = uint32_t(slot) << 8 | uint32_t(use & 1) << 12 | (dst >> 4) << 16;
        narrow ? ++thin : ++wide;
      }
      more = walk.next(A, L, ahead);
      if (more) rows_ahead = rows_of(ahead);
      const int first_page = more ? page_of(rows_ahead, ahead.j0) : -1;  // in flight under this piece's chunks
      auto record = [&](int j) {  // a chunk's steps
        const uint32_t ends = (j + 1 == pc.j1 ? PgStep::kQRelease : 0u) | (j == pc.j0 ? PgStep::kQWait : 0u);
        if (pc.pair) {
          const uint32_t f = ends | (j == pc.j0 ? PgStep::kFirst : 0u);
          steps[step % kPgSteps] = f | PgStep::kMore | q_bits[0];
          steps[(step + 1) % kPgSteps] = f | q_bits[1];
        } else {
          steps[step % kPgSteps] = ends | (j - pc.j0 < 2 ? PgStep::kFirst : 0u) | q_bits[0];
        }
      };
      // (The test hook ends a piece early: a look at each tile made pages of 16 rows 2 % slower.)
      const unsigned into = unsigned(A.skip_tile - tile);
      const bool cut = into < 2u * unsigned(pc.j1 - pc.j0);
      const int end = cut ? pc.j0 + int(into / 2) : pc.j1;
      for (int j = pc.j0; j < end && !failed; ++j) {
        const int next_page = j + 1 < pc.j1 ? page_of(rows, j + 1) : first_page;
        const int nq = pc.pair ? 2 : 1;
        if (kBoth && !__all_sync(kFull, pg_wait(b_empty + 8 * slot_k, phase_k, polls) &&
                                            pg_wait(b_empty + 8 * slot_v, phase_v, polls))) {
          failed = true;
          break;
        }
        int at = page;
        if (at < 0 || at >= A.pages) {  // one past the pool: the copy reads zeros
          at = A.pages;
          if (unsigned(rows.row0 + j * kPgKeys) < unsigned(rows.limit)) atomicOr(A.status, 2);
        }
#pragma unroll
        for (int v = 0; v < 2; ++v, ++tile) {
          const int r = v ? slot_v : slot_k;
          if (!kBoth && !pg_warp_wait(b_empty + 8 * r, v ? phase_v : phase_k, polls)) {
            failed = true;
            break;
          }
          const uint32_t bar = b_full + 8 * r, dst = s_ring + r * kTB + box_rows;
          if (lane == 0) {
            if (v == 0) record(j);  // published by the arrival
            mbar_arrive_expect_tx(bar, kTB);
          }
          __syncwarp();
          if (lane < npg) {
#pragma unroll
            for (int x = 0; x < kBoxes; ++x)
              tma_load_4d(dst + x * kBox, v ? &A.vmap : &A.kmap, 64 * x, 0, pc.h, at, bar);
          }
        }
        if ((slot_k += 2) >= kRing) slot_k -= kRing, phase_k ^= 1;
        if ((slot_v += 2) >= kRing) slot_v -= kRing, phase_v ^= 1;
        step += nq;
        page = next_page;
      }
      if (cut && !failed) {
        failed = true;
        if ((into & 1) && pg_warp_wait(b_empty + 8 * slot_k, phase_k, polls)) {
          // the values alone are missing: the keys' slot counts as full, with what it holds
          if (lane == 0) {
            record(end);
            mbar_arrive(b_full + 8 * slot_k);
          }
          bare = 1;
        }
      }
    }
    if (!failed) {  // tell the MMA warps that the steps end here
      if (!pg_warp_wait(b_empty + 8 * slot_k, phase_k, polls)) {
        failed = true;
      } else {
        if (lane == 0) {
          steps[step % kPgSteps] = PgStep::kStop;
          mbar_arrive(b_full + 8 * slot_k);
        }
        bare = 1;
      }
    }
    // Whichever warp gives up on a wait, the copies in flight land before the CTA can exit (each
    // wait bounded; all are there at once where nothing failed).
    for (int i = tile - 1; i >= 0 && i >= tile - kRing + bare; --i)
      pg_warp_wait(b_full + 8 * (i % kRing), (i / kRing) & 1, kWaitPolls);
    for (int i = wide - 1; i >= 0 && i >= wide - 2; --i)
      pg_warp_wait(b_qfull + 8 * (i & 1), (i >> 1) & 1, kWaitPolls);
    for (int i = thin - 1; i >= 0 && i >= thin - 4; --i)
      pg_warp_wait(b_qfull + 8 * (2 + (i & 3)), (i >> 2) & 1, kWaitPolls);
  } else if (warp == kPgQkWarp) {
    // ================================================================ S = Q K^T
    // The MMA warps run as whole warps and let one lane issue: their addresses and descriptors
    // are then the same in every lane for the compiler too, and stay in uniform registers (issued
    // from inside a one-lane branch an MMA took 57 clocks, 30 this way).
    constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    const uint32_t negate = A.negate ? kPgNegateA : 0u;
    const uint32_t idesc = pg_idesc(kFmt, kPgHalf, false) | negate;
    const uint32_t idesc_whole = pg_idesc(kFmt, kPgKeys, false) | negate;
    const uint64_t desc = tc_desc(0, 16);
    const bool leader = pg_elect();
    int r = kRing - 2, phase = 1;  // ring slot and phase parity of the newest K
    for (int n = 0;;) {
      if ((r += 2) >= kRing) {
        r -= kRing;
        phase ^= 1;
      }
      if (!pg_warp_wait(b_full + 8 * r, phase, polls)) {
        failed = true;
        break;
      }
      // a pair's chunk has two steps, whose halves take turns: both streams move on together
      const uint32_t rec = steps[n % kPgSteps];
      const int many = rec & PgStep::kMore ? 2 : 1;
      const uint32_t rec1 = many == 2 ? steps[(n + 1) % kPgSteps] : rec;
      if (leader)
        for (int t = 0; t < many; ++t) mbar_arrive(b_rec + 8 * ((n + t) & 3));  // the P V warp may read them too
      if (rec & PgStep::kStop) break;
      if (rec & PgStep::kQWait) {
        if (!pg_warp_wait(b_qfull + 8 * ((rec >> 8) & 15u), (rec >> 12) & 1u, polls)) failed = true;
        if (many == 2 && !pg_warp_wait(b_qfull + 8 * ((rec1 >> 8) & 15u), (rec1 >> 12) & 1u, polls)) failed = true;
        if (failed) break;
      }
      const uint64_t kd = desc + ((s_ring + r * kTB) >> 4);
      if (many == 1) {
        // One step on the chunk: its 128 keys in one go (an MMA of 64 keys holds the tensor core as
        // long as one of 128).
        const int s = n & 1;
        if (n >= 2 && (!pg_warp_wait(b_pv + 16 * s, ((n >> 1) - 1) & 1, polls) ||
                       !pg_warp_wait(b_pv + 16 * s + 8, ((n >> 1) - 1) & 1, polls))) {
          failed = true;
          break;
        }
        tc_fence_after();
        const uint64_t qd = desc + (rec >> 16);
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (kk >> 2) * (kBox >> 4) + (kk & 3) * 2;
            tc_mma(s * 128, qd + off, kd + off, idesc_whole, kk > 0);
          }
          tc_commit(b_s + 16 * s);
          tc_commit(b_s + 16 * s + 8);
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll 1
          for (int t = 0; t < many; ++t) {
            const int s = (n + t) & 1;
            // the buffer is free once the product of two steps ago has read its probabilities
            if (n + t >= 2 && !pg_warp_wait(b_pv + 8 * (2 * s + h), (((n + t) >> 1) - 1) & 1, polls)) {
              failed = true;
              break;
            }
            tc_fence_after();
            const uint64_t qd = desc + ((t ? rec1 : rec) >> 16);
            if (leader) {
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk) {
                const uint32_t off = (kk >> 2) * (kBox >> 4) + (kk & 3) * 2;
                tc_mma(s * 128 + h * kPgHalf, qd + off, kd + off + h * (kPgHalf * 128 >> 4), idesc, kk > 0);
              }
              tc_commit(b_s + 8 * (2 * s + h));
            }
          }
          if (failed) break;
        }
      }
      if (failed) break;
      if (leader) {
        tc_commit(b_empty + 8 * r);
        if (rec & PgStep::kQRelease) {
          tc_commit(b_qempty + 8 * ((rec >> 8) & 15u));
          if (many == 2) tc_commit(b_qempty + 8 * ((rec1 >> 8) & 15u));
        }
      }
      n += many;
    }
    if (leader) tc_commit(b_done);  // TMEM is freed only after every MMA has completed
    pg_warp_wait(b_done, 0, kWaitPolls);
  } else if (warp == kPgPvWarp) {
    // ================================================================ O += P V
    constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t idesc = pg_idesc(kFmt, D, true);
    const uint64_t desc = tc_desc(0, kBox);
    const bool leader = pg_elect();
    int r = 1, phase = 0;  // ring slot and phase parity of the chunk's V
    for (int n = 0;;) {
      if (!pg_warp_wait(b_rec + 8 * (n & 3), (n >> 2) & 1, polls)) {
        failed = true;
        break;
      }
      const uint32_t rec = steps[n % kPgSteps];  // a pair's two steps are alike here
      if (rec & PgStep::kStop) break;
      const int many = rec & PgStep::kMore ? 2 : 1;
      if (many == 2 && !pg_warp_wait(b_rec + 8 * ((n + 1) & 3), ((n + 1) >> 2) & 1, polls)) failed = true;
      if (failed || !pg_warp_wait(b_full + 8 * r, phase, polls)) {
        failed = true;
        break;
      }
      const uint64_t vd = desc + ((s_ring + r * kTB) >> 4);
      const bool first = rec & PgStep::kFirst;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll 1
        for (int t = 0; t < many; ++t) {
          const int s = (n + t) & 1;
          if (!pg_warp_wait(b_p + 8 * (2 * s + h), ((n + t) >> 1) & 1, polls)) {
            failed = true;
            break;
          }
          tc_fence_after();
          if (leader) {
#pragma unroll
            for (int kk = 0; kk < kPgHalf / 16; ++kk)
              tc_mma_ta(kPgO + s * 128, s * 128 + h * kPgHalf + kk * 8, vd + (4 * h + kk) * (2048 >> 4), idesc,
                        h > 0 || kk > 0 || !first);
            tc_commit(b_pv + 8 * (2 * s + h));
          }
        }
        if (failed) break;
      }
      if (failed) break;
      if (leader) tc_commit(b_empty + 8 * r);
      if ((r += 2) >= kRing) {
        r -= kRing;
        phase ^= 1;
      }
      n += many;
    }
    if (leader) tc_commit(b_done);
    pg_warp_wait(b_done, 0, kWaitPolls);
  } else {
    // ================================================================ softmax: warpgroup s, a thread per query row
    const int s = warp >> 2, row = tid & 127, wq = warp & 3;
    const uint32_t lanes = uint32_t(wq * 32) << 16;
    const uint32_t t_s = tmem + s * 128 + lanes, t_o = tmem + kPgO + s * 128 + lanes;
    const uint64_t scale2 = pg_pair(A.scale_log2, A.scale_log2);
    int step = 0, chunk = 0, syncs = 0;  // steps and chunks before this piece; barriers of the warpgroup
    auto arrive = [&](uint32_t bar) {  // the warp's, once every lane is here
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto wg_sync = [&]() -> bool {  // the warpgroup's threads, bounded
      arrive(b_wg + 8 * s);
      return pg_warp_wait(b_wg + 8 * s, (syncs++) & 1, polls);
    };
    // whether prefix row r of tile `tile` belongs to a sequence that has the whole prefix
    auto takes_part = [&](int tile, int r) { return paged_len(A, tile * A.per_tile + r / A.group) >= A.shared; };
    PagedPiece pc;
    while (!failed && walk.next(A, L, pc)) {
      const int n = pc.j1 - pc.j0;
      const int t = (step & 1) ^ s;  // the tile, or the first of the piece's chunks, of this stream
      const int inc = pc.pair ? 1 : 2;
      const int end = pc.own ? pc.len - paged_own_row(A, pc.len) : A.shared;
      const int tile = pc.which + (pc.pair ? t : 0);
      const int rows = pc.own ? A.group : imin(A.per_tile, A.batch - tile * A.per_tile) * A.group;
      const bool narrow = pc.own || narrow_prefix;   // warp wq takes a quarter of the keys
      const bool idle = !narrow && wq * 32 >= rows;  // no row of this warp holds a query
      float mref = kNegInf, l = 0.f;
      for (int c = pc.pair ? 0 : t; c < n && !failed; c += inc) {
        const int st = pc.pair ? step + 2 * c + t : step + c;
        const int limit = end - (pc.j0 + c) * kPgKeys;  // keys of this chunk that count
        const uint32_t phase = (st >> 1) & 1;
        if (!pg_warp_wait(b_s + 16 * s, phase, polls)) {
          failed = true;
          break;
        }
        if (limit < kPgKeys && limit % A.page_size != 0) {
          // The last page's rows past the end hold anything: zeros instead, so that their
          // probability of 0 gives 0.  (This step's scores are there, so the slot's tile before has
          // been read and the barrier is in this tile's phase.)
          const int i = 2 * (chunk + c) + 1;
          if (!pg_warp_wait(b_full + 8 * (i % kRing), (i / kRing) & 1, polls)) {
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
        if (narrow) {  // both halves at once: a warp's keys are in one of them
          if (!pg_warp_wait(b_s + 16 * s + 8, phase, polls)) {
            failed = true;
            break;
          }
          tc_fence_after();
          uint32_t r[32], pk[16], none[16];
          tc_ld_raw(t_s + 32 * wq, r);
          tc_wait_ld();
          // (the product before is complete: the second half's scores were issued after it)
          if (!pg_half_step<T, D>(r, limit - 32 * wq, lane < rows, c < inc, A.scale_log2, scale2, t_o, b_pv + 16 * s + 8,
                                  phase ^ 1, polls, mref, l, pk)) {
            failed = true;
            break;
          }
#pragma unroll
          for (int x = 0; x < 16; ++x) none[x] = 0u;
#pragma unroll
          for (int x = 0; x < 4; ++x) {  // no probability for the other warps' keys
            if (x == wq)
              tc_st_raw(t_s + (x >> 1) * kPgHalf + (x & 1) * 16, pk);
            else
              tc_st_raw(t_s + (x >> 1) * kPgHalf + (x & 1) * 16, none);
          }
          tc_wait_st();
          tc_fence_before();
          arrive(b_p + 16 * s);
          arrive(b_p + 16 * s + 8);
          continue;
        }
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          if (h == 1 && !pg_warp_wait(b_s + 16 * s + 8, phase, polls)) {
            failed = true;
            break;
          }
          tc_fence_after();
          if (!idle) {
            uint32_t r[64], pk[32];
            tc_ld_raw(t_s + h * kPgHalf, r);
            tc_wait_ld();
            // the half step before on this stream: its product is complete before O may be rescaled
            if (!pg_half_step<T, D>(r, limit - h * kPgHalf, row < rows, c < inc && h == 0, A.scale_log2, scale2, t_o,
                                    b_pv + 16 * s + 8 * (h ^ 1), phase ^ h ^ 1, polls, mref, l, pk)) {
              failed = true;
              break;
            }
            tc_st_raw(t_s + h * kPgHalf, pk);  // over the half's own scores
            tc_wait_st();
          }
          tc_fence_before();
          arrive(b_p + 16 * s + 8 * h);
        }
      }
      const size_t slot = size_t(int(blockIdx.x) + pc.unit) * 2 + t;
      float* o_to = pc.own ? A.o_own + slot * A.group * D : A.o_prefix + slot * kPgTile * D;
      float2* ml_to = pc.own ? A.ml_own + slot * A.group : A.ml_prefix + slot * kPgTile;
      if (!failed && !pc.pair && t >= n) {  // one chunk: nothing on this stream
        if (row < rows) ml_to[row] = make_float2(kNegInf, 0.f);
      } else if (!failed) {
        // ---- this stream's partial result of the piece
        const int st = pc.pair ? step + 2 * (n - 1) + t : step + t + (n - 1 - t) / 2 * 2;  // the last step
        if (!pg_warp_wait(b_pv + 8 * (2 * s + 1), (st >> 1) & 1, polls)) failed = true;
        tc_fence_after();
        if (narrow) {
          // the four warps' results over their keys, joined in shared memory
          float* part = reinterpret_cast<float*>(gbase + kTB + s * (G_::kMergeBytes / 2));  // [4][8][D]
          float2* ml = g_ml + s * 4 * kPgNarrow;
          if (lane < rows) ml[wq * kPgNarrow + lane] = pg_partial(mref, l);
#pragma unroll
          for (int x = 0; x < D; x += 32) {
            uint32_t o[32];
            tc_ld_raw(t_o + x, o);
            tc_wait_ld();
            if (lane < rows) {  // 16-byte words of a row turned by the row, against bank conflicts
#pragma unroll
              for (int y = 0; y < 32; y += 4)
                *reinterpret_cast<uint4*>(part + (wq * kPgNarrow + lane) * D + (((x + y) >> 2) ^ lane) * 4) =
                    make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]);
            }
          }
          if (!wg_sync()) failed = true;
          for (int i = row; i < rows * D && !failed; i += 128) {
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
            if (!pc.own && !takes_part(tile, g)) m = kNegInf;
            o_to[pc.own ? i : ((d >> 2) * kPgTile + g) * 4 + (d & 3)] = o;
            if (d == 0) ml_to[g] = make_float2(m, sum);
          }
          if (!wg_sync()) failed = true;
        } else if (!idle && !failed) {
          const bool counts = row < rows;
#pragma unroll
          for (int x = 0; x < D; x += 32) {
            uint32_t o[32];
            tc_ld_raw(t_o + x, o);
            tc_wait_ld();
            if (counts) {  // a warp's rows side by side: 512 bytes per store
#pragma unroll
              for (int y = 0; y < 32; y += 4)
                *reinterpret_cast<uint4*>(o_to + (((x + y) >> 2) * kPgTile + row) * 4) =
                    make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]);
            }
          }
          // a sequence without the whole prefix does not take part
          if (counts) ml_to[row] = takes_part(tile, row) ? pg_partial(mref, l) : make_float2(kNegInf, 0.f);
        }
        tc_fence_before();
      }
      step += pc.pair ? 2 * n : n;
      chunk += n;
    }
  }
  if (failed) atomicOr(flag, 1);
  allow_dependents();  // (at the start, the waiting combine made 2 streams on a 1K prompt 1 us slower)
  tc_fence_before();
  __syncthreads();
  if (*flag != 0 && tid == 0) atomicOr(A.status, 1);
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_held), "n"(kPgTmemCols) : "memory");
  }
}

// Joins the partials of the G query rows of one (sequence, kv head) per CTA, in two steps: the
// weights 2^(m - max m) of each row's partials (prefix pieces, then own pieces, in line order,
// two streams each), then the weighted sums, 16 bytes of a row per thread.  Where a row has
// fewer words than the CTA threads, teams of threads share its partials and their sums are
// added in team order: the result does not depend on scheduling.  Bound by the latency of
// three dependent reads (bounds, maxima, words): 4 us for 512 CTAs, 12 us for 2048, in part under
// the attention's tail.
constexpr int kPgCombineThreads = 256;

// Which of NaN (bit 0), +infinity (1) and -infinity (2) the values of dims 4 x .. 4 x + 3 hold in
// the rows [0, len) of sequence b, kv head h: 3 bits a dim.  By a whole warp, a row per lane.
template <typename T, int D>
__device__ __noinline__ unsigned pg_value_kinds(const PagedArgs& A, int b, int h, int len, int x) {
  unsigned kinds = 0;
  for (int r = threadIdx.x & 31; r < len; r += 32) {
    const int page = (r < A.shared ? A.table : A.table + b * A.table_sb)[r / A.page_size];
    if (page < 0 || page >= A.pages) continue;
    const T* row = reinterpret_cast<const T*>(A.v) + page * A.v_sp + h * A.v_sh + r % A.page_size * D + 4 * x;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float v = Elem<T>::to_f(row[k]);
      kinds |= (isnan(v) ? 1u : !isinf(v) ? 0u : v > 0.f ? 2u : 4u) << (3 * k);
    }
  }
  return __reduce_or_sync(kFull, kinds);
}

template <typename T, int D>
__global__ void __launch_bounds__(kPgCombineThreads) sink_paged_combine_kernel(const __grid_constant__ PagedArgs A) {
  extern __shared__ float w[];  // [G][parts], then the teams' sums
  __shared__ float inv[kPgNarrow];
  __shared__ float4 sums[kPgCombineThreads];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = A.group;
  const int b = int(blockIdx.x) / A.heads_kv, h = int(blockIdx.x) - b * A.heads_kv;
  grid_dependency_wait();
  allow_dependents();
  // ---- where the partials are: CTAs [c.x, c.y] of the prefix unit and of the own unit (bounds are
  // read beside the length, before it is known whether they count; kept within the grid, since a
  // CTA that gave up on a wait leaves them unwritten)
  const int len = paged_len(A, b);
  const int tile = b / A.per_tile, grp = tile >> 1, unit = b * A.heads_kv + h;
  const int unit_p = h * ((A.tiles + 1) / 2) + grp;
  auto held = [&](int2 c) {
    c.x = imax(0, imin(c.x, A.ctas - 1));
    return make_int2(c.x, imax(c.x, imin(c.y, A.ctas - 1)));
  };
  const int2 cp = A.shared > 0 ? held(A.bounds[unit_p]) : make_int2(0, 0), co = held(A.bounds[A.units + unit]);
  const bool has_p = A.shared > 0 && len >= A.shared, has_o = paged_own_chunks(A, len) > 0;
  const bool pair = 2 * grp + 1 < A.tiles;
  const int subs = pair ? 1 : 2, sub0 = pair ? tile & 1 : 0;  // streams of a prefix piece with this tile
  const size_t slot_p = has_p ? size_t(cp.x + unit_p) * 2 : 0, slot_o = has_o ? size_t(co.x + unit) * 2 : 0;
  const size_t row_p = size_t(b - tile * A.per_tile) * G;
  const int n_p = has_p ? (cp.y - cp.x + 1) * subs : 0, n = n_p + (has_o ? (co.y - co.x + 1) * 2 : 0);
  auto part_p = [&](int i) { return slot_p + (subs == 2 ? i : 2 * i + sub0); };  // its [2]-slot
  constexpr int kWords = D / 4;
  const int items = G * kWords;                     // 16-byte words of the G rows, rows fastest
  const int teams = kPgCombineThreads / items;      // 1 to 16
  const int team = tid / items, item = tid - team * items;
  const int x = item / G, g = item - x * G;
  auto word = [&](int i) {  // this thread's word of partial i
    return *reinterpret_cast<const float4*>(
        i < n_p ? A.o_prefix + (part_p(i) * kPgTile * kWords + size_t(x) * kPgTile + row_p + g) * 4
                : A.o_own + ((slot_o + i - n_p) * G + g) * D + 4 * x);
  };
  constexpr int kAhead = 4;  // partials whose words are on their way while the weights are made
  float4 v[kAhead];
  if (team < teams) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (team + k * teams < n) v[k] = word(team + k * teams);
  }
  for (int gg = warp; gg < G; gg += kPgCombineThreads / 32) {
    auto ml_of = [&](int i) {
      return i < n_p ? A.ml_prefix[part_p(i) * kPgTile + row_p + gg] : A.ml_own[(slot_o + i - n_p) * G + gg];
    };
    const float2 first = lane < n ? ml_of(lane) : make_float2(kNegInf, 0.f);
    float mx = first.x;
    for (int i = lane + 32; i < n; i += 32) mx = fmaxf(mx, ml_of(i).x);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, off));
    float sum = 0.f;
    for (int i = lane; i < n; i += 32) {
      const float2 ml = i == lane ? first : ml_of(i);
      const float f = ml.x == kNegInf ? 0.f : pg_exp2(ml.x - mx);
      if (ml.x != kNegInf) sum = fmaf(f, ml.y, sum);
      w[gg * n + i] = ml.x == kNegInf ? -1.f : f;  // -1: nothing there
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(kFull, sum, off);
    if (lane == 0) inv[gg] = sum;
  }
  __syncthreads();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (team < teams) {
    auto add = [&](int i, const float4& p) {
      const float f = w[g * n + i];
      if (f < 0.f) return;
      o.x = fmaf(f, p.x, o.x);
      o.y = fmaf(f, p.y, o.y);
      o.z = fmaf(f, p.z, o.z);
      o.w = fmaf(f, p.w, o.w);
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (team + k * teams < n) add(team + k * teams, v[k]);
#pragma unroll 4
    for (int i = team + kAhead * teams; i < n; i += teams) add(i, word(i));
  }
  sums[tid] = o;
  __syncthreads();
  if (team == 0) {
    for (int k = 1; k < teams; ++k) {
      const float4 v = sums[k * items + item];
      o.x += v.x;
      o.y += v.y;
      o.z += v.z;
      o.w += v.w;
    }
  }
  // (a sum of 0 over rows that are there is that of scores all -infinity: 0 / 0, as in the formula)
  const float total = team == 0 ? inv[g] : 0.f, r = 1.f / total;
  float y[4] = {o.x * r, o.y * r, o.z * r, o.w * r};
  // A narrow tile meets every value with the probability 0 of the warps whose key it is not, and 0
  // times an infinity is NaN; so is it where a probability or weight that is not 0 rounds to 0.
  // Where the sum of probabilities is a number, a NaN is taken back to what the values say: the
  // infinity that is there, if it is of one sign and no NaN beside it (of a row whose score is
  // -infinity too: its probability of exactly 0 is not told from one that rounds to 0).
  const bool odd = total != 0.f && total == total && (y[0] != y[0] || y[1] != y[1] || y[2] != y[2] || y[3] != y[3]);
  for (unsigned left = __ballot_sync(kFull, odd); left != 0; left &= left - 1) {
    const int src = __ffs(left) - 1;
    const unsigned kinds = pg_value_kinds<T, D>(A, b, h, len, __shfl_sync(kFull, x, src));
    if (lane == src) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned kind = (kinds >> (3 * k)) & 7u;
        if (y[k] != y[k] && (kind == 2u || kind == 4u)) y[k] = kind == 2u ? -kNegInf : kNegInf;
      }
    }
  }
  if (team == 0) {
    T* out = reinterpret_cast<T*>(A.out) + b * A.o_sb + (h * G + g) * A.o_sh + 4 * x;
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = Elem<T>::from_f(len == 0 ? 0.f : y[k]);
  }
}

}  // namespace sinkb200
