// Rotary positions of up to three tensors in one launch: the rotation of q and k (forward and
// backward) and the paged cache's append (k rotated into its pages, v copied into its pages,
// q rotated beside them).
//
// A pair (x1, x2) of a head at position p, frequency f_i:
//   y1 = x1 c - x2 s,  y2 = x2 c + x1 s,   c = a cos(p f_i), s = a sin(p f_i),
// pairs (x_i, x_{i + R/2}) in the half layout, (x_{2i}, x_{2i+1}) interleaved, i < R/2; the
// dims from R on pass through.  The backward pass is the rotation by -p f_i.
//
// The angle p f_i and its reduction to a quarter turn are formed in fp64 (a position of 2^20
// leaves fp32 no fraction of a turn worth having), sin and cos of the remainder and the
// rotation itself in fp32, and the result is rounded once to the tensor's type.
//
// Bound: memory (every element read once and written once).  q and k of 4 x 8192 tokens, 40
// heads of 64, bf16: 57 to 61 us, 5.5 to 5.9 TB/s, 0.84 to 0.90 of a plain copy's rate, issue
// slots 67 % busy (three rows in flight per thread 63 us, five CTAs per SM 76 us, streaming cache
// hints within 1 %); a ragged append of 8 x 4096 tokens, 48 heads of 64: 51 to 52 us; one token:
// 3 us.
#pragma once

#include "sink_common.cuh"

namespace sinkb200 {

constexpr int kRotThreads = 256;
constexpr int kRotCtasPerSm = 4;  // CTAs of the kernel that an SM holds (64 registers a thread)
constexpr int kRotMaxHalf = 256;  // pairs of a head at most (head_dim <= 512)

// One tensor [batch, heads, tokens, D], its last dimension contiguous.
struct RotSeg {
  const char* src;
  char* dst;
  int64_t s_sb, s_sh, s_st;  // element strides of the source
  int64_t d_sb, d_sh, d_st;  // of a dense destination; d_sh alone for a paged one
  int heads;
  int rotate;  // 0: copied
  int paged;   // the destination row: 0 dense, 1 the token's slot of the k pages, 2 of the v pages
};

struct RotArgs {
  RotSeg seg[3];
  int segs;
  int batch, tokens, D;
  const double* inv_freq;  // [half]
  int half, interleaved;
  float scale, sign;       // sign -1: the inverse rotation
  // dense positions: pos[b * pos_sb + t]
  const int64_t* pos;
  int64_t pos_sb;
  // paged: token t < counts[b] (at most `tokens`) of sequence b has position lens[b] - counts[b] + t
  const int32_t* lens;
  const int32_t* counts;   // null: `tokens` for every sequence
  const int32_t* table;
  int64_t table_sb;
  int table_width, page_size, pages;
  int64_t kp_s, vp_s;      // element strides between pages of k and v
  int* status;
  // how the threads of a CTA share the work: `units` threads per row, `groups` teams of them
  // per token (each takes every groups-th head), team_tokens tokens per CTA
  int units, groups, team_tokens;
};

// cos and sin of p * f, |p * f| up to 2^52 or so: quarter turns are taken off in fp64, what is
// left (at most an eighth of a turn) loses 2^-27 half turns to fp32.
__device__ __forceinline__ void rot_cos_sin(double p, double f, float& c, float& s) {
  const double u = p * f * 0.63661977236758134308;  // quarter turns
  const double n = rint(u);
  float sn, cs;
  sincospif(0.5f * static_cast<float>(u - n), &sn, &cs);
  const int k = static_cast<int>(static_cast<long long>(n) & 3);
  c = (k & 1) ? sn : cs;
  s = (k & 1) ? cs : sn;
  if (k == 1 || k == 2) c = -c;
  if (k >= 2) s = -s;
}

// N elements as one access of N * sizeof(T) bytes (a power of two, 16 at most).
template <int BYTES>
struct RotWord;
template <>
struct RotWord<16> { using type = uint4; };
template <>
struct RotWord<8> { using type = uint2; };
template <>
struct RotWord<4> { using type = uint32_t; };
template <>
struct RotWord<2> { using type = uint16_t; };

template <typename T, int VEC>
union RotVec {
  typename RotWord<VEC * int(sizeof(T))>::type word;
  T e[VEC];
  __device__ __forceinline__ RotVec() {}
};

constexpr int kRotAhead = 2;  // rows whose loads a thread issues together

// A thread owns VEC pairs of a token -- their cosines and sines stay in its registers -- and
// walks rows (heads of all tensors, one after another): A.units threads cover a row's pairs,
// A.groups such teams share a token's rows, and a CTA takes A.team_tokens tokens.  Per row and
// thread two vectors of VEC elements are loaded and stored (16 bytes each where sizes and
// alignment allow), the first rows' loads before the angles are formed.  The angles are formed
// once per pair and team instead of once per pair and head, without barrier or shared memory.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotThreads, kRotCtasPerSm) sink_rotate_kernel(const __grid_constant__ RotArgs A) {
  using E = Elem<T>;
  using V = RotVec<T, VEC>;
  using W = typename RotWord<VEC * int(sizeof(T))>::type;
  grid_dependency_wait();
  allow_dependents();
  const int slot_of = int(threadIdx.x) / A.units, unit = int(threadIdx.x) - slot_of * A.units;
  const int token_of = slot_of / A.groups, group = slot_of - token_of * A.groups;
  if (token_of >= A.team_tokens) return;
  const unsigned token = blockIdx.x * unsigned(A.team_tokens) + token_of;  // batch * tokens < 2^31
  if (token >= unsigned(A.batch) * unsigned(A.tokens)) return;
  const int b = int(token / unsigned(A.tokens)), t = int(token - unsigned(b) * unsigned(A.tokens));
  int count = A.tokens;
  if (A.counts != nullptr) count = imax(0, imin(A.counts[b], A.tokens));
  const int rows = A.seg[0].heads + A.seg[1].heads + A.seg[2].heads;  // unused segments have none

  auto segment_of = [&](int r, int& h) {
    int g = 0;
    h = r;
    if (h >= A.seg[0].heads) {
      h -= A.seg[0].heads;
      g = 1;
      if (h >= A.seg[1].heads) {
        h -= A.seg[1].heads;
        g = 2;
      }
    }
    return g;
  };
  // the pair's vectors: VEC elements half apart, or 2 * VEC consecutive ones
  const int o1 = INTERLEAVED ? 2 * VEC * unit : VEC * unit;
  const int o2 = INTERLEAVED ? o1 + VEC : o1 + A.half;
  V x1[kRotAhead], x2[kRotAhead];
  auto load = [&](int r0) {
#pragma unroll
    for (int j = 0; j < kRotAhead; ++j) {
      const int r = r0 + j * A.groups;
      if (r < rows) {
        int h;
        const RotSeg& S = A.seg[segment_of(r, h)];
        const T* src = reinterpret_cast<const T*>(S.src) + b * S.s_sb + t * S.s_st + h * S.s_sh;
        x1[j].word = *reinterpret_cast<const W*>(src + o1);
        x2[j].word = *reinterpret_cast<const W*>(src + o2);
      }
    }
  };
  const bool in_count = t < count;
  if (A.half > 0 && in_count) load(group);

  int64_t p;
  int64_t row_k = 0, row_v = 0;
  bool live = true;
  if (A.pos != nullptr) {
    p = A.pos[b * A.pos_sb + t];
  } else {
    p = int64_t(A.lens[b]) - count + t;
    live = in_count && p >= 0;
    if (live) {
      const int64_t at = p / A.page_size;
      const int page = at < A.table_width ? A.table[b * A.table_sb + at] : -1;
      if (page < 0 || page >= A.pages) {
        atomicOr(A.status, 2);
        live = false;
      } else {
        const int64_t slot = p - at * A.page_size;
        row_k = page * A.kp_s + slot * A.D;
        row_v = page * A.vp_s + slot * A.D;
      }
    }
  }
  auto dest = [&](const RotSeg& S, int h) {
    return reinterpret_cast<T*>(S.dst) +
           (S.paged == 1 ? row_k : S.paged == 2 ? row_v : b * S.d_sb + t * S.d_st) + h * S.d_sh;
  };

  if (A.half > 0) {
    float c[VEC], s[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      rot_cos_sin(static_cast<double>(p), A.inv_freq[unit * VEC + i], c[i], s[i]);
      c[i] *= A.scale;
      s[i] *= A.scale * A.sign;
    }
    for (int r0 = group; r0 < rows; r0 += kRotAhead * A.groups) {
      if (r0 != group && live) load(r0);
#pragma unroll
      for (int j = 0; j < kRotAhead; ++j) {
        const int r = r0 + j * A.groups;
        if (r >= rows) continue;
        int h;
        const RotSeg& S = A.seg[segment_of(r, h)];
        if (!live && S.paged) continue;
        T* dst = dest(S, h);
        V y1, y2;
        if (!live) {
          y1.word = y2.word = W{};
        } else if (S.rotate) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            // elements i of the two vectors, or pair i of their 2 * VEC consecutive ones
            const int k1 = INTERLEAVED ? 2 * i : i, k2 = INTERLEAVED ? 2 * i + 1 : VEC + i;
            const float a = E::to_f(k1 < VEC ? x1[j].e[k1 % VEC] : x2[j].e[k1 % VEC]);
            const float d = E::to_f(k2 < VEC ? x1[j].e[k2 % VEC] : x2[j].e[k2 % VEC]);
            (k1 < VEC ? y1 : y2).e[k1 % VEC] = E::from_f(a * c[i] - d * s[i]);
            (k2 < VEC ? y1 : y2).e[k2 % VEC] = E::from_f(d * c[i] + a * s[i]);
          }
        } else {
          y1.word = x1[j].word;
          y2.word = x2[j].word;
        }
        *reinterpret_cast<W*>(dst + o1) = y1.word;
        *reinterpret_cast<W*>(dst + o2) = y2.word;
      }
    }
  }
  // the dims that pass through
  if (2 * A.half < A.D) {
    for (int r = group; r < rows; r += A.groups) {
      int h;
      const RotSeg& S = A.seg[segment_of(r, h)];
      if (!live && S.paged) continue;
      const T* src = reinterpret_cast<const T*>(S.src) + b * S.s_sb + t * S.s_st + h * S.s_sh;
      T* dst = dest(S, h);
#pragma unroll 4
      for (int o = 2 * A.half + unit * VEC; o < A.D; o += A.units * VEC)
        *reinterpret_cast<W*>(dst + o) = live ? *reinterpret_cast<const W*>(src + o) : W{};
    }
  }
}

}  // namespace sinkb200
