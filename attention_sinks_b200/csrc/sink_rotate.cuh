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
// Bound: memory (every element read once and written once).
#pragma once

#include "sink_common.cuh"

namespace sinkb200 {

constexpr int kRotThreads = 256;
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
  // paged: token t of sequence b has position lens[b] - counts[b] + t (t < counts[b] <= tokens)
  const int32_t* lens;
  const int32_t* counts;   // null: `tokens` for every sequence
  const int32_t* table;
  int64_t table_sb;
  int table_width, page_size, pages;
  int64_t kp_s, vp_s;      // element strides between pages of k and v
  int* status;
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

// One CTA per token: the angles' cos and sin once for all heads, then the heads' elements.
template <typename T>
__global__ void __launch_bounds__(kRotThreads) sink_rotate_kernel(const RotArgs A) {
  using E = Elem<T>;
  __shared__ float2 cs[kRotMaxHalf];
  grid_dependency_wait();
  allow_dependents();
  const int b = int(blockIdx.x) / A.tokens, t = int(blockIdx.x) - b * A.tokens;
  int64_t p;
  int64_t row_k = 0, row_v = 0;
  bool live = true;
  if (A.pos != nullptr) {
    p = A.pos[b * A.pos_sb + t];
  } else {
    const int n = A.counts != nullptr ? A.counts[b] : A.tokens;
    p = int64_t(A.lens[b]) - n + t;
    live = t < n && p >= 0;
    if (live) {
      const int64_t at = p / A.page_size;
      const int page = at < A.table_width ? A.table[b * A.table_sb + at] : -1;
      if (page < 0 || page >= A.pages) {
        if (threadIdx.x == 0) atomicOr(A.status, 2);
        live = false;
      } else {
        const int64_t slot = p - at * A.page_size;
        row_k = page * A.kp_s + slot * A.D;
        row_v = page * A.vp_s + slot * A.D;
      }
    }
  }
  for (int i = threadIdx.x; i < A.half; i += kRotThreads) {
    float c, s;
    rot_cos_sin(static_cast<double>(p), A.inv_freq[i], c, s);
    cs[i] = make_float2(c * A.scale, s * A.scale * A.sign);
  }
  __syncthreads();
  for (int g = 0; g < A.segs; ++g) {
    const RotSeg& S = A.seg[g];
    if (!live && S.paged) continue;
    const T* src = reinterpret_cast<const T*>(S.src) + b * S.s_sb + t * S.s_st;
    T* dst = reinterpret_cast<T*>(S.dst) + (S.paged == 1 ? row_k : S.paged == 2 ? row_v : b * S.d_sb + t * S.d_st);
    const int half = S.rotate ? A.half : 0;
    const int per_row = A.D - half;  // a pair or a lone element each
    for (int i = threadIdx.x; i < S.heads * per_row; i += kRotThreads) {
      const int h = i / per_row, c = i - h * per_row;
      const T* x = src + h * S.s_sh;
      T* y = dst + h * S.d_sh;
      if (c < half) {
        const int i1 = A.interleaved ? 2 * c : c, i2 = A.interleaved ? 2 * c + 1 : c + half;
        const float x1 = E::to_f(x[i1]), x2 = E::to_f(x[i2]);
        const float2 w = cs[c];
        y[i1] = E::from_f(live ? x1 * w.x - x2 * w.y : 0.f);
        y[i2] = E::from_f(live ? x2 * w.x + x1 * w.y : 0.f);
      } else {
        y[c + half] = live ? x[c + half] : E::from_f(0.f);
      }
    }
  }
}

}  // namespace sinkb200
