// Decode attention over a paged cache whose sequences may share their first pages.
//
//   out[b, h] = sum_j softmax_j(scale q[b, h] . K_j) V_j   over the rows j < lens[b].
#pragma once

#include "sink_chunk.cuh"

namespace sinkb200 {

struct PagedArgs {
  const char* k;
  const char* v;
  const int32_t* table;
  const int32_t* lens;
  int* status;
  const char* q;
  char* out;
  int64_t table_sb, k_sp, k_sh, v_sp, v_sh, q_sb, q_sh, o_sb, o_sh;
  int batch, heads_kv, group, page_size, pages, table_width, shared;
  float scale_log2;
};

// One warp per query row, keys one after another.
template <typename T, int D>
__global__ void __launch_bounds__(256) sink_paged_simple_kernel(const PagedArgs A) {
  using E = Elem<T>;
  grid_dependency_wait();
  const int b = int(blockIdx.x) / A.heads_kv, h = int(blockIdx.x) - b * A.heads_kv;
  const int g = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int N = D / 32;
  const T* q = reinterpret_cast<const T*>(A.q) + b * A.q_sb + (h * A.group + g) * A.q_sh;
  float x[N], o[N], m = kNegInf, l = 0.f;
  for (int i = 0; i < N; ++i) {
    x[i] = E::to_f(q[lane * N + i]) * A.scale_log2;
    o[i] = 0.f;
  }
  int n = A.lens[b];
  if (n > A.table_width * A.page_size) {
    n = A.table_width * A.page_size;
    if (threadIdx.x == 0) atomicOr(A.status, 2);
  }
  for (int j = 0; j < n; ++j) {
    const int page = A.table[(j < A.shared ? 0 : b * A.table_sb) + j / A.page_size];
    if (page < 0 || page >= A.pages) {
      if (threadIdx.x == 0) atomicOr(A.status, 2);
      continue;
    }
    const int slot = j % A.page_size;
    const T* k = reinterpret_cast<const T*>(A.k) + page * A.k_sp + h * A.k_sh + slot * D + lane * N;
    const T* v = reinterpret_cast<const T*>(A.v) + page * A.v_sp + h * A.v_sh + slot * D + lane * N;
    float s = 0.f;
    for (int i = 0; i < N; ++i) s += x[i] * E::to_f(k[i]);
    for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(kFull, s, off);
    const float mn = fmaxf(m, s), a = exp2f(m - mn), p = exp2f(s - mn);
    m = mn;
    l = l * a + p;
    for (int i = 0; i < N; ++i) o[i] = o[i] * a + p * E::to_f(v[i]);
  }
  T* out = reinterpret_cast<T*>(A.out) + b * A.o_sb + (h * A.group + g) * A.o_sh;
  for (int i = 0; i < N; ++i) out[lane * N + i] = E::from_f(l > 0.f ? o[i] / l : 0.f);
}

}  // namespace sinkb200
