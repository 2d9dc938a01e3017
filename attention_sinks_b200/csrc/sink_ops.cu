// C ABI of the rotation, paged-append and paged-attention operators
// (include/sinkcache_b200.h): argument checks and launches.
#include <climits>
#include <cstring>

#include "../../include/sinkcache_b200.h"
#include "sink_host.h"
#include "sink_paged.cuh"
#include "sink_rotate.cuh"

using namespace sinkb200;

namespace {

int elem_size(int32_t dt) {
  switch (dt) {
    case SINK_DTYPE_F32: return 4;
    case SINK_DTYPE_BF16: return 2;
    case SINK_DTYPE_F16: return 2;
    default: return 0;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int64_t kPagedMaxRows = 1 << 24;  // batch * query heads: row indexes stay in int

constexpr float kLog2e = 1.4426950408889634f;

// Launch with programmatic stream serialization: the kernel's launch overlaps its
// predecessor's tail, and it waits for the predecessor's memory before it touches any.
template <typename... Params, typename... Args>
int32_t launch(void (*kern)(Params...), dim3 grid, int threads, int smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kern, args...);
  if (err != cudaSuccess) return err;
  return counted(cudaGetLastError());
}

// ---------------------------------------------------------------- rotation and append

int32_t check_rotation(const sink_rotation_t* r, int D) {
  if (!r) return SINK_OK;
  if (r->rot_half < 0 || r->rot_half > kRotMaxHalf || 2 * r->rot_half > D) return SINK_EINVAL;
  if (r->rot_half > 0 && !r->inv_freq) return SINK_EINVAL;
  return SINK_OK;
}

void fill_rotation(RotArgs& A, const sink_rotation_t* r) {
  A.scale = A.sign = 1.f;
  if (!r || r->rot_half == 0) return;
  A.inv_freq = r->inv_freq;
  A.half = r->rot_half;
  A.interleaved = r->interleaved ? 1 : 0;
  A.scale = r->scale;
  A.sign = r->inverse ? -1.f : 1.f;
}

// A dense source and destination of the same shape.
int32_t dense_seg(RotSeg& s, const sink_rows_t* x, const sink_rows_t* y, int rotate) {
  if (!x->data || !y->data || x->heads < 1) return SINK_EINVAL;
  if (y->heads != x->heads || y->n != x->n) return SINK_EINVAL;
  if (y->dtype != x->dtype) return SINK_EDTYPE;
  s.src = static_cast<const char*>(x->data);
  s.dst = static_cast<char*>(y->data);
  s.s_sb = x->stride_b;
  s.s_sh = x->stride_h;
  s.s_st = x->stride_t;
  s.d_sb = y->stride_b;
  s.d_sh = y->stride_h;
  s.d_st = y->stride_t;
  s.heads = x->heads;
  s.rotate = rotate;
  s.paged = 0;
  return SINK_OK;
}

// Elements per access: the largest power of two of at most 16 bytes that divides the pairs, the
// head and every stride, and that every base address is aligned to.
int rotate_vector(const RotArgs& A, int es) {
  uint64_t bits = uint64_t(A.half) | uint64_t(A.D);
  uint64_t addr = 0;
  for (int i = 0; i < A.segs; ++i) {
    const RotSeg& s = A.seg[i];
    bits |= uint64_t(s.s_sb) | uint64_t(s.s_sh) | uint64_t(s.s_st) | uint64_t(s.d_sb) | uint64_t(s.d_sh) |
            uint64_t(s.d_st);
    addr |= reinterpret_cast<uintptr_t>(s.src) | reinterpret_cast<uintptr_t>(s.dst);
  }
  bits |= uint64_t(A.kp_s) | uint64_t(A.vp_s);
  int vec = 16 / es;
  while (vec > 1 && ((bits & uint64_t(vec - 1)) || (addr & uint64_t(vec * es - 1)))) vec >>= 1;
  return vec;
}

constexpr int kRotRowsPerThread = 8;

template <typename T, int VEC>
int32_t launch_rotate_v(RotArgs A, int sms, cudaStream_t st) {
  A.units = (A.half > 0 ? A.half : A.D) / VEC;
  if (A.units > kRotThreads) A.units = kRotThreads;
  const int slots = kRotThreads / A.units;
  int heads = 0;
  for (int i = 0; i < A.segs; ++i) heads += A.seg[i].heads;
  // Rows per thread: what fills the device's CTA slots once, so that a small step is one wave
  // with every load in flight, and at most kRotRowsPerThread, so that a large one has waves
  // for the scheduler to even out.
  const int64_t tokens = int64_t(A.batch) * A.tokens;
  const int64_t threads = int64_t(sms) * kRotCtasPerSm * slots;
  int64_t per = (tokens * heads + threads - 1) / threads;
  per = per > kRotRowsPerThread ? kRotRowsPerThread : per;
  int groups = int((heads + per - 1) / per);
  if (groups > slots) groups = slots;
  per = (heads + groups - 1) / groups;
  A.groups = int((heads + per - 1) / per);  // the fewest teams of that many rows
  A.team_tokens = slots / A.groups;
  const dim3 grid(unsigned((tokens + A.team_tokens - 1) / A.team_tokens));
  if (A.interleaved) return launch(sink_rotate_kernel<T, VEC, true>, grid, kRotThreads, 0, st, A);
  return launch(sink_rotate_kernel<T, VEC, false>, grid, kRotThreads, 0, st, A);
}

template <typename T>
int32_t launch_rotate_t(const RotArgs& A, int sms, cudaStream_t st) {
  constexpr int kMax = 16 / int(sizeof(T));
  const int vec = rotate_vector(A, int(sizeof(T)));
  if (vec == kMax) return launch_rotate_v<T, kMax>(A, sms, st);
  if (vec == kMax / 2) return launch_rotate_v<T, kMax / 2>(A, sms, st);
  if constexpr (kMax == 8) {
    if (vec == 2) return launch_rotate_v<T, 2>(A, sms, st);
  }
  return launch_rotate_v<T, 1>(A, sms, st);
}

int32_t launch_rotate(const RotArgs& A, int dtype, cudaStream_t st) {
  if (int64_t(A.batch) * A.tokens > INT_MAX) return SINK_EINVAL;
  int dev = 0;
  const int sms = device_sms(&dev);
  if (sms <= 0) return SINK_EDEVICE;
  switch (dtype) {
    case SINK_DTYPE_BF16: return launch_rotate_t<__nv_bfloat16>(A, sms, st);
    case SINK_DTYPE_F16: return launch_rotate_t<__half>(A, sms, st);
    case SINK_DTYPE_F32: return launch_rotate_t<float>(A, sms, st);
    default: return SINK_EDTYPE;
  }
}

// ---------------------------------------------------------------- paged cache

int32_t check_paged(const sink_paged_kv_t* c) {
  if (!c || !c->k || !c->v || !c->table || !c->lens || !c->status) return SINK_EINVAL;
  if (c->batch < 1 || c->heads_kv < 1 || c->pages < 1 || c->table_width < 1) return SINK_EINVAL;
  if (c->page_size < 1 || int64_t(c->table_width) * c->page_size > INT_MAX) return SINK_EINVAL;
  if (c->table_stride < 0 || c->k_stride_p < 0 || c->k_stride_h < 0 || c->v_stride_p < 0 || c->v_stride_h < 0)
    return SINK_ELAYOUT;
  if (elem_size(c->dtype) == 0) return SINK_EDTYPE;
  if (c->head_dim < 1 || c->head_dim > 2 * kRotMaxHalf) return SINK_EHEADDIM;
  return SINK_OK;
}

template <typename T>
int32_t launch_paged_t(int D, const PagedArgs& A, cudaStream_t st) {
  const dim3 grid(unsigned(A.batch * A.heads_kv));
  if (D == 64) return launch(sink_paged_simple_kernel<T, 64>, grid, 32 * A.group, 0, st, A);
  return launch(sink_paged_simple_kernel<T, 128>, grid, 32 * A.group, 0, st, A);
}

}  // namespace

namespace sinkb200 {

int32_t prepare_paged(int dev) {
  (void)dev;
  return SINK_OK;
}

}  // namespace sinkb200

extern "C" {

int32_t sink_rotary(int32_t batch, int32_t head_dim, const sink_rows_t* q, const sink_rows_t* q_out,
                    const sink_rows_t* k, const sink_rows_t* k_out, const int64_t* positions,
                    int64_t positions_stride_b, const sink_rotation_t* rot, void* stream) {
  if (!q || !q_out || !positions || !rot || (k == nullptr) != (k_out == nullptr)) return SINK_EINVAL;
  if (batch < 1 || q->n < 1) return SINK_EINVAL;
  if (elem_size(q->dtype) == 0) return SINK_EDTYPE;
  if (head_dim < 1 || head_dim > 2 * kRotMaxHalf) return SINK_EHEADDIM;
  int32_t rc = check_rotation(rot, head_dim);
  if (rc) return rc;
  RotArgs A;
  std::memset(&A, 0, sizeof(A));
  if ((rc = dense_seg(A.seg[0], q, q_out, 1))) return rc;
  A.segs = 1;
  if (k) {
    if (k->dtype != q->dtype) return SINK_EDTYPE;
    if (k->n != q->n) return SINK_EINVAL;
    if ((rc = dense_seg(A.seg[1], k, k_out, 1))) return rc;
    A.segs = 2;
  }
  A.batch = batch;
  A.tokens = q->n;
  A.D = head_dim;
  A.pos = positions;
  A.pos_sb = positions_stride_b;
  fill_rotation(A, rot);
  return launch_rotate(A, q->dtype, static_cast<cudaStream_t>(stream));
}

int32_t sink_paged_append(const sink_paged_kv_t* kv, const sink_rows_t* k_new, const sink_rows_t* v_new,
                          const int32_t* counts, const sink_rows_t* q, const sink_rows_t* q_out,
                          const sink_rotation_t* rot, void* stream) {
  int32_t rc = check_paged(kv);
  if (rc) return rc;
  if (!k_new || !v_new || !k_new->data || !v_new->data || (q == nullptr) != (q_out == nullptr)) return SINK_EINVAL;
  if (k_new->dtype != kv->dtype || v_new->dtype != kv->dtype || (q && q->dtype != kv->dtype)) return SINK_EDTYPE;
  if (k_new->heads != kv->heads_kv || v_new->heads != kv->heads_kv) return SINK_EINVAL;
  if (k_new->n < 1 || v_new->n != k_new->n || (q && q->n != k_new->n)) return SINK_EINVAL;
  if ((rc = check_rotation(rot, kv->head_dim))) return rc;
  RotArgs A;
  std::memset(&A, 0, sizeof(A));
  const sink_rows_t* rows[2] = {k_new, v_new};
  for (int i = 0; i < 2; ++i) {
    RotSeg& s = A.seg[i];
    s.src = static_cast<const char*>(rows[i]->data);
    s.dst = static_cast<char*>(i ? kv->v : kv->k);
    s.s_sb = rows[i]->stride_b;
    s.s_sh = rows[i]->stride_h;
    s.s_st = rows[i]->stride_t;
    s.d_sh = i ? kv->v_stride_h : kv->k_stride_h;
    s.heads = kv->heads_kv;
    s.rotate = i == 0;
    s.paged = i + 1;
  }
  A.segs = 2;
  if (q) {
    if ((rc = dense_seg(A.seg[2], q, q_out, 1))) return rc;
    A.segs = 3;
  }
  A.batch = kv->batch;
  A.tokens = k_new->n;
  A.D = kv->head_dim;
  A.lens = kv->lens;
  A.counts = counts;
  A.table = kv->table;
  A.table_sb = kv->table_stride;
  A.table_width = kv->table_width;
  A.page_size = kv->page_size;
  A.pages = kv->pages;
  A.kp_s = kv->k_stride_p;
  A.vp_s = kv->v_stride_p;
  A.status = kv->status;
  fill_rotation(A, rot);
  return launch_rotate(A, kv->dtype, static_cast<cudaStream_t>(stream));
}

int32_t sink_paged_attention(const sink_rows_t* q, const sink_paged_kv_t* kv, int32_t shared_len, float scale,
                             void* out, int64_t out_stride_b, int64_t out_stride_h, void* workspace,
                             size_t workspace_bytes, void* stream) {
  int32_t rc = check_paged(kv);
  if (rc) return rc;
  if (!q || !q->data || !out || q->n != 1) return SINK_EINVAL;
  const int32_t D = kv->head_dim, page = kv->page_size;
  if (kv->dtype != SINK_DTYPE_BF16 && kv->dtype != SINK_DTYPE_F16) return SINK_EDTYPE;
  if (q->dtype != kv->dtype) return SINK_EDTYPE;
  if (D != 64 && D != 128) return SINK_EHEADDIM;
  if (q->heads < kv->heads_kv || q->heads % kv->heads_kv || q->heads / kv->heads_kv > 8) return SINK_EGROUP;
  if (page != 16 && page != 32 && page != 64 && page != 128) return SINK_EINVAL;
  if (shared_len < 0 || shared_len % page || shared_len > kv->table_width * page) return SINK_EINVAL;
  if (int64_t(kv->batch) * q->heads > kPagedMaxRows) return SINK_EINVAL;
  // tiled copies: page, head and query rows on 16-byte boundaries (strides of 8 elements)
  if (!aligned16(kv->k) || !aligned16(kv->v) || !aligned16(q->data)) return SINK_ELAYOUT;
  if ((kv->k_stride_p | kv->k_stride_h | kv->v_stride_p | kv->v_stride_h | q->stride_b | q->stride_h) & 7)
    return SINK_ELAYOUT;
  if (!workspace || workspace_bytes < 256 || !aligned16(workspace)) return SINK_EWORKSPACE;
  int dev = 0;
  const int sms = device_sms(&dev);
  if (sms <= 0) return SINK_EDEVICE;
  if (workspace_bytes < sink_paged_workspace_bytes(kv->batch, kv->heads_kv, q->heads, D, shared_len, sms))
    return SINK_EWORKSPACE;
  PagedArgs A;
  std::memset(&A, 0, sizeof(A));
  A.k = static_cast<const char*>(kv->k);
  A.v = static_cast<const char*>(kv->v);
  A.table = kv->table;
  A.lens = kv->lens;
  A.status = kv->status;
  A.q = static_cast<const char*>(q->data);
  A.out = static_cast<char*>(out);
  A.table_sb = kv->table_stride;
  A.k_sp = kv->k_stride_p;
  A.k_sh = kv->k_stride_h;
  A.v_sp = kv->v_stride_p;
  A.v_sh = kv->v_stride_h;
  A.q_sb = q->stride_b;
  A.q_sh = q->stride_h;
  A.o_sb = out_stride_b;
  A.o_sh = out_stride_h;
  A.batch = kv->batch;
  A.heads_kv = kv->heads_kv;
  A.group = q->heads / kv->heads_kv;
  A.page_size = page;
  A.pages = kv->pages;
  A.table_width = kv->table_width;
  A.shared = shared_len;
  A.scale_log2 = scale * kLog2e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return kv->dtype == SINK_DTYPE_BF16 ? launch_paged_t<__nv_bfloat16>(D, A, st) : launch_paged_t<__half>(D, A, st);
}

size_t sink_paged_workspace_bytes(int32_t batch, int32_t heads_kv, int32_t heads_q, int32_t head_dim,
                                  int32_t shared_len, int32_t num_sms) {
  (void)shared_len;
  if (batch < 1 || heads_kv < 1 || heads_q < heads_kv || heads_q % heads_kv || heads_q / heads_kv > 8) return 0;
  if ((head_dim != 64 && head_dim != 128) || num_sms < 1 || shared_len < 0) return 0;
  if (int64_t(batch) * heads_q > kPagedMaxRows) return 0;
  return 256;
}

}  // extern "C"
