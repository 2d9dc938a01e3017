// C ABI of the rotation, paged-append and paged-attention operators
// (include/sinkcache_b200.h): argument checks and launches.
#include <atomic>
#include <climits>
#include <cmath>
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
constexpr int64_t kPagedMaxChunks = 1 << 22;  // batch * kv heads * chunks of a table's row, per SM: the
                                              // cost of a CTA's part stays below 2^29 (PagedWalk)

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

// (Measured at 8 x 2048 tokens of 24 heads, forward and backward: 2 rows 118 us, 4 87, 8 79, 12 76,
// 16 and more 76; a ragged append of 8 x 4096 tokens: 98, 69, 56, 52, then 55-58.)
constexpr int kRotRowsPerThread = 12;

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

// Workspace of one attention call.
struct PagedPlan {
  int per_tile = 0, tiles = 0;
  int units = 0;  // of the prefix
  size_t o_prefix = 0, ml_prefix = 0, o_own = 0, ml_own = 0, bounds = 0, total = 0;
};

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Weights of a combine CTA: a float per query row and partial (two streams of the prefix pieces
// and of the own pieces, at most one of each per CTA of the attention).
size_t combine_smem(int sms, int G) { return size_t(4) * sms * G * 4; }

bool plan_paged(int64_t batch, int heads_kv, int heads_q, int D, int64_t shared, int sms, PagedPlan& p) {
  if (batch < 1 || heads_kv < 1 || heads_q < heads_kv || heads_q % heads_kv || heads_q / heads_kv > 8) return false;
  if ((D != 64 && D != 128) || shared < 0 || sms < 1 || combine_smem(sms, 8) > 48 * 1024) return false;
  if (batch * heads_q > kPagedMaxRows) return false;
  const int G = heads_q / heads_kv;
  p.per_tile = int(batch < kPgTile / G ? batch : kPgTile / G);
  p.tiles = int((batch + p.per_tile - 1) / p.per_tile);
  // a piece of CTA c and unit u has slot c + u, with a partial for each of the two streams
  p.units = shared > 0 ? heads_kv * ((p.tiles + 1) / 2) : 0;
  const size_t slots_p = shared > 0 ? size_t(sms) + p.units : 0;
  const size_t slots_o = size_t(sms) + size_t(batch) * heads_kv;
  size_t off = 0;
  p.o_prefix = off;
  off += align256(slots_p * 2 * kPgTile * D * 4);
  p.ml_prefix = off;
  off += align256(slots_p * 2 * kPgTile * 8);
  p.o_own = off;
  off += align256(slots_o * 2 * G * D * 4);
  p.ml_own = off;
  off += align256(slots_o * 2 * G * 8);
  p.bounds = off;
  off += align256((size_t(p.units) + size_t(batch) * heads_kv) * 8);
  p.total = off;
  return true;
}

int32_t encode(CUtensorMap* map, int32_t dtype, int rank, const void* data, const cuuint64_t* dims,
               const cuuint64_t* strides, const cuuint32_t* box) {
  auto f = tensor_map_encoder();
  if (f == nullptr) return SINK_EDEVICE;
  const cuuint32_t unit[4] = {1, 1, 1, 1};
  const CUresult r = f(map, dtype == SINK_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                     : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                       cuuint32_t(rank), const_cast<void*>(data), dims, strides, box, unit,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? SINK_OK : SINK_ELAYOUT;
}

// A pool [pages, Hkv, page_size, D], boxes of 64 columns of one page.
int32_t encode_pool(CUtensorMap* map, const void* data, const sink_paged_kv_t* c, int64_t stride_p, int64_t stride_h) {
  const cuuint64_t row = cuuint64_t(c->head_dim) * 2;
  const cuuint64_t sh = c->heads_kv > 1 ? cuuint64_t(stride_h) * 2 : row * c->page_size;
  const cuuint64_t sp = c->pages > 1 ? cuuint64_t(stride_p) * 2 : sh * c->heads_kv;
  const cuuint64_t dims[4] = {cuuint64_t(c->head_dim), cuuint64_t(c->page_size), cuuint64_t(c->heads_kv),
                              cuuint64_t(c->pages)};
  const cuuint64_t strides[3] = {row, sh, sp};
  const cuuint32_t box[4] = {64, cuuint32_t(c->page_size), 1, 1};
  return encode(map, c->dtype, 4, data, dims, strides, box);
}

// Queries [B, Hq, D], boxes of 64 columns x G heads x `seqs` sequences.
int32_t encode_query(CUtensorMap* map, const sink_rows_t* q, int batch, int D, int G, int seqs) {
  const cuuint64_t sh = q->heads > 1 ? cuuint64_t(q->stride_h) * 2 : cuuint64_t(D) * 2;
  const cuuint64_t sb = batch > 1 ? cuuint64_t(q->stride_b) * 2 : sh * q->heads;
  const cuuint64_t dims[3] = {cuuint64_t(D), cuuint64_t(q->heads), cuuint64_t(batch)};
  const cuuint64_t strides[2] = {sh, sb};
  const cuuint32_t box[3] = {64, cuuint32_t(G), cuuint32_t(seqs)};
  return encode(map, q->dtype, 3, q->data, dims, strides, box);
}

template <typename T, int D>
int32_t launch_paged_d(const PagedArgs& A, cudaStream_t st) {
  const int32_t rc = launch(sink_paged_kernel<T, D>, dim3(unsigned(A.ctas)), kPgThreads, PgGeom<D>::kSmem, st, A);
  if (rc) return rc;
  return launch(sink_paged_combine_kernel<T, D>, dim3(unsigned(A.batch * A.heads_kv)), kPgCombineThreads,
                int(combine_smem(A.ctas, A.group)), st, A);
}

template <typename T>
int32_t launch_paged_t(int D, const PagedArgs& A, cudaStream_t st) {
  return D == 64 ? launch_paged_d<T, 64>(A, st) : launch_paged_d<T, 128>(A, st);
}

template <typename T>
cudaError_t allow_paged_smem() {
  cudaError_t e = cudaFuncSetAttribute(sink_paged_kernel<T, 64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       PgGeom<64>::kSmem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(sink_paged_kernel<T, 128>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             PgGeom<128>::kSmem);
  return e;
}

}  // namespace

namespace sinkb200 {

int32_t prepare_paged(int dev) {
  static std::atomic<uint64_t> done{0};  // one bit per device
  const uint64_t bit = uint64_t(1) << dev;
  if (done.load(std::memory_order_acquire) & bit) return SINK_OK;
  cudaError_t e = allow_paged_smem<__nv_bfloat16>();
  if (e == cudaSuccess) e = allow_paged_smem<__half>();
  if (e != cudaSuccess) return e;
  if (tensor_map_encoder() == nullptr) return SINK_EDEVICE;
  done.fetch_or(bit, std::memory_order_acq_rel);
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
  const bool q_rows = (q->heads == 1 || q->stride_h >= D) && (kv->batch == 1 || q->stride_b >= D);
  const bool k_rows = (kv->heads_kv == 1 || (kv->k_stride_h >= D && kv->v_stride_h >= D)) &&
                      (kv->pages == 1 || (kv->k_stride_p >= D && kv->v_stride_p >= D));
  if (!q_rows || !k_rows) return SINK_ELAYOUT;
  if (!std::isfinite(scale)) return SINK_EINVAL;
  // a sequence's rows, rounded up to a chunk, and the chunks of all sequences together stay in int
  if (int64_t(kv->table_width) * page > INT_MAX - kPgKeys) return SINK_EINVAL;
  const int64_t chunks = int64_t(kv->batch) * ((int64_t(kv->table_width) * page + kPgKeys - 1) / kPgKeys);
  if (chunks > INT_MAX) return SINK_EINVAL;
  if (!workspace || workspace_bytes < 256 || !aligned16(workspace)) return SINK_EWORKSPACE;
  int dev = 0;
  const int sms = device_sms(&dev);
  if (sms <= 0) return SINK_EDEVICE;
  if (chunks * kv->heads_kv > sms * kPagedMaxChunks) return SINK_EINVAL;
  PagedPlan plan;
  if (!plan_paged(kv->batch, kv->heads_kv, q->heads, D, shared_len, sms, plan)) return SINK_EINVAL;
  if (workspace_bytes < plan.total) return SINK_EWORKSPACE;
  if ((rc = prepare_paged(dev))) return rc;
  PagedArgs A;
  std::memset(&A, 0, sizeof(A));
  A.group = q->heads / kv->heads_kv;
  if ((rc = encode_pool(&A.kmap, kv->k, kv, kv->k_stride_p, kv->k_stride_h))) return rc;
  if ((rc = encode_pool(&A.vmap, kv->v, kv, kv->v_stride_p, kv->v_stride_h))) return rc;
  if ((rc = encode_query(&A.qtile, q, kv->batch, D, A.group, plan.per_tile))) return rc;
  if ((rc = encode_query(&A.qgroup, q, kv->batch, D, A.group, 1))) return rc;
  A.table = kv->table;
  A.lens = kv->lens;
  A.status = kv->status;
  A.out = static_cast<char*>(out);
  A.v = static_cast<const char*>(kv->v);
  A.v_sp = kv->v_stride_p;
  A.v_sh = kv->v_stride_h;
  A.table_sb = kv->table_stride;
  A.o_sb = out_stride_b;
  A.o_sh = out_stride_h;
  char* ws = static_cast<char*>(workspace);
  A.o_prefix = reinterpret_cast<float*>(ws + plan.o_prefix);
  A.ml_prefix = reinterpret_cast<float2*>(ws + plan.ml_prefix);
  A.o_own = reinterpret_cast<float*>(ws + plan.o_own);
  A.ml_own = reinterpret_cast<float2*>(ws + plan.ml_own);
  A.bounds = reinterpret_cast<int2*>(ws + plan.bounds);
  A.units = plan.units;
  A.batch = kv->batch;
  A.heads_kv = kv->heads_kv;
  A.page_size = page;
  A.pages = kv->pages;
  A.table_width = kv->table_width;
  A.shared = shared_len;
  A.per_tile = plan.per_tile;
  A.tiles = plan.tiles;
  A.ctas = sms;
  A.negate = scale < 0.f;
  const int64_t inject = take_fail_next_wait();
  A.wait_polls = inject < 0 ? kWaitPolls : int(inject & 0x7fffffff);
  A.skip_tile = inject < 0 ? -1 : int(inject >> 32);
  // a scale of 0 (uniform weights) becomes the smallest normal number, so that a masked score
  // of -infinity stays one
  A.scale_log2 = std::fmax(std::fabs(scale) * kLog2e, 1.17549435e-38f);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return kv->dtype == SINK_DTYPE_BF16 ? launch_paged_t<__nv_bfloat16>(D, A, st)
                                      : launch_paged_t<__half>(D, A, st);
}

size_t sink_paged_workspace_bytes(int32_t batch, int32_t heads_kv, int32_t heads_q, int32_t head_dim,
                                  int32_t shared_len, int32_t num_sms) {
  PagedPlan plan;
  return plan_paged(batch, heads_kv, heads_q, head_dim, shared_len, num_sms, plan) ? plan.total : 0;
}

}  // extern "C"
