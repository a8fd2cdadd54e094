// fa_qk_norm_rotary and its backward: norm and rotation of every head of q and k in one pass (formulas in fa_norm.h), where elementwise
// operations read and write the tensors several times over.
//   backward, with g = R_t^T dy, xh = x r:   dx = r (g w - xh mean(g w xh)),   dw = sum over rows and heads of g xh
// HBM-bound both ways: forward one read and one write of q and k, backward two reads (the gradient and x, whose norm is formed again: cheaper than
// another tensor of them) and one write.
//
// A thread owns one 16-byte place (head, chunk) of a row and walks rows with it, so that the divisions that find the place are made once
// (as in fa_rotary.hip); workgroups hold whole rows where a row is at most 512 threads wide.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/flash_attn_gfx950.h"
#include "fa_check.h"
#include "fa_norm.h"
#include "fa_paged_index.h"

namespace fa {

namespace {

struct NormPart {
  const void* x;
  const void* dy;  // backward
  void* out;       // y, or dx
  const void* w;
  void* dw;
  int64_t x_rs, x_hs, dy_rs, dy_hs, out_rs, out_hs;  // elements
  int heads;
  int per_row;         // threads of a row
  int threads;         // threads of the part's workgroups that work: the rows of a workgroup times per_row, or a piece of a row
  int rows_per_group;  // rows that a workgroup takes at a time
  int pieces;          // workgroups of a row
  int blocks;          // of the part
  int first_block;
};

struct NormParams {
  NormPart part[2];
  const void* cos;
  const void* sin;
  const int32_t* positions;
  const int32_t* rows_end;  // null, or where the rows that count end
  int n_rows, seqlen, table_rows;
  float eps;
  int w_fp32;
  int rows;        // in flight
  float* partial;  // backward: [blocks of both parts][D] sums of the weights' gradients
};

template <typename T>
struct Turned {  // a row's cos and sin values for one chunk
  typename Elem<T>::vec4 c, s;
  FA_DEVICE void load(const NormParams& p, int row, int ch, int half) {
    int t = p.positions ? p.positions[row] : (int)((unsigned)row % (unsigned)p.seqlen);
    t = table_row(t, p.table_rows);
    const int64_t at = (int64_t)t * half + ch * 4;
    c = *reinterpret_cast<const typename Elem<T>::vec4*>(reinterpret_cast<const T*>(p.cos) + at);
    s = *reinterpret_cast<const typename Elem<T>::vec4*>(reinterpret_cast<const T*>(p.sin) + at);
  }
};

template <typename V>
FA_DEVICE void to_float(V v, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] = (float)v[i];
}
template <typename T>
FA_DEVICE typename Elem<T>::vec8 to_elem(const float (&x)[8]) {
  typename Elem<T>::vec8 v;
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = (T)x[i];
  return v;
}

// Rows a thread of the forward has in flight: one where there are few, whose time is a chain of latencies.
constexpr int kNormRows = 4;
inline int norm_rows(int64_t n_rows, int heads, int D) { return n_rows * heads * (D / 8) <= 256 * 1024 ? 1 : kNormRows; }

struct Place {  // of a thread in its part
  int row0, step, head, ch;
  bool on;
};
FA_DEVICE int rows_of(const NormParams& p) { return p.rows_end ? keys_in_reach(*p.rows_end, p.n_rows) : p.n_rows; }
template <int CH>
FA_DEVICE Place place_of(const NormPart& q, int block) {
  const int tid = threadIdx.x;
  const int group = block / q.pieces, piece = block - group * q.pieces;
  const int j0 = piece * (int)blockDim.x + tid;
  const int local = j0 / q.per_row, j = j0 - local * q.per_row;
  Place pl;
  pl.on = q.pieces == 1 ? tid < q.threads : j0 < q.per_row;
  pl.row0 = group * q.rows_per_group + local;
  pl.step = q.blocks / q.pieces * q.rows_per_group;
  pl.head = j / CH;
  pl.ch = j % CH;
  return pl;
}

template <typename T, int D, bool kTurn, int kRows>
__global__ void __launch_bounds__(512) qk_norm_rotary_kernel(const NormParams p) {
  constexpr int CH = D / 8;
  const bool second = (int)blockIdx.x >= p.part[1].first_block;
  const NormPart& q = p.part[second];
  const Place pl = place_of<CH>(q, (int)blockIdx.x - q.first_block);
  if (!pl.on) return;
  const int n_rows = rows_of(p);
  float w[8];
  load_weights<T>(q.w, p.w_fp32 != 0, pl.ch, w);
  const T* const src = reinterpret_cast<const T*>(q.x) + (int64_t)pl.head * q.x_hs + pl.ch * 8;
  T* const dst = reinterpret_cast<T*>(q.out) + (int64_t)pl.head * q.out_hs + pl.ch * 8;
  for (int64_t row0 = pl.row0; row0 < n_rows; row0 += (int64_t)kRows * pl.step) {
    typename Elem<T>::vec8 v[kRows];
    Turned<T> t[kRows];
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      const int64_t row = row0 + (int64_t)i * pl.step;
      if (row < n_rows) {
        v[i] = bitcast<typename Elem<T>::vec8>(ld_global16(src + row * q.x_rs));
        if (kTurn) t[i].load(p, (int)row, pl.ch, D / 2);
      }
    }
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      const int64_t row = row0 + (int64_t)i * pl.step;
      if (row < n_rows) {
        float x[8];
        to_float(v[i], x);
        const float r = inverse_rms<CH>(x, p.eps);
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = x[k] * r * w[k];
        if (kTurn) turn(x, t[i].c, t[i].s);
        st_global16(dst + row * q.out_rs, bitcast<u32x4>(to_elem<T>(x)));
      }
    }
  }
}

// The rows that a thread of the backward has in flight: two tensors of them.
constexpr int kNormBwdRows = 2;

template <typename T, int D, bool kTurn>
__global__ void __launch_bounds__(512) qk_norm_rotary_bwd_kernel(const NormParams p) {
  constexpr int CH = D / 8;
  __shared__ float sums[512 * 9];  // (a thread's eight, padded: neighbouring threads' lie in different banks)
  const bool second = (int)blockIdx.x >= p.part[1].first_block;
  const NormPart& q = p.part[second];
  const Place pl = place_of<CH>(q, (int)blockIdx.x - q.first_block);
  float dw[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (pl.on) {
    const int n_rows = rows_of(p);
    float w[8];
    load_weights<T>(q.w, p.w_fp32 != 0, pl.ch, w);
    const T* const xs = reinterpret_cast<const T*>(q.x) + (int64_t)pl.head * q.x_hs + pl.ch * 8;
    const T* const gs = reinterpret_cast<const T*>(q.dy) + (int64_t)pl.head * q.dy_hs + pl.ch * 8;
    T* const dst = reinterpret_cast<T*>(q.out) + (int64_t)pl.head * q.out_hs + pl.ch * 8;
    for (int64_t row0 = pl.row0; row0 < n_rows; row0 += (int64_t)kNormBwdRows * pl.step) {
      typename Elem<T>::vec8 vx[kNormBwdRows], vg[kNormBwdRows];
      Turned<T> t[kNormBwdRows];
#pragma unroll
      for (int i = 0; i < kNormBwdRows; i++) {
        const int64_t row = row0 + (int64_t)i * pl.step;
        if (row < n_rows) {
          vx[i] = bitcast<typename Elem<T>::vec8>(ld_global16(xs + row * q.x_rs));
          vg[i] = bitcast<typename Elem<T>::vec8>(ld_global16(gs + row * q.dy_rs));
          if (kTurn) t[i].load(p, (int)row, pl.ch, D / 2);
        }
      }
#pragma unroll
      for (int i = 0; i < kNormBwdRows; i++) {
        const int64_t row = row0 + (int64_t)i * pl.step;
        if (row < n_rows) {
          float x[8], g[8];
          to_float(vx[i], x);
          to_float(vg[i], g);
          const float r = inverse_rms<CH>(x, p.eps);
          if (kTurn) turn_back(g, t[i].c, t[i].s);
          float m = 0.f;
#pragma unroll
          for (int k = 0; k < 8; k++) {
            x[k] *= r;
            dw[k] = __builtin_fmaf(g[k], x[k], dw[k]);
            g[k] *= w[k];
            m = __builtin_fmaf(g[k], x[k], m);
          }
          m = vector_sum<CH>(m) * (1.f / D);
#pragma unroll
          for (int k = 0; k < 8; k++) x[k] = r * (g[k] - x[k] * m);
          st_global16(dst + row * q.out_rs, bitcast<u32x4>(to_elem<T>(x)));
        }
      }
    }
  }
  // the workgroup's sums: element e of every thread whose chunk holds it, in the threads' order
#pragma unroll
  for (int k = 0; k < 8; k++) sums[threadIdx.x * 9 + k] = dw[k];
  __syncthreads();
  for (int e = threadIdx.x; e < D; e += blockDim.x) {
    float s = 0.f;
    for (int j = e / 8; j < (int)blockDim.x; j += CH) s += sums[j * 9 + e % 8];
    p.partial[(int64_t)blockIdx.x * D + e] = s;
  }
}

// The workgroups' sums added up: a workgroup for 16 weights of one part, 64 rows of 16 lanes, joined in LDS.  A fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) norm_weights_kernel(const NormParams p, int D) {
  __shared__ float sums[1024];
  const int cols = D / 16;
  const NormPart& q = p.part[(int)blockIdx.x / cols];
  const int col = (int)blockIdx.x % cols * 16 + (threadIdx.x & 15);
  const float* const from = p.partial + (int64_t)q.first_block * D + col;
  float s = 0.f;
#pragma unroll 4
  for (int b = threadIdx.x >> 4; b < q.blocks; b += 64) s += from[(int64_t)b * D];
  sums[threadIdx.x] = s;
  __syncthreads();
  for (int half = 512; half >= 16; half >>= 1) {
    if ((int)threadIdx.x < half) sums[threadIdx.x] += sums[threadIdx.x + half];
    __syncthreads();
  }
  if (threadIdx.x < 16) {
    s = sums[threadIdx.x];
    if (p.w_fp32) reinterpret_cast<float*>(q.dw)[col] = s;
    else reinterpret_cast<T*>(q.dw)[col] = (T)s;
  }
}

// How the launches are cut.  The workgroups of both parts, shared by their sizes, walk on over the rows: as many as give a compute unit about 20 waves in the
// forward and 16 in the backward (whose workgroups each leave a row of sums, too).  us of the forward with four workgroups a compute unit whatever their size / so: 32768
// rows of 16 + 4 heads, d = 128 71.6 / 67.9 (a workgroup for every four rows 85.8; as it is now 63, 5.4 TB/s), 16000 of 32 + 8 (eight waves a workgroup) 91 / 77, 65536 of 2 x 12,
// d = 64 86.5 / 78.4, 24000 of 2 x 12 63 / 55; with 24 waves 69.8, -, 77.5, 53.8.  Backward, 16 waves / 20: 64000 rows of 2 x 8 heads, d = 32 48 / 63, 11200 of
// 2 x 20, d = 128 74 / 100, 48000 of 24 + 8, d = 64 118 / 141, the others alike.
constexpr int kForwardWaves = 20, kBackwardWaves = 16;

void cut(NormPart* part, int heads, int D, int n_rows, int rows_in_flight, int most_blocks, int first_block) {
  part->heads = heads;
  part->per_row = heads * (D / 8);
  part->first_block = first_block;
  part->blocks = 0;
  part->pieces = part->rows_per_group = 1;
  part->threads = 0;
  if (heads == 0 || n_rows == 0) return;
  if (part->per_row <= 512) {
    part->rows_per_group = part->per_row >= 256 ? 1 : 256 / part->per_row;
    part->threads = part->rows_per_group * part->per_row;
  } else {
    part->pieces = (part->per_row + 255) / 256;
  }
  const int64_t groups = ((int64_t)n_rows + part->rows_per_group - 1) / part->rows_per_group;
  int64_t n = (groups + rows_in_flight - 1) / rows_in_flight;
  if (most_blocks > 0) n = std::min<int64_t>(n, std::max(1, most_blocks / part->pieces));
  part->blocks = (int)(n * part->pieces);
}

int block_threads(const NormParams& p) {
  int t = 64;
  for (const NormPart& q : p.part) t = std::max(t, q.pieces > 1 ? 256 : (q.threads + 63) / 64 * 64);
  return t;
}

int cut_parts(NormParams* p, const fa_qk_norm_args* a, bool bwd) {
  const int n = (int)a->n_rows, D = a->head_dim, all = std::max(1, a->nheads_q + a->nheads_k);
  // (pieces of a row are 256 threads wide: parts that share a launch with a wider one keep to rows of their own)
  const int per_row = std::max(1, std::max(a->nheads_q, a->nheads_k) * (D / 8));
  const int threads = per_row > 512 ? 256 : (per_row >= 256 ? 1 : 256 / per_row) * per_row;
  const int64_t most = walking_workgroups((threads + 63) / 64, bwd ? kBackwardWaves : kForwardWaves);
  const int64_t q_share = std::max<int64_t>(1, most * a->nheads_q / all), k_share = std::max<int64_t>(1, most * a->nheads_k / all);
  const int rows = bwd ? kNormBwdRows : norm_rows(n, all, D);
  cut(&p->part[0], a->nheads_q, D, n, rows, (int)q_share, 0);
  cut(&p->part[1], a->nheads_k, D, n, rows, (int)k_share, p->part[0].blocks);
  p->rows = rows;
  return p->part[0].blocks + p->part[1].blocks;
}

int check_sizes(const fa_qk_norm_args* a, const char* name) {
  FA_REQUIRE(a && a->struct_bytes == sizeof(fa_qk_norm_args), "%s: struct size mismatch", name);
  FA_REQUIRE(a->dtype == FA_FP16 || a->dtype == FA_BF16, "%s: dtype must be fp16 or bf16", name);
  FA_REQUIRE(a->weight_dtype == a->dtype || a->weight_dtype == FA_FP32, "%s: weights must be of the tensors' dtype or fp32", name);
  FA_REQUIRE(a->head_dim == 16 || a->head_dim == 32 || a->head_dim == 64 || a->head_dim == 128, "%s: head_dim must be 16, 32, 64 or 128, got %d", name,
             a->head_dim);
  FA_REQUIRE(a->n_rows >= 0 && a->n_rows < ((int64_t)1 << 30), "%s: n_rows must be in [0, 2^30)", name);
  FA_REQUIRE(a->nheads_q >= 0 && a->nheads_k >= 0 && a->nheads_q <= 65536 && a->nheads_k <= 65536, "%s: bad number of heads", name);
  FA_REQUIRE(a->n_rows * std::max(a->nheads_q, a->nheads_k) < ((int64_t)1 << 33), "%s: 2^33 vectors or more", name);  // (workgroups are counted in 32 bits)
  return FA_OK;
}

int check(const fa_qk_norm_args* a, bool bwd, const char* name) {
  const int rc = check_sizes(a, name);
  if (rc) return rc;
  FA_REQUIRE(a->eps >= 0.f, "%s: eps must not be negative", name);
  FA_REQUIRE(((reinterpret_cast<uintptr_t>(a->rows_end) | reinterpret_cast<uintptr_t>(a->positions)) & 3) == 0, "%s: integers must be 4-byte aligned", name);
  if (a->n_rows == 0) return FA_OK;
  FA_REQUIRE((a->cos_table == nullptr) == (a->sin_table == nullptr), "%s: cos_table and sin_table come together", name);
  if (a->cos_table) {
    FA_REQUIRE(((reinterpret_cast<uintptr_t>(a->cos_table) | reinterpret_cast<uintptr_t>(a->sin_table)) & 7) == 0, "%s: tables must be 8-byte aligned", name);
    FA_REQUIRE(a->table_rows >= 1 && (a->positions || a->seqlen >= 1), "%s: empty table or no positions", name);
    FA_REQUIRE(a->positions || a->seqlen <= a->table_rows, "%s: the tables have %d rows, the sequence %d positions", name, a->table_rows, a->seqlen);
  }
  for (int k = 0; k < 2; k++) {
    const int heads = k ? a->nheads_k : a->nheads_q, D = a->head_dim;
    if (heads == 0) continue;
    const void* x = k ? a->k : a->q;
    const void* w = k ? a->k_weight : a->q_weight;
    const void* dy = k ? a->dk_out : a->dq_out;
    const void* out = bwd ? (k ? a->dk : a->dq) : (k ? a->k_out : a->q_out);
    FA_REQUIRE(x && w && out && (!bwd || (dy && (k ? a->dk_weight : a->dq_weight))), "%s: null pointer", name);
    FA_REQUIRE(aligned16(x) && aligned16(out) && (!bwd || aligned16(dy)), "%s: tensors must be 16-byte aligned", name);
    FA_REQUIRE(stride_ok(k ? a->k_row_stride : a->q_row_stride) && stride_ok(k ? a->k_head_stride : a->q_head_stride) &&
                   (!bwd || (stride_ok(k ? a->dk_out_row_stride : a->dq_out_row_stride) && stride_ok(k ? a->dk_out_head_stride : a->dq_out_head_stride))),
               "%s: strides must be multiples of 8 elements in [0, 2^24)", name);
    const int64_t ors = bwd ? (k ? a->dk_row_stride : a->dq_row_stride) : (k ? a->k_out_row_stride : a->q_out_row_stride);
    const int64_t ohs = bwd ? (k ? a->dk_head_stride : a->dq_head_stride) : (k ? a->k_out_head_stride : a->q_out_head_stride);
    FA_REQUIRE(stride_ok(ors) && stride_ok(ohs) && (a->n_rows == 1 || ors >= D) && (heads == 1 || ohs >= D),
               "%s: written rows and heads must not overlap", name);
  }
  return FA_OK;
}

NormParams params(const fa_qk_norm_args* a, bool bwd) {
  NormParams p{};
  for (int k = 0; k < 2; k++) {
    NormPart& q = p.part[k];
    q.x = k ? a->k : a->q;
    q.w = k ? a->k_weight : a->q_weight;
    q.x_rs = k ? a->k_row_stride : a->q_row_stride;
    q.x_hs = k ? a->k_head_stride : a->q_head_stride;
    q.dy = k ? a->dk_out : a->dq_out;
    q.dy_rs = k ? a->dk_out_row_stride : a->dq_out_row_stride;
    q.dy_hs = k ? a->dk_out_head_stride : a->dq_out_head_stride;
    q.out = bwd ? (k ? a->dk : a->dq) : (k ? a->k_out : a->q_out);
    q.out_rs = bwd ? (k ? a->dk_row_stride : a->dq_row_stride) : (k ? a->k_out_row_stride : a->q_out_row_stride);
    q.out_hs = bwd ? (k ? a->dk_head_stride : a->dq_head_stride) : (k ? a->k_out_head_stride : a->q_out_head_stride);
    q.dw = k ? a->dk_weight : a->dq_weight;
  }
  p.cos = a->cos_table;
  p.sin = a->sin_table;
  p.positions = a->positions;
  p.rows_end = a->rows_end;
  p.n_rows = (int)a->n_rows;
  p.seqlen = a->seqlen > 0 ? a->seqlen : 1;
  p.table_rows = a->table_rows;
  p.eps = a->eps;
  p.w_fp32 = a->weight_dtype == FA_FP32;
  return p;
}

template <typename T, int D, bool kTurn>
void launch_norm_d(const NormParams& p, int blocks, int threads, bool bwd, hipStream_t stream) {
  if (bwd) hipLaunchKernelGGL((qk_norm_rotary_bwd_kernel<T, D, kTurn>), dim3(blocks), dim3(threads), 0, stream, p);
  else if (p.rows == 1) hipLaunchKernelGGL((qk_norm_rotary_kernel<T, D, kTurn, 1>), dim3(blocks), dim3(threads), 0, stream, p);
  else hipLaunchKernelGGL((qk_norm_rotary_kernel<T, D, kTurn, kNormRows>), dim3(blocks), dim3(threads), 0, stream, p);
}

template <typename T>
hipError_t launch_norm(const NormParams& p, int D, int blocks, bool bwd, hipStream_t stream) {
  const int threads = block_threads(p);
#define FA_NORM_D(D_)                                                           \
  case D_:                                                                      \
    if (p.cos) launch_norm_d<T, D_, true>(p, blocks, threads, bwd, stream);     \
    else launch_norm_d<T, D_, false>(p, blocks, threads, bwd, stream);          \
    break;
  switch (D) {
    FA_NORM_D(16)
    FA_NORM_D(32)
    FA_NORM_D(64)
    FA_NORM_D(128)
    default: return hipErrorInvalidValue;
  }
#undef FA_NORM_D
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !bwd) return e;
  const int parts = p.part[1].dw != nullptr ? 2 : 1;  // (keys without heads: no workgroup, a gradient of zeros)
  hipLaunchKernelGGL(norm_weights_kernel<T>, dim3((unsigned)(parts * (D / 16))), dim3(1024), 0, stream, p, D);
  return hipGetLastError();
}

}  // namespace
}  // namespace fa

extern "C" {

int fa_qk_norm_rotary(const fa_qk_norm_args* a) {
  const int rc = fa::check(a, false, "fa_qk_norm_rotary");
  if (rc || a->n_rows == 0) return rc;
  fa::NormParams p = fa::params(a, false);
  const int blocks = fa::cut_parts(&p, a, false);
  if (blocks == 0) return FA_OK;
  const hipStream_t stream = reinterpret_cast<hipStream_t>(a->stream);
  FA_LAUNCH(a->dtype == FA_FP16 ? fa::launch_norm<_Float16>(p, a->head_dim, blocks, false, stream)
                                : fa::launch_norm<__bf16>(p, a->head_dim, blocks, false, stream));
  return FA_OK;
}

size_t fa_qk_norm_rotary_bwd_workspace_bytes(const fa_qk_norm_args* a) {
  if (fa::check_sizes(a, "fa_qk_norm_rotary_bwd") != FA_OK) return 0;
  fa::NormParams p{};
  return (size_t)fa::cut_parts(&p, a, true) * a->head_dim * sizeof(float);
}

int fa_qk_norm_rotary_bwd(const fa_qk_norm_args* a) {
  const int rc = fa::check(a, true, "fa_qk_norm_rotary_bwd");
  if (rc) return rc;
  FA_REQUIRE(a->n_rows > 0, "fa_qk_norm_rotary_bwd: no rows (the weights' gradients would be left as they are)");
  FA_REQUIRE(a->nheads_q > 0, "fa_qk_norm_rotary_bwd: no query heads");
  fa::NormParams p = fa::params(a, true);
  const int blocks = fa::cut_parts(&p, a, true);
  const size_t need = (size_t)blocks * a->head_dim * sizeof(float);
  if (!a->workspace || a->workspace_bytes < need || !fa::aligned16(a->workspace))
    return fa::fail(FA_ERR_WORKSPACE, "fa_qk_norm_rotary_bwd: needs %zu bytes of 16-byte aligned workspace", need);
  p.partial = reinterpret_cast<float*>(a->workspace);
  const hipStream_t stream = reinterpret_cast<hipStream_t>(a->stream);
  FA_LAUNCH(a->dtype == FA_FP16 ? fa::launch_norm<_Float16>(p, a->head_dim, blocks, true, stream)
                                : fa::launch_norm<__bf16>(p, a->head_dim, blocks, true, stream));
  return FA_OK;
}

}  // extern "C"
