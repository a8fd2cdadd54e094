// fa_paged_key_weights: to the weight of every key of a paged cache is added what it receives of the new tokens' attention,
//   w[h, j] += sum over rows r of exp(scale q_r . k_j - lse_r)      (rows: the tokens and heads of the group, fa_paged_fwd.h)
// the probabilities formed again from the forward's lse: no second pass over V, no maxima.
//
// A wave owns 32 keys, their fragments in registers (read once, straight from the pages), and streams the rows past them in tiles of 32 that the
// workgroup's four waves share through LDS: S = Q K^T leaves a key in a lane, so that its sum stays in the lane's register and has one
// owner.  Few rows: bound by the read of K.  Many: by the exponentials, one per score.
#include "fa_paged_fwd.h"

namespace fa {

namespace {

struct WeightsParams {
  PagedFwdParams f;
  uint32_t group_magic;  // ceil(2^32 / G), for numbers of at most 2^16: x / G = x * magic >> 32 (G = 1: not used)
};

template <int D>
struct WCfg {
  static constexpr int kTile = 32 * D * 2;
  static constexpr int kRowOff = 2 * kTile;  // per buffer: 32 lse, 32 limits
  static constexpr int kLds = 2 * kTile + 2 * 256;
};

}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(256) fa_paged_weights_kernel(const WeightsParams wp) {
  using C = WCfg<D>;
  using E = Elem<T>;
  using vec8 = typename E::vec8;
  constexpr int CH = D / 8;
  const PagedFwdParams& p = wp.f;
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[C::kLds];

  const int blocks = (p.c.max_keys + 127) / 128;
  const int pair = blockIdx.x / blocks, kblock = (int)blockIdx.x - pair * blocks;
  const int b = pair / p.c.HK, h = pair - b * p.c.HK;
  int q_begin = 0, Lq = 0;
  if (!paged_rows(p.c, b, &q_begin, &Lq)) return;
  const int Lk = paged_len(p.c, b), G = p.c.G, rows = Lq * G;
  if (kblock * 128 >= Lk) return;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hf = lane >> 5;
  const int key0 = kblock * 128 + wave * 32;  // of this wave
  const bool live = key0 < Lk;
  const float cs = p.scale_log2;
  const auto per_group = [&](int x) { return G == 1 ? x : (int)__umulhi((uint32_t)x, wp.group_magic); };

  // ---- this wave's keys (past the end: the last one, whose sum is not stored)
  const int32_t* const table = p.c.table + (int64_t)b * p.c.table_rs;
  const int key = key0 + c < Lk ? key0 + c : Lk - 1;
  vec8 kreg[D / 16];
  {
    const int g0 = key0 >> 4, last = (Lk - 1) >> 4;
    const int ga = g0 < last ? g0 : last, gb = g0 + 1 < last ? g0 + 1 : last;
    const char* const pa = p.c.k + page_of_group(p.c, table, ga) * p.c.k_ps + h * p.c.k_hs;
    const char* const pb = p.c.k + page_of_group(p.c, table, gb) * p.c.k_ps + h * p.c.k_hs;
    const int slot = key & ((1 << p.c.page_log2) - 1);
    const char* const at = ((key >> 4) == ga ? pa : pb) + slot * p.c.k_ss + hf * 16;
#pragma unroll
    for (int ks = 0; ks < D / 16; ks++) kreg[ks] = bitcast<vec8>(ld_global16(at + ks * 32));
  }

  // ---- rows: from the first that sees the workgroup's first key on
  const int past = Lk - Lq + 1;  // row r sees the keys below past + r / G
  int row_first = 0;
  if (p.causal) {
    const int tok = kblock * 128 - past + 1;
    row_first = tok > 0 ? tok * G : 0;
  }
  const int tile0 = row_first >> 5, ntiles = (rows + 31) >> 5;
  // the next tile's first row as (token, head of the group)
  int tok0 = __builtin_amdgcn_readfirstlane((tile0 * 32) / G), head0 = __builtin_amdgcn_readfirstlane(tile0 * 32 - tok0 * G);
  constexpr int RPI = 64 / CH;                        // rows per direct-to-LDS instruction
  constexpr int TI = 32 / RPI > 0 ? 32 / RPI : 1;     // instructions of a tile
  const int rl = lane / CH, pch = lane % CH;
  auto stage = [&](int it, int buf) {
    const char* const qb = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.q) + (int64_t)(q_begin + tok0) * p.q_rs + (int64_t)h * G * p.q_hs);
#pragma unroll
    for (int i = 0; i < TI; i++) {
      if (TI >= 4 ? (i & 3) != wave : i != wave) continue;
      int r = i * RPI + rl;
      const int sw = tile_swz<D, kSwzRow>(r);
      const int most = rows - 1 - it * 32;
      r = r < most ? r : most;
      const int x = head0 + r, t = per_group(x), g = x - t * G;
      dma16(qb, (uint32_t)(t * p.q_rs * 2 + g * p.q_hs * 2) + 16u * (uint32_t)(pch ^ sw), lds_raw + buf * C::kTile + i * 1024);
    }
  };
  // a row's lse (in log2 units; +inf: no row, or one that sees nothing) and limit
  float lse_next = INFINITY;
  int limit_next = 0;
  auto fetch_row = [&](int it) {  // wave 0, lanes below 32
    const int r = it * 32 + c;
    lse_next = INFINITY;
    limit_next = 0;
    if (wave == 0 && hf == 0 && r < rows) {
      const int x = head0 + c, t = per_group(x), g = x - t * G;
      const float v = p.lse[((int64_t)b * p.c.H + h * G + g) * p.sq_r + tok0 + t];
      lse_next = v == -INFINITY ? INFINITY : v * kLog2e;
      limit_next = p.causal ? past + tok0 + t : Lk;
    }
  };
  auto store_row = [&](int buf) {
    if (wave == 0 && hf == 0) {
      reinterpret_cast<float*>(lds_raw + C::kRowOff + buf * 256)[c] = lse_next;
      reinterpret_cast<int*>(lds_raw + C::kRowOff + buf * 256 + 128)[c] = limit_next;
    }
  };
  int first_tok = tok0;  // of the tile in hand
  auto advance = [&]() {
    const int x = head0 + 32, t = __builtin_amdgcn_readfirstlane(per_group(x));
    tok0 += t;
    head0 = x - t * G;
  };
  int qoff[D / 16];
#pragma unroll
  for (int ks = 0; ks < D / 16; ks++) qoff[ks] = frag_off<D, kSwzRow>(c, ks * 2 + hf);

  float sum = 0.f;
  int it = tile0, buf = 0;
  if (it < ntiles) {
    stage(it, 0);
    fetch_row(it);
    store_row(0);
    advance();
  }
  while (it < ntiles) {
    if (it + 1 < ntiles) fetch_row(it + 1);
    wait_vmem();
    __syncthreads();
    const int next_tok = tok0;
    if (it + 1 < ntiles) {
      stage(it + 1, buf ^ 1);
      store_row(buf ^ 1);
      advance();
    }
    const int* const limits = reinterpret_cast<const int*>(lds_raw + C::kRowOff + buf * 256 + 128);
    const float* const lses = reinterpret_cast<const float*>(lds_raw + C::kRowOff + buf * 256);
    const T* const Qs = reinterpret_cast<const T*>(lds_raw + buf * C::kTile);
    if (live) {
      f32x16 s;
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ks++) s = E::mfma32(*reinterpret_cast<const vec8*>(Qs + qoff[ks]), kreg[ks], s);
      const bool mask = p.causal && past + first_tok < key0 + 32;  // the tile's first row does not see all of the wave's keys
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const f32x4 l4 = *reinterpret_cast<const f32x4*>(lses + 8 * j + 4 * hf);
        f32x4 e;
#pragma unroll
        for (int i = 0; i < 4; i++) e[i] = fast_exp2(__builtin_fmaf(s[4 * j + i], cs, -l4[i]));
        if (mask) {
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (key >= limits[8 * j + 4 * hf + i]) e[i] = 0.f;
        }
        sum += (e[0] + e[1]) + (e[2] + e[3]);
      }
    }
    first_tok = next_tok;
    buf ^= 1;
    it++;
  }
  sum = half_sum(sum);
  if (hf == 0 && key0 + c < Lk) {
    const int page = table[key >> p.c.page_log2];
    if (page_is_one(page, p.c.n_pages)) {
      float* const w = p.c.weights + (((int64_t)page * p.c.HK + h) << p.c.page_log2) + (key & ((1 << p.c.page_log2) - 1));
      *w += sum;
    }
  }
}

namespace {
template <typename T>
hipError_t launch_t(const WeightsParams& p, int head_dim, hipStream_t stream) {
  const int64_t n = (int64_t)p.f.c.B * p.f.c.HK * ((p.f.c.max_keys + 127) / 128);
  if (n >= ((int64_t)1 << 31)) return hipErrorInvalidValue;
  const dim3 grid((unsigned)n);
  switch (head_dim) {
    case 16: hipLaunchKernelGGL((fa_paged_weights_kernel<T, 16>), grid, dim3(256), 0, stream, p); break;
    case 32: hipLaunchKernelGGL((fa_paged_weights_kernel<T, 32>), grid, dim3(256), 0, stream, p); break;
    case 64: hipLaunchKernelGGL((fa_paged_weights_kernel<T, 64>), grid, dim3(256), 0, stream, p); break;
    case 128: hipLaunchKernelGGL((fa_paged_weights_kernel<T, 128>), grid, dim3(256), 0, stream, p); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}
}  // namespace

hipError_t launch_paged_key_weights(const PagedFwdParams& f, int dtype, int head_dim, hipStream_t stream) {
  WeightsParams p{f, f.c.G > 1 ? (uint32_t)((((uint64_t)1 << 32) + f.c.G - 1) / f.c.G) : 0u};
  return dtype == 0 ? launch_t<_Float16>(p, head_dim, stream) : launch_t<__bf16>(p, head_dim, stream);
}

}  // namespace fa
