// Attention of a few rows a key head (decoding: one new token of each sequence, or a handful, times the heads of a group) over a paged cache:
// every key and value is read once and used for at most 32 rows, a stream of K and V that HBM bounds.
//
// A wave owns 32-key tiles: it stages them into a double buffer of its own by direct-to-LDS loads, counts its outstanding loads instead of meeting the
// other waves, and multiplies in the orientation S^T = K Q^T, O^T = V^T P^T (a lane is a row); the workgroup's waves join their partial results in
// LDS at the end of a pair.  Lengths differ and are known on the device only, so the launch does not cut sequences into equal numbers of pieces: all
// units of kDecodeUnit keys of all pairs are laid out in one line, and each of the resident workgroups takes an equal share of it - the end of one
// pair, some whole pairs, the beginning of another.  Pairs that more than one workgroup has touched are joined by a second kernel.  Pairs that fill
// the device by themselves, and short ones, have a workgroup each (the rule, with both sides' times, is fa_paged_api.hip's).
// 32 x 8 pairs of 4096 .. 16384 keys, d = 128, 1.34 GB: 239 us, 5.6 TB/s; 8 pairs of 16000 23, 12 of 500 keys, d = 64, 7.8: a chain of latencies.
#include "fa_paged_line.h"

namespace fa {

namespace {

template <int D, int NW_>
struct Cfg {
  static constexpr int NW = NW_;
  static constexpr int BN = 32;
  static constexpr int DV = D < 32 ? 32 : D;
  static constexpr int kTile = BN * D * 2;
  static constexpr int kWave = 2 * 2 * kTile;     // two stages of (K tile, V tile)
  static constexpr int kSlack = D < 32 ? 64 : 0;  // the 32-wide transposed reads run past a 16-wide V row
  static constexpr int XS = DV + 4;               // merge: floats per (wave, row)
  static constexpr int kMerge = NW * 32 * XS * 4 + 3 * NW * 32 * 4;
  static constexpr int kTiles = NW * kWave + kSlack;
  static constexpr int kLds = kTiles > kMerge ? kTiles : kMerge;
};

}  // namespace

// Waves per SIMD that registers are to allow: without a bound the compiler puts the products into accumulation registers and moves them out one by one (d = 64, 32 x 8
// pairs of 4096 .. 16384 keys 135 us, with the bound 132; d = 32 75.6, 73.4).  At d = 128 LDS allows one.
constexpr int decode_bound(int head_dim, int waves) { return head_dim == 128 ? 1 : (waves == 8 ? 2 : (head_dim == 64 ? 3 : 4)); }

template <typename T, int D, int NW_>
__global__ void __launch_bounds__(64 * NW_, decode_bound(D, NW_)) fa_paged_decode_kernel(const PagedFwdParams p) {
  using C = Cfg<D, NW_>;
  using E = Elem<T>;
  using vec8 = typename E::vec8;
  constexpr int NW = C::NW, BN = C::BN, DV = C::DV;
  using KStager = GroupStager<D, kSwzRow>;
  using VStager = GroupStager<D, kSwzTr>;
  constexpr int NI = 2 * KStager::NI;  // loads of a tile's K, and of its V
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[C::kLds];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hf = lane >> 5;
  const float cs = p.scale_log2;

  KStager ks_;
  VStager vs_;
  ks_.init(lane, p.c.k_ss);
  vs_.init(lane, p.c.v_ss);
  unsigned char* const lds_wave = lds_raw + wave * C::kWave;
  int koff[D / 16], voff[DV / 32];
#pragma unroll
  for (int ks = 0; ks < D / 16; ks++) koff[ks] = frag_off<D, kSwzRow>(c, ks * 2 + hf);
#pragma unroll
  for (int db = 0; db < DV / 32; db++) voff[db] = tr_off<D, kSwzTr>(0, db * 4, lane);

  // ---- this workgroup's share of the line: [u, u_end), from `at` on
  int64_t u, u_end;
  Spot at;
  if (p.groups > 0) {
    const int sums0 = unit_sums(p.c, 0);
    const int64_t units = all_units(p.c, sums0);
    const int n = sharers(p, units);
    if ((int)blockIdx.x >= n || units == 0) return;
    u = share_begin(units, blockIdx.x, n);
    u_end = share_begin(units, blockIdx.x + 1, n);
    at = spot_of(p.c, u, sums0);
  } else {  // one pair
    const int b = blockIdx.x / p.c.HK, keys = paged_len(p.c, b);
    at = Spot{b, (int)blockIdx.x - b * p.c.HK, 0, keys <= kDecodeUnit ? 1 : (keys + kDecodeUnit - 1) / kDecodeUnit};
    u = 0;
    u_end = at.units;
  }

  bool first = true;
  while (u < u_end) {
    const int b = __builtin_amdgcn_readfirstlane(at.b), h = __builtin_amdgcn_readfirstlane(at.h);
    const int unit0 = __builtin_amdgcn_readfirstlane(at.unit), pair_units = __builtin_amdgcn_readfirstlane(at.units);
    const int unit1 = u_end - u < pair_units - unit0 ? unit0 + (int)(u_end - u) : pair_units;
    // a tile's two groups of 16 keys: their pages are asked for a step before they are needed, those of the first two tiles together with the lengths
    const int32_t* const table = p.c.table + (int64_t)b * p.c.table_rs;
    const int k_lo = unit0 * kDecodeUnit;
    int page[2], page2[2];
    auto ask = [&](int t, int (&to)[2]) {
#pragma unroll
      for (int j = 0; j < 2; j++) to[j] = page_of_group(p.c, table, (k_lo >> 4) + 2 * t + j);
    };
    ask(wave, page);
    ask(wave + NW, page2);
    int q_begin = 0, Lq = 0;
    if (!paged_rows(p.c, b, &q_begin, &Lq)) return;  // (on the line such a sequence has no units)
    const int Lk = paged_len(p.c, b), G = p.c.G, rows = Lq * G;
    const int k_hi = Lk < unit1 * kDecodeUnit ? Lk : unit1 * kDecodeUnit;
    const int ntiles = k_hi > k_lo ? (k_hi - k_lo + BN - 1) / BN : 0;
    const char* const kb = p.c.k + h * p.c.k_hs;
    const char* const vb = p.c.v + h * p.c.v_hs;
    const int last_group = (Lk - 1) >> 4;

    auto issue = [&](int t, int stage, const int (&pages)[2]) {
      unsigned char* const dst = lds_wave + stage * 2 * C::kTile;
      const int g0 = (k_lo >> 4) + 2 * t;
      const bool both = g0 < last_group;  // (else the tile's second half repeats the last key, in the first one's page)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int g = both ? g0 + j : g0, pg = both ? pages[j] : pages[0];
        ks_.issue(kb + pg * p.c.k_ps + slot_of_group(p.c, g) * p.c.k_ss, p.c.k_ss, g < last_group ? 15 : (Lk - 1) & 15, dst + j * KStager::kBytes);
      }
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int g = both ? g0 + j : g0, pg = both ? pages[j] : pages[0];
        vs_.issue(vb + pg * p.c.v_ps + slot_of_group(p.c, g) * p.c.v_ss, p.c.v_ss, g < last_group ? 15 : (Lk - 1) & 15, dst + C::kTile + j * VStager::kBytes);
      }
    };

    int t = wave, stage = 0;
    if (t < ntiles) issue(t, 0, page);
    if (t + NW < ntiles) issue(t + NW, 1, page2);
    const int row = c < rows ? c : rows - 1;  // (columns past the last row repeat it and are dropped at the end)
    const int tok = row / G;
    vec8 qreg[D / 16];
    {
      const T* qp = reinterpret_cast<const T*>(p.q) + (int64_t)(q_begin + tok) * p.q_rs + (int64_t)(h * G + (row - tok * G)) * p.q_hs + hf * 8;
#pragma unroll
      for (int ks = 0; ks < D / 16; ks++) qreg[ks] = bitcast<vec8>(ld_global16(qp + ks * 16));
      // waited for here (with the first two tiles): the main loop counts this wave's outstanding loads, these are not to be among them
      wait_vmcnt<0>();
#pragma unroll
      for (int ks = 0; ks < D / 16; ks++) asm volatile("" : "+v"(qreg[ks]));
    }
    const int limit = p.causal ? Lk - Lq + tok + 1 : Lk;
    const int least_limit = p.causal ? Lk - Lq + 1 : Lk;  // of row 0

    f32x16 o_acc[DV / 32];
#pragma unroll
    for (int i = 0; i < DV / 32; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) o_acc[i][r] = 0.f;
    float m_i = -INFINITY, l_i = 0.f, u_i = 0.f;  // l_i, u_i: this lane's share, the other half's in lane ^ 32

    for (; t < ntiles; t += NW) {
      const bool next = t + NW < ntiles;  // its 2 * NI loads were issued after this tile's
      if (next) wait_vmcnt<3 * NI>();
      else wait_vmcnt<NI>();
      if (t + 2 * NW < ntiles) ask(t + 2 * NW, page);
      const T* const Ks = reinterpret_cast<const T*>(lds_wave + stage * 2 * C::kTile);
      const T* const Vs = Ks + BN * D;
      f32x16 s;
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ks++) s = E::mfma32(*reinterpret_cast<const vec8*>(Ks + koff[ks]), qreg[ks], s);
      const int n0 = k_lo + t * BN;
      if (n0 + BN > least_limit) {
        const int dead = limit - n0 - 4 * hf;
#pragma unroll
        for (int r = 0; r < 16; r++)
          if (8 * (r >> 2) + (r & 3) >= dead) s[r] = -INFINITY;
      }
      float mt = s[0];
#pragma unroll
      for (int r = 1; r < 16; r++) mt = fmaxf(mt, s[r]);
      mt = half_max(mt);
      if (__any(mt > m_i)) {
        const float m_new = fmaxf(m_i, mt);
        const float alpha = m_new == -INFINITY ? 1.f : fast_exp2((m_i - m_new) * cs);
        m_i = m_new;
        l_i *= alpha;
        u_i *= alpha;
#pragma unroll
        for (int i = 0; i < DV / 32; i++) o_acc[i] = o_acc[i] * alpha;
      }
      const float mc = (m_i == -INFINITY ? 0.f : m_i) * cs;
      vec8 pb[2];
#pragma unroll
      for (int tt = 0; tt < 2; tt++) {
        f32x8 pf;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          pf[i] = fast_exp2(__builtin_fmaf(s[8 * tt + i], cs, -mc));
          u_i += pf[i];
        }
        pb[tt] = cvt8<T>(pf);
        l_i = sum8_acc(pb[tt], l_i);
      }
      if (next) wait_vmcnt<2 * NI>();
      else wait_vmcnt<0>();
#pragma unroll
      for (int tt = 0; tt < 2; tt++)
#pragma unroll
        for (int db = 0; db < DV / 32; db++) {
          const T* vp = Vs + 16 * tt * D + voff[db];
          const u32x2 lo = lds_read_tr16(vp), hi = lds_read_tr16(vp + 8 * D);
          o_acc[db] = E::mfma32(bitcast<vec8>(u32x4{lo[0], lo[1], hi[0], hi[1]}), pb[tt], o_acc[db]);
        }
      if (t + 2 * NW < ntiles) {
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the stage has been read before it is refilled
        issue(t + 2 * NW, stage, page);
      }
      stage ^= 1;
    }

    // ---- the waves' partial results joined: row r of wave w at X[(w * 32 + r) * XS], m, l and u behind all rows
    __syncthreads();
    float* const X = reinterpret_cast<float*>(lds_raw);
    float* const Xm = X + NW * 32 * C::XS;
    float* const Xl = Xm + NW * 32;
    float* const Xu = Xl + NW * 32;
    l_i = half_sum(l_i);
    u_i = half_sum(u_i);
    if (c < rows) {
      if (hf == 0) {
        Xm[wave * 32 + c] = m_i;
        Xl[wave * 32 + c] = l_i;
        Xu[wave * 32 + c] = u_i;
      }
#pragma unroll
      for (int db = 0; db < DV / 32; db++)
#pragma unroll
        for (int g4 = 0; g4 < 4; g4++) {
          f32x4 x;
#pragma unroll
          for (int i = 0; i < 4; i++) x[i] = o_acc[db][g4 * 4 + i];
          *reinterpret_cast<f32x4*>(X + (wave * 32 + c) * C::XS + db * 32 + g4 * 8 + hf * 4) = x;
        }
    }
    __syncthreads();
    const bool whole = unit0 == 0 && unit1 == pair_units;
    float* const part_o = whole ? nullptr : p.part + ((int64_t)blockIdx.x * 2 + (first ? 0 : 1)) * (kPartRows * (D + 3));
    for (int idx = tid; idx < rows * (D / 4); idx += 64 * NW) {
      const int r = idx / (D / 4), d0 = idx % (D / 4) * 4;
      float m = Xm[r];
#pragma unroll
      for (int w = 1; w < NW; w++) m = fmaxf(m, Xm[w * 32 + r]);
      const float mu = m == -INFINITY ? 0.f : m;
      float l = 0.f, us = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; w++) {
        const float f = fast_exp2((Xm[w * 32 + r] - mu) * cs);  // 0 for a wave without keys
        l = __builtin_fmaf(Xl[w * 32 + r], f, l);
        us = __builtin_fmaf(Xu[w * 32 + r], f, us);
        o = o + *reinterpret_cast<const f32x4*>(X + (w * 32 + r) * C::XS + d0) * f;
      }
      if (whole) {
        store_row_piece<T>(p, q_begin, h, r, d0, o * (l > 0.f ? fast_rcp(l) : 1.f));
        if (d0 == 0) store_lse(p, b, h, r, lse_of(m, us, cs));
      } else {
        *reinterpret_cast<f32x4*>(part_o + r * D + d0) = o;
        if (d0 == 0) {
          float* const ml = part_o + kPartRows * D + r;
          ml[0] = m;
          ml[kPartRows] = l;
          ml[2 * kPartRows] = us;
        }
      }
    }
    first = false;
    u += unit1 - unit0;
    if (u >= u_end) return;
    if (!next_pair(p.c, &at)) return;  // (never: the line does not end here)
    __syncthreads();  // the joined results have been read before the tiles come in over them
  }
}

namespace {

// The pairs that the ends of the workgroups' shares have cut (blockIdx.x: a pair; blockIdx.y and the threads share its rows): D / 4 threads over a row's
// elements, times lanes over its parts - as many as there are, rounded up to a power of two -, times rows side by side.  The lanes' results are
// joined in LDS, in the same order each time.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_decode_join_kernel(const PagedFwdParams p) {
  constexpr int kCols = D / 4, kLanes = 256 / kCols;
  __shared__ f32x4 os[256];
  __shared__ PartRow ms[256];
  const int b = blockIdx.x / p.c.HK, h = (int)blockIdx.x - b * p.c.HK;
  int64_t units = 0, begin = 0;  // of all pairs; where this one's lie
  int pair_units = 0;
  for (int first = 0; first < p.c.B; first += 64) {
    const int sums = unit_sums(p.c, first), k = b - first;
    if (k >= 0 && k < 64) {
      const int upto = k > 0 ? __builtin_amdgcn_readlane(sums, k > 0 ? k - 1 : 0) : 0;
      pair_units = __builtin_amdgcn_readlane(sums, k) - upto;
      begin = (units + upto) * p.c.HK + (int64_t)h * pair_units;
    }
    units += __builtin_amdgcn_readlane(sums, 63);
  }
  units *= p.c.HK;
  int q_begin = 0, Lq = 0;
  if (pair_units == 0 || !paged_rows(p.c, b, &q_begin, &Lq)) return;
  const int n = sharers(p, units);
  const auto share_of = [&](int64_t u) { return (int)(((u + 1) * n - 1) / units); };  // (the last w with units * w / n <= u)
  const int w0 = share_of(begin), w1 = share_of(begin + pair_units - 1);
  if (w0 == w1) return;  // whole
  const float cs = p.scale_log2;
  constexpr int kEach = kPartRows * (D + 3);
  // the pair is the last of share w0, and its first, too, if the share begins with it; it is the first of the others'
  const int first_slot = share_begin(units, w0, n) == begin ? 0 : 1;
  int lanes = 2;
  while (lanes < kLanes && lanes < w1 - w0 + 1) lanes *= 2;
  const int col = threadIdx.x % kCols, at = threadIdx.x / kCols, lane = at & (lanes - 1), side = at / lanes, beside = kLanes / lanes;
  const int rows = Lq * p.c.G;
  for (int r0 = blockIdx.y * beside; r0 < rows; r0 += gridDim.y * beside) {
    const int r = r0 + side;
    JoinedRow x;
    if (r < rows)
      for (int i = w0 + lane; i <= w1; i += lanes) {
        const float* const s = p.part + ((int64_t)i * 2 + (i == w0 ? first_slot : 0)) * kEach;
        const float* const ml = s + kPartRows * D + r;
        x.add(PartRow{ml[0], ml[kPartRows], ml[2 * kPartRows]}, *reinterpret_cast<const f32x4*>(s + r * D + col * 4), cs);
      }
    x.across<kCols>(lane, lanes, cs, os, ms);
    if (lane == 0 && r < rows) {
      store_row_piece<T>(p, q_begin, h, r, col * 4, x.o * (x.a.l > 0.f ? fast_rcp(x.a.l) : 1.f));
      if (col == 0) store_lse(p, b, h, r, lse_of(x.a.m, x.a.u, cs));
    }
  }
}

template <typename T, int D>
hipError_t launch_d(const PagedFwdParams& p, hipStream_t stream) {
  const unsigned pairs = (unsigned)(p.c.B * p.c.HK);
  const dim3 grid(p.groups > 0 ? (unsigned)p.groups : pairs);
  if (p.wide) hipLaunchKernelGGL((fa_paged_decode_kernel<T, D, kDecodeWide(D)>), grid, dim3(64 * kDecodeWide(D)), 0, stream, p);
  else hipLaunchKernelGGL((fa_paged_decode_kernel<T, D, kDecodeWaves(D)>), grid, dim3(64 * kDecodeWaves(D)), 0, stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.groups == 0) return e;
  const unsigned rows = (unsigned)(p.c.max_sq * p.c.G), side = pairs < 1024 ? 1024 / pairs : 1;  // (workgroups beside each other for a pair's rows)
  hipLaunchKernelGGL((paged_decode_join_kernel<T, D>), dim3(pairs, rows < side ? rows : side), dim3(256), 0, stream, p);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_t(const PagedFwdParams& p, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 16: return launch_d<T, 16>(p, stream);
    case 32: return launch_d<T, 32>(p, stream);
    case 64: return launch_d<T, 64>(p, stream);
    case 128: return launch_d<T, 128>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_paged_decode(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return dtype == 0 ? launch_t<_Float16>(p, head_dim, stream) : launch_t<__bf16>(p, head_dim, stream);
}

}  // namespace fa
