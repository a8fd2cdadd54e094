// fa_paged_evict: every key head of a sequence keeps `budget` keys, the newest and the heaviest; the kept ones that lie behind slot `budget` move into
// the holes that the others leave before it.  Nothing else moves: the order of a cache's keys does not matter to attention, and a decode step that is
// one key over its budget moves one key.
//
// A workgroup per (sequence, key head) finds the weight of the budget-th key by a radix selection over the weights' bits, mapped to integers of
// the same order (three digits of 11, 11 and 10 bits, counted in LDS), where the newest keys come above every weight; keys of just that weight stay
// from the lowest slot on.  Holes and moving keys are numbered by prefix sums in slot order, so the n-th hole takes the n-th key, and left in the
// workspace; a second kernel copies them, a launch of many workgroups, since sources and destinations are different slots.
// Bound by one read of weights and positions (8 bytes a slot) and two passes over each moved vector.
#include <algorithm>

#include "fa_paged.h"

namespace fa {

namespace {

struct EvictParams {
  PagedCache c;
  const int32_t* next;
  int32_t* new_len;
  int budget, recent, cap;  // cap: most moves of a head
  int32_t* counts;          // [B * HK]
  int32_t* moves;           // [B * HK][2][cap]: holes, keys that come
};

// (8 x 8 heads of 4915 .. 16384 keys to 4096, two caches in turn, the copies of weights and positions that a pass begins with included: 60.1 us; 512 threads 67.2)
constexpr int kEvictThreads = 1024;
constexpr uint32_t kNewest = 0xffffffffu;
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

// A weight as an unsigned integer of the same order; NaN as -inf, -0 as 0
FA_DEVICE uint32_t ordered(float w) {
  const uint32_t u = __float_as_uint(w != w ? -INFINITY : w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Copies `moves` (at most kMovesPerGroup) of a head's keys and values: first where each comes from and goes to, into LDS, then 16 bytes a thread at a time,
// four of them in flight (8 x 8 heads cut from 4915 .. 16384 keys to 4096, d = 128, 149 MB: the pass of above 60.1 us, with two 60.9,
// with eight 95.4; as the case of perf/operators.py is timed 62.9).
constexpr int kMovesPerGroup = 64;
struct MoveSpots {
  int64_t at[kMovesPerGroup][4];  // k from, k to (negative: nowhere), v from, v to: bytes
};
template <int D, int kThreads>
FA_DEVICE void move_keys(const EvictParams& p, int b, int h, const int32_t* holes, const int32_t* comes, int moves, MoveSpots& spots) {
  constexpr int CH = D / 8, kEach = kMovesPerGroup * 2 * CH / kThreads, kFly = kEach < 1 ? 1 : (kEach < 4 ? kEach : 4);
  const int mask = (1 << p.c.page_log2) - 1;
  if ((int)threadIdx.x < moves) {
    const int32_t* const table = p.c.table + (int64_t)b * p.c.table_rs;
    const int to = holes[threadIdx.x], from = comes[threadIdx.x];
    const int to_page = table[to >> p.c.page_log2], from_page = page_in_pool(table[from >> p.c.page_log2], p.c.n_pages);
    int64_t* const at = spots.at[threadIdx.x];
    at[0] = from_page * p.c.k_ps + (from & mask) * p.c.k_ss + h * p.c.k_hs;
    at[2] = from_page * p.c.v_ps + (from & mask) * p.c.v_ss + h * p.c.v_hs;
    if (page_is_one(to_page, p.c.n_pages)) {
      at[1] = to_page * p.c.k_ps + (to & mask) * p.c.k_ss + h * p.c.k_hs;
      at[3] = to_page * p.c.v_ps + (to & mask) * p.c.v_ss + h * p.c.v_hs;
      const int64_t d = (((int64_t)to_page * p.c.HK + h) << p.c.page_log2) + (to & mask);
      const int64_t s = (((int64_t)from_page * p.c.HK + h) << p.c.page_log2) + (from & mask);
      p.c.weights[d] = p.c.weights[s];
      p.c.positions[d] = p.c.positions[s];
    } else {
      at[1] = at[3] = -1;
    }
  }
  __syncthreads();
  const int n = moves * 2 * CH;
  for (int i0 = threadIdx.x; i0 < n; i0 += kThreads * kFly) {
    u32x4 x[kFly];
#pragma unroll
    for (int f = 0; f < kFly; f++) {
      const int i = i0 + f * kThreads;
      if (i < n) x[f] = ld_global16((i / CH & 1 ? p.c.v : p.c.k) + spots.at[i / (2 * CH)][i / CH & 1 ? 2 : 0] + i % CH * 16);
    }
#pragma unroll
    for (int f = 0; f < kFly; f++) {
      const int i = i0 + f * kThreads;
      if (i < n) {
        const int64_t to = spots.at[i / (2 * CH)][i / CH & 1 ? 3 : 1];
        if (to >= 0) st_global16((i / CH & 1 ? p.c.v : p.c.k) + to + i % CH * 16, x[f]);
      }
    }
  }
}

// Sum of the values that the waves before this one left in x (one a wave); *all: of all of them
template <int kWaves>
FA_DEVICE int before_wave(const int* x, int wave, int* all) {
  const int lane = threadIdx.x & 63;
  const int pre = wave_prefix_sum(lane < kWaves ? x[lane] : 0);
  *all = __builtin_amdgcn_readlane(pre, kWaves - 1);
  return wave > 0 ? __builtin_amdgcn_readlane(pre, wave > 0 ? wave - 1 : 0) : 0;
}

// kCap: keys whose mapped weights are kept in LDS (0: read again in every pass).  kMoveD: 0, or the head dimension where a head has at most
// kMovesPerGroup moves: the workgroup then makes them itself, without another launch.
template <int kCap, int kMoveD>
__global__ void __launch_bounds__(kEvictThreads) paged_evict_kernel(const EvictParams p) {
  constexpr int kThreads = kEvictThreads, kWaves = kThreads / 64;
  __shared__ __attribute__((aligned(16))) uint32_t keys[kCap > 0 ? kCap : 4];
  __shared__ int hist[2048];
  __shared__ int sums[2][kWaves];
  __shared__ uint32_t found[3];  // digit, keys above it, keys of it
  const int b = blockIdx.x / p.c.HK, h = (int)blockIdx.x - b * p.c.HK;
  const int L = paged_len(p.c, b);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (h == 0 && tid == 0) p.new_len[b] = L < p.budget ? L : p.budget;
  if (L <= p.budget) {
    if (kMoveD == 0 && tid == 0) p.counts[blockIdx.x] = 0;
    return;
  }
  const int64_t newest = (int64_t)p.next[b] - p.recent;
  const int32_t* const table = p.c.table + (int64_t)b * p.c.table_rs;
  const int mask = (1 << p.c.page_log2) - 1;
  auto read_key = [&](int j) {
    const int page = page_in_pool(table[j >> p.c.page_log2], p.c.n_pages);
    const int64_t at = (((int64_t)page * p.c.HK + h) << p.c.page_log2) + (j & mask);
    const uint32_t k = ordered(p.c.weights[at]);
    return p.c.positions[at] >= newest ? kNewest : k;
  };
  auto key_of = [&](int j) { return kCap > 0 ? keys[j] : read_key(j); };
  // (the lanes whose digit is the first one's count as one: keys of equal weight, such as those that have received nothing yet, would queue up)
  auto count = [&](uint32_t digit) {
    const bool like_first = digit == (uint32_t)__builtin_amdgcn_readfirstlane((int)digit);
    const uint64_t same = __ballot(like_first);
    if (!like_first) atomicAdd(&hist[digit], 1);
    else if (lane == (int)__builtin_ctzll(same)) atomicAdd(&hist[digit], __popcll(same));
  };

  // ---- the budget-th largest key
  uint32_t prefix = 0;
  int want = p.budget;  // of the keys that begin with `prefix`
  for (int pass = 0; pass < 3; pass++) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < 2048; i += kThreads) hist[i] = 0;
    __syncthreads();
    if (kCap > 0 && pass == 0) {
      // four slots a thread (a page holds 16 at least), the pages of its next ones asked for before
      constexpr int kAhead = 4;
      for (int q0 = tid * 4; q0 < L; q0 += kThreads * 4 * kAhead) {
        int64_t at[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
          const int q = q0 + i * kThreads * 4;
          const int page = page_in_pool(table[(q < L ? q : L - 1) >> p.c.page_log2], p.c.n_pages);
          at[i] = (((int64_t)page * p.c.HK + h) << p.c.page_log2) + (q & mask);
        }
        f32x4 w[kAhead];
        i32x4 pos[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++)
          if (q0 + i * kThreads * 4 < L) {
            w[i] = *reinterpret_cast<const f32x4*>(p.c.weights + at[i]);
            pos[i] = *reinterpret_cast<const i32x4*>(p.c.positions + at[i]);
          }
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
          const int q = q0 + i * kThreads * 4;
          if (q < L) {
            u32x4 k;
#pragma unroll
            for (int e = 0; e < 4; e++) {
              k[e] = pos[i][e] >= newest ? kNewest : ordered(w[i][e]);
              if (q + e < L) count(k[e] >> 21);
            }
            *reinterpret_cast<u32x4*>(keys + q) = k;
          }
        }
      }
    } else if (kCap > 0) {
      for (int q = tid * 4; q < L; q += kThreads * 4) {
        const u32x4 k = *reinterpret_cast<const u32x4*>(keys + q);
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (q + e < L && (k[e] >> (shift + bits)) == prefix) count((k[e] >> shift) & ((1 << bits) - 1));
      }
    } else {
#pragma unroll 4
      for (int j = tid; j < L; j += kThreads) {
        const uint32_t k = key_of(j);
        if (pass == 0 || (k >> (shift + bits)) == prefix) count((k >> shift) & ((1 << bits) - 1));
      }
    }
    __syncthreads();
    // thread t holds kBins digits from 2047 - kBins t down: prefix sums count from the largest digit on
    constexpr int kBins = 2048 / kThreads;
    int bin[kBins], mine = 0;
#pragma unroll
    for (int i = 0; i < kBins; i++) {
      bin[i] = hist[2047 - kBins * tid - i];
      mine += bin[i];
    }
    const int incl = wave_prefix_sum(mine);
    if (lane == 63) sums[0][wave] = incl;
    __syncthreads();
    int unused;
    int above = incl - mine + before_wave<kWaves>(sums[0], wave, &unused);
#pragma unroll
    for (int i = 0; i < kBins; i++) {
      if (above < want && want <= above + bin[i]) {
        found[0] = 2047 - kBins * tid - i;
        found[1] = above;
        found[2] = bin[i];
      }
      above += bin[i];
    }
    __syncthreads();
    prefix = (prefix << bits) | found[0];
    want -= (int)found[1];
    __syncthreads();  // (found and hist are written again)
  }
  const uint32_t edge = prefix;  // keys above it stay, and the first `want` that equal it

  // ---- slots in order: a wave takes a run of whole 64s
  const int run = (L + kThreads - 1) / kThreads * 64;
  const int j0 = wave * run, j1 = j0 + run < L ? j0 + run : L;
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  int ties_end = INT32_MAX;  // keys that equal the edge stay below this slot
  if ((int)found[2] > want) {
    int ties = 0;
    for (int j = j0 + lane; j < j1; j += 64) ties += key_of(j) == edge;
    ties = __builtin_amdgcn_readlane(wave_prefix_sum(ties), 63);
    if (lane == 0) sums[0][wave] = ties;
    __syncthreads();
    int unused;
    int tie = before_wave<kWaves>(sums[0], wave, &unused);
    if (tie < want && want <= tie + ties) {
      for (int j = j0 + lane; j - lane < j1; j += 64) {
        const bool tied = j < j1 && key_of(j) == edge;
        const uint64_t all = __ballot(tied);
        if (tied && tie + __popcll(all & below) == want - 1) found[0] = (uint32_t)j + 1;
        tie += __popcll(all);
      }
    }
    __syncthreads();
    ties_end = (int)found[0];
  }
  // A slot takes part in a move if it is below the budget and its key goes, or behind it and its key stays.  There are as many of the one kind as of the other, and
  // all of the first come before the second: one count in slot order numbers both.
  const auto moves_at = [&](int j) {
    const uint32_t k = key_of(j);
    return (k > edge || (k == edge && j < ties_end)) == (j >= p.budget);
  };
  int here = 0;
#pragma unroll 4
  for (int j = j0 + lane; j < j1; j += 64) here += moves_at(j);
  here = __builtin_amdgcn_readlane(wave_prefix_sum(here), 63);
  if (lane == 0) sums[1][wave] = here;
  __syncthreads();
  __shared__ int32_t own_moves[kMoveD > 0 ? 2 * kMovesPerGroup : 1];
  int32_t* const holes = kMoveD > 0 ? own_moves : p.moves + (int64_t)blockIdx.x * 2 * p.cap;
  const int cap = kMoveD > 0 ? kMovesPerGroup : p.cap;
  int all;
  int rank = before_wave<kWaves>(sums[1], wave, &all);
  const int moves = all / 2 < cap ? all / 2 : cap;  // (as many as the cap, by its definition)
  if (kMoveD == 0 && tid == 0) p.counts[blockIdx.x] = moves;
  constexpr int kAtOnce = 4;
  for (int j = j0 + lane; j - lane < j1; j += 64 * kAtOnce) {
    bool one[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; i++) one[i] = j + i * 64 < j1 && moves_at(j + i * 64);
#pragma unroll
    for (int i = 0; i < kAtOnce; i++) {
      const uint64_t ones = __ballot(one[i]);
      const int at = j + i * 64, n = rank + __popcll(ones & below), to = at < p.budget ? n : n - all / 2;
      if (one[i] && (unsigned)to < (unsigned)cap) holes[at < p.budget ? to : cap + to] = at;
      rank += __popcll(ones);
    }
  }
  if constexpr (kMoveD > 0) {
    __shared__ MoveSpots spots;
    __syncthreads();
    move_keys<kMoveD, kThreads>(p, b, h, holes, holes + cap, moves, spots);
  }
}

// A workgroup copies 64 of a head's moves.
template <int D>
__global__ void __launch_bounds__(256) paged_move_kernel(const EvictParams p) {
  __shared__ MoveSpots spots;
  const int pair = blockIdx.y, n = p.counts[pair];
  const int first = blockIdx.x * kMovesPerGroup;
  if (first >= n) return;
  const int32_t* const holes = p.moves + (int64_t)pair * 2 * p.cap;
  const int b = pair / p.c.HK;
  move_keys<D, 256>(p, b, pair - b * p.c.HK, holes + first, holes + p.cap + first, n - first < kMovesPerGroup ? n - first : kMovesPerGroup, spots);
}

struct EvictPlan {
  int cap;
  size_t bytes;
};
EvictPlan evict_plan(const fa_paged_evict_args* a) {
  const int max_keys = (int)std::min<int64_t>(a->cache.max_seqlen_k, (int64_t)a->cache.table_cols * a->cache.page_size);
  EvictPlan pl;
  pl.cap = std::max(0, std::min(a->budget, max_keys - a->budget));
  pl.bytes = (size_t)a->cache.batch * a->cache.nheads_k * ((size_t)2 * pl.cap + 1) * 4;
  return pl;
}

template <int D>
hipError_t launch_evict_d(const EvictParams& p, hipStream_t stream) {
  const dim3 pairs((unsigned)(p.c.B * p.c.HK));
  const bool few = p.cap <= kMovesPerGroup;  // (decoding: a step or a few of them over the budget)
  // (LDS decides how many heads a compute unit selects for at once: two, at more than 16384 keys one)
#define FA_EVICT(CAP)                                                                                             \
  do {                                                                                                            \
    if (few) hipLaunchKernelGGL((paged_evict_kernel<CAP, D>), pairs, dim3(kEvictThreads), 0, stream, p);          \
    else hipLaunchKernelGGL((paged_evict_kernel<CAP, 0>), pairs, dim3(kEvictThreads), 0, stream, p);              \
  } while (0)
  if (p.c.max_keys <= 4096) FA_EVICT(4096);
  else if (p.c.max_keys <= 16384) FA_EVICT(16384);
  else if (p.c.max_keys <= 32768) FA_EVICT(32768);
  else FA_EVICT(0);
#undef FA_EVICT
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || few) return e;
  const unsigned gx = (unsigned)((p.cap + kMovesPerGroup - 1) / kMovesPerGroup);
  hipLaunchKernelGGL(paged_move_kernel<D>, dim3(gx, pairs.x), dim3(256), 0, stream, p);  // (at most 65535 heads: see check_sizes)
  return hipGetLastError();
}
hipError_t launch_evict(const EvictParams& p, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 16: return launch_evict_d<16>(p, stream);
    case 32: return launch_evict_d<32>(p, stream);
    case 64: return launch_evict_d<64>(p, stream);
    case 128: return launch_evict_d<128>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

int check_sizes(const fa_paged_evict_args* a, const char* name) {
  FA_REQUIRE(a && a->struct_bytes == sizeof(fa_paged_evict_args), "%s: struct size mismatch", name);
  const int rc = check_paged_cache(&a->cache, false, false, false, name);
  if (rc) return rc;
  FA_REQUIRE(a->budget > 0 && a->recent >= 0, "%s: budget must be positive, recent not negative", name);
  FA_REQUIRE((int64_t)a->cache.batch * a->cache.nheads_k <= 65535, "%s: more than 65535 key heads of sequences", name);
  return FA_OK;
}

}  // namespace
}  // namespace fa

extern "C" {

size_t fa_paged_evict_workspace_bytes(const fa_paged_evict_args* a) {
  return fa::check_sizes(a, "fa_paged_evict") == FA_OK ? fa::evict_plan(a).bytes : 0;
}

int fa_paged_evict(const fa_paged_evict_args* a) {
  const char* const name = "fa_paged_evict";
  int rc = fa::check_sizes(a, name);
  if (rc == FA_OK) rc = fa::check_paged_cache(&a->cache, true, true, false, name);
  if (rc) return rc;
  const fa_paged_cache& c = a->cache;
  FA_REQUIRE(c.k_slot_stride >= c.head_dim && c.v_slot_stride >= c.head_dim && (c.nheads_k == 1 || (c.k_head_stride >= c.head_dim && c.v_head_stride >= c.head_dim)) &&
                 (c.n_pages == 1 || (c.k_page_stride >= c.head_dim && c.v_page_stride >= c.head_dim)),
             "%s: the cache's slots, heads and pages must not overlap", name);
  FA_REQUIRE(c.key_weights && c.key_positions && a->next_positions && a->new_seqlens_k, "%s: key_weights, key_positions, next_positions and new_seqlens_k are needed", name);
  FA_REQUIRE(fa::aligned16(c.key_weights) && fa::aligned16(c.key_positions), "%s: key_weights and key_positions must be 16-byte aligned", name);
  FA_REQUIRE(a->new_seqlens_k != c.seqlens_k, "%s: new_seqlens_k may not be seqlens_k", name);
  FA_REQUIRE(((reinterpret_cast<uintptr_t>(a->next_positions) | reinterpret_cast<uintptr_t>(a->new_seqlens_k)) & 3) == 0, "%s: integers must be 4-byte aligned", name);
  const fa::EvictPlan pl = fa::evict_plan(a);
  if (!a->workspace || a->workspace_bytes < pl.bytes || (reinterpret_cast<uintptr_t>(a->workspace) & 3))
    return fa::fail(FA_ERR_WORKSPACE, "%s: needs %zu bytes of 4-byte aligned workspace", name, pl.bytes);
  fa::EvictParams p{};
  p.c = fa::paged_cache(&c);
  p.next = a->next_positions;
  p.new_len = a->new_seqlens_k;
  p.budget = a->budget;
  p.recent = a->recent;
  p.cap = pl.cap;
  p.counts = reinterpret_cast<int32_t*>(a->workspace);
  p.moves = p.counts + (size_t)c.batch * c.nheads_k;
  FA_LAUNCH(fa::launch_evict(p, c.head_dim, reinterpret_cast<hipStream_t>(a->stream)));
  return FA_OK;
}

}  // extern "C"
