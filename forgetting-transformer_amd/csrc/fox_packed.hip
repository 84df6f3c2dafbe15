// Forgetting Attention over packed sequences for gfx950: forward and backward.
//
// The sequences lie one after the other, their ends in cu_q and cu_k on the device.  Query i of a sequence of m queries and n keys sees the keys
// j <= i + n - m of it; H query heads share Hk key heads, every query head has gates of its own:
//   s_ij = sm_scale q_i.k_j + c_i - c_j,  c_j = sum of the gates up to j,  o = softmax(s) v;  a row that sees no key is zero
//   dP = dO V^T,  delta_i = sum_j P_ij dP_ij,  dS = P (dP - delta),  dq = sm_scale dS K,  dk = sm_scale dS^T Q,  dv = P^T dO,
//   dc_j = -sum_i dS_ij  (a row of dS adds up to zero),  dg_l = sum_{j >= l} dc_j.
//
// Who knows how long the sequences are is the device.  Two workgroups make the plan, the lists of all tiles of queries and of keys, while the others form the
// sums of the gates; the attention kernels are launched for as many tiles as there can be (a partial one for every sequence) and those past the
// list end at once.  The longest walks come first.
//
// A tile whose walk is longer than a workgroup's share of all of them is cut into parts, each a workgroup's: long documents or pieces of long prompts next to short
// ones would otherwise be walked by a few workgroups at the end.  The part that arrives last adds them up, in their order.
//
// The gates' gradient is a difference of sums over whole rows and columns of dS, so it is formed from 32-bit values throughout, where the rest of the backward can
// live with the 16 bits of its operands:
// - c is kept in 64 bits; the kernels subtract a reference near their tile before they round.  Off the diagonal the reference lies between a tile's queries and its
//   keys, so that a bias is a sum of two terms of one sign and off by its own rounding.  On the diagonal two terms as large as the gates of 128 keys would cancel: there every
//   bias is the difference of two pairs of 32-bit numbers.  (One reference for all tiles and 32 bits: dg at gates of -2.1 off by 2e-4 of itself;
//   now sequences of 600 and 700 tokens, D 128 and 32, by 4e-6 and 5e-6 of its norm, gates of -3 by 1.3e-5, gates near 0 by 2e-6.)
// - The row sum of the forward adds the probabilities before they are rounded for the matrix instruction.
// - o.do is off by the rounding of o and of P; what is missing of delta is sum_j P_ij (dP_ij - o.do), which the dQ kernel has at its end.  It stores
//   the sum of the two for the dK/dV kernel.
#include <algorithm>
#include <cmath>

#include "fox_common.hpp"
#include "fox_kernels.hpp"
#include "fox_tiles.hpp"

namespace fox {

namespace {

constexpr int kPackedTile = 128;   // rows of a tile of either kind
static_assert(kPackedTile == kFwdBM && kPackedTile == kKvBN && kKvBM == kKvBN, "a tile is what a workgroup keeps");
// Log gates below this close like it: -inf itself would make the difference of two sums behind it undefined.  NaN stays NaN (fmaxf would drop it): so are the rows behind it then, and the
// gradients that such a row takes part in.
constexpr float kLowestGate = -1e6f;
__device__ __forceinline__ float bounded_gate(float g) { return g < kLowestGate ? kLowestGate : g; }
// Least shares, in 64 keys and 128 rows of a head (2 / 4 / 8, us: six pieces of up to 64 tokens behind up to 900, 12 heads 13.6 / 13.1 / 15.1, longer ones the same).
constexpr int kQueryShare = 4, kKeyShare = 4, kNoShare = 0x7fffffff;
// Parts for a share of units, at most, in halves: three from two shares on, four from one on.
constexpr int kQueryOver = 3, kKeyOver = 4;

// ---------------------------------------------------------------------------
// Plan
// ---------------------------------------------------------------------------
__device__ __forceinline__ int wave_max_scan(int x, int lane) {   // maximum over lanes 0 .. own, of values >= 0
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off);
    if (lane >= off) x = max(x, y);
  }
  return x;
}

__device__ __forceinline__ int wave_sum_scan(int x, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  return x;
}

// Place of a walk in the order of its group: shorter ones come later, in steps of a quarter of a power of two.
constexpr int kOrderLengths = 64, kOrderGroups = 16;
__device__ __forceinline__ int order_of(int units) {
  return kOrderLengths - 1 - min(max((int)(__float_as_uint((float)units) >> 21) - (127 << 2), 0), kOrderLengths - 1);
}

// How a walk of `units` is cut: parts of at most `share`, but no more than the root of the units, since one workgroup reads all parts again.  Where
// rows are the parts, part * ceil(units / parts) is below the units for every part: none is empty.
struct Share {
  int whole;       // walks up to this stay whole
  float inverse;   // of the share
};
__device__ __forceinline__ int parts_of(int units, Share share) {
  return units <= share.whole ? 1 : min((int)((float)units * share.inverse) + 1, (int)__builtin_amdgcn_sqrtf((float)units));
}
// x / y of integers below 2^24
__device__ __forceinline__ int quotient(int x, int y) {
  const int q = (int)((float)x * __builtin_amdgcn_rcpf((float)y)), r = x - q * y;
  return r < 0 ? q - 1 : r >= y ? q + 1 : q;
}
// Tiles of keys that a tile of queries walks
__device__ __forceinline__ int key_tiles(int m, int n, int tile) {
  const int hi = min(n, n - m + (tile + 1) * kPackedTile);
  return hi > 0 ? (hi + kFwdBN - 1) / kFwdBN : 0;
}
// First row, in steps, that a tile of keys walks, and the steps
__device__ __forceinline__ int first_row(int m, int n, int tile) { return max(tile * kKvBN - (n - m), 0) / kKvBM * kKvBM; }
__device__ __forceinline__ int row_steps(int m, int n, int tile) {
  const int lo = first_row(m, n, tile);
  return m > lo ? (m - lo + kKvBM - 1) / kKvBM : 0;
}
// The parts of a tile of keys: by the group's heads first (dc is a head's then), each head's rows only where there are more parts than heads.
struct KeyParts {
  int heads, rows, head_span, row_span;   // parts either way; heads and steps of a part
};
__device__ __forceinline__ KeyParts key_parts(int steps, int group, int parts) {
  KeyParts p;
  const int heads = min(parts, group), rows = max(min(quotient(parts, group), steps), 1);
  p.head_span = quotient(group + heads - 1, heads);
  p.heads = quotient(group + p.head_span - 1, p.head_span);
  p.row_span = max(quotient(steps + rows - 1, rows), 1);
  p.rows = max(quotient(steps + p.row_span - 1, p.row_span), 1);
  return p;
}

// At least the units of a sequence's tiles of queries (keys), in 64 keys (128 rows of a head).
__device__ __forceinline__ int64_t query_units(int m, int n) {
  const int64_t p = (int64_t)n - m, tiles = (m + kPackedTile - 1) / kPackedTile, t0 = p < 0 ? min(-p / kPackedTile, tiles) : 0, c = tiles - t0;
  return (c * p + c * (t0 + tiles + 1) * (kPackedTile / 2) + kFwdBN - 1) / kFwdBN + c;
}
__device__ __forceinline__ int64_t key_units(int m, int n, int group) {
  const int64_t p = (int64_t)n - m, tiles = (n + kPackedTile - 1) / kPackedTile, a = p < 0 ? 0 : min(p / kPackedTile + 1, tiles), c = tiles - a;
  return ((a * m + c * n - c * (a + tiles - 1) * (kPackedTile / 2)) / kKvBM + 2 * tiles) * group;
}

constexpr int kNearSequences = 128;   // so many lie in LDS
struct PlanMemory {
  int4 seqs[kNearSequences];
  int buckets[kOrderGroups * kOrderLengths];
  unsigned long long units;
  int slots, top[2][16], waves[16];
};

// An end of a sequence among `rows` rows.  One behind them is left out: cut to them, its sequence would be aligned at another key.
__device__ __forceinline__ int end_within(int end, int rows) { return end > rows ? 0 : max(end, 0); }

// The list of the tiles of queries, or of those of keys, by one workgroup of NT threads.  Ends that decrease are brought into order and those outside the tensors left out, so
// that no tile leaves them.
template <int NT, bool KEYS>
__device__ __forceinline__ void make_plan(const PackedK& a, PlanMemory& mem) {
  constexpr int WAVES = NT / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), S = a.B + kPackedOuter;
  const int extra = KEYS ? a.k_extra : a.q_extra;
  const bool near = S <= kNearSequences;
  int4* const seqs = near ? mem.seqs : a.plan.seqs + (KEYS ? S : 0);
  static_assert(NT == kOrderGroups * kOrderLengths, "a bucket a thread");
  mem.buckets[tid] = 0;
  if (tid == 0) {
    mem.units = 0;
    mem.slots = 0;
  }
  if (!KEYS) {
    for (int i = tid; i < a.q_extra * a.H; i += NT) a.q_arrived[i] = 0;
  }
  int top_q = 0, top_k = 0;   // largest end so far
  int64_t units = 0;
  for (int b0 = 0; b0 < a.B; b0 += NT) {
    const int b = b0 + tid;
    const bool in = b < a.B;
    auto q_end = [&](int i) { return in ? end_within(a.cu_q[i], a.T) : 0; };
    auto k_end = [&](int i) { return in ? end_within(a.cu_k[i], a.N) : 0; };
    const int sq = q_end(b), sk = k_end(b), last_q = q_end(b + 1), last_k = k_end(b + 1);
    int q = wave_max_scan(sq, lane), k = wave_max_scan(sk, lane);
    __syncthreads();
    if (lane == 63) {
      mem.top[0][wave] = q;
      mem.top[1][wave] = k;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
      q = max(q, mem.top[0][w]);
      k = max(k, mem.top[1][w]);
    }
    q = max(q, top_q);
    k = max(k, top_k);
    const int q1 = max(q, last_q), k1 = max(k, last_k);
    if (in) {
      const int4 s = make_int4(q, q1 - q, k, k1 - k);
      seqs[b] = s;
      if (near && !KEYS) a.plan.seqs[b] = s;
      units += KEYS ? key_units(s.y, s.w, a.group) : query_units(s.y, s.w);
      // what belongs to none of them
      if (b == 0) {
        seqs[a.B] = make_int4(0, q, 0, 0);
        seqs[a.B + 2] = make_int4(0, 0, 0, k);
      }
      if (b == a.B - 1) {
        seqs[a.B + 1] = make_int4(q1, a.T - q1, 0, 0);
        seqs[a.B + 3] = make_int4(0, 0, k1, a.N - k1);
      }
    }
    for (int w = 0; w < WAVES; ++w) {
      top_q = max(top_q, mem.top[0][w]);
      top_k = max(top_k, mem.top[1][w]);
    }
  }
  if (units > 0) atomicAdd(&mem.units, (unsigned long long)units);
  __syncthreads();
  if (near && !KEYS && tid < kPackedOuter) a.plan.seqs[a.B + tid] = seqs[a.B + tid];
  // A workgroup's share: so many that no more parts than `extra` come of it.  Walks of queries stay whole up to two shares: the longest start first, and
  // a part costs a start and a merge.  (Two / one, us: 8 x 768 tokens, 12 heads, D 64: forward 22.3 / 29.0, dQ 28.6 / 37.2; pieces of prompts of up to 12800 keys 155 / 170; documents of
  // 150 to 2048 tokens 34.8 / 36.0 and 44.1 / 45.9.  dK/dV of those, whose workgroups are fewer and walk in longer steps: 63.6 / 49.0.)
  Share share{kNoShare, 0.f};
  if (extra > 0) {
    const unsigned long long u = max(((KEYS ? kKeyOver : kQueryOver) * mem.units / 2 + extra) / extra, (unsigned long long)(KEYS ? kKeyShare : kQueryShare));
    share.whole = (int)min(KEYS ? u : 2 * u, (unsigned long long)kNoShare);
    share.inverse = 1.0f / (float)u;
  }
  auto tiles_of = [&](int4 s) { return ((KEYS ? s.w : s.y) + kPackedTile - 1) / kPackedTile; };
  // sequences whose keys (queries) an XCD's cache holds together are a group; within it the longest walks come first
  const int groups = KEYS ? a.k_groups : a.q_groups;
  const float per_token = (float)groups / (float)(KEYS ? a.T : a.N);
  struct Tile {
    int parts, bucket;
  };
  auto tile_of = [&](int4 s, int t) {
    const int steps = KEYS ? row_steps(s.y, s.w, t) : 0, units = KEYS ? steps * a.group : key_tiles(s.y, s.w, t);
    Tile r;
    r.parts = parts_of(units, share);
    const int first = min((int)((float)(KEYS ? s.x : s.z) * per_token), groups - 1) * kOrderLengths;
    r.bucket = first + order_of(r.parts > 1 ? quotient(min(units, 1 << 23), r.parts) : units);
    if (KEYS && r.parts > 1) {
      const KeyParts p = key_parts(steps, a.group, r.parts);
      r.parts = p.heads * p.rows;
    }
    return r;
  };
  // Every tile of every sequence: a lane takes those of a short one, the lanes of a wave those of a long one.
  auto each_tile = [&](auto&& f) {
    for (int b0 = 0; b0 < S; b0 += NT) {
      const int b = b0 + lane * WAVES + wave;
      const int4 s = b < S ? seqs[b] : make_int4(0, 0, 0, 0);
      const int tiles = tiles_of(s);
      constexpr int SHORT = 4;
      for (int t = 0; t < (tiles <= SHORT ? tiles : 0); ++t) f(s, t);
      for (uint64_t left = __ballot(tiles > SHORT); left; left &= left - 1) {
        const int from = __builtin_ctzll(left);
        const int4 w = make_int4(__builtin_amdgcn_readlane(s.x, from), __builtin_amdgcn_readlane(s.y, from), __builtin_amdgcn_readlane(s.z, from),
                                 __builtin_amdgcn_readlane(s.w, from));
        for (int t = lane, n = tiles_of(w); t < n; t += 64) f(w, t);
      }
    }
  };
  // parts of a bucket, their first places, and each tile's among them (any order within a bucket)
  each_tile([&](int4 s, int t) {
    const Tile x = tile_of(s, t);
    atomicAdd(&mem.buckets[x.bucket], x.parts);
  });
  __syncthreads();
  const int own = mem.buckets[tid];
  int end = wave_sum_scan(own, lane);
  if (lane == 63) mem.waves[wave] = end;
  __syncthreads();
  for (int w = 0; w < wave; ++w) end += mem.waves[w];
  mem.buckets[tid] = end - own;
  if (tid == NT - 1) {
    a.plan.counts[KEYS] = end;
    if (!KEYS && !a.lse) a.plan.counts[1] = 0;   // (a backward of it all the same finds no tiles)
  }
  __syncthreads();
  PackedItem* const items = KEYS ? a.plan.k_items : a.plan.q_items;
  each_tile([&](int4 s, int t) {
    const Tile x = tile_of(s, t);
    PackedItem* const at = items + atomicAdd(&mem.buckets[x.bucket], x.parts);
    PackedItem it{s.x, s.y, s.z, s.w, t, 0, x.parts, 0};
    if (x.parts > 1) it.slot = atomicAdd(&mem.slots, x.parts);
    for (; it.part < x.parts; ++it.part) at[it.part] = it;
  });
}

// ---------------------------------------------------------------------------
// Sums of the gates
// ---------------------------------------------------------------------------
// Running sums of one row of n values by NT threads, from its first element on or from its last.  fp64; load(j) and store(j, sum) take the place in the row.
// Lanes take neighbouring places, so that a line of (N, H) gates is fetched once for the two or more tokens in it (eight places a lane: 12800 tokens of 16 heads 20.0 us for 13.8).
// Bound by the CU's own path to L2: a row is one workgroup's, and it reads the gates of all heads for its own.
template <int NT, bool REVERSE, typename Load, typename Store>
__device__ __forceinline__ void sum_row(int n, Load load, Store store) {
  constexpr int PER = 8, WAVES = NT / 64;
  __shared__ double wave_tot[2][WAVES];
  const int tid = threadIdx.x % NT, lane = tid & 63, wave = tid >> 6;
  double carry = 0.0;
  int turn = 0;
  for (int base = 0; base < n; base += NT * PER, turn ^= 1) {
    const int at = base + wave * 64 * PER + lane;   // a wave's places follow each other, and so do those of a load
    float x[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int i = min(at + 64 * e, n - 1), j = REVERSE ? n - 1 - i : i;
      x[e] = load(j);
    }
    double v[PER], run = 0.0;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const double incl = wave_scan(at + 64 * e < n ? (double)x[e] : 0.0);
      v[e] = run + incl;
      run += of_lane(incl, 63);
    }
    double before = carry, total = run;
    if constexpr (WAVES > 1) {
      if (lane == 63) wave_tot[turn][wave] = run;
      __syncthreads();   // (the other buffer of the two was read in front of it)
      total = 0.0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const double t = wave_tot[turn][w];
        if (w < wave) before += t;
        total += t;
      }
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if (at + 64 * e < n) store(REVERSE ? n - 1 - (at + 64 * e) : at + 64 * e, before + v[e]);
    }
    carry += total;
  }
}

__device__ __forceinline__ int wave_max(int x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x = max(x, __shfl_xor(x, off));
  return x;
}
// Where the keys of sequence b <= B begin: behind every earlier end, as in the plan, so that no two rows have a place in common.  b is a wave's, b0 that of the workgroup's first one.  Every
// thread of the workgroup of NT calls it.  Ends that do not decrease cost the comparisons alone, without the maxima (the launch without / with them, us: 64 sequences
// of 100 tokens, 16 heads, 8.2 / 9.2, 4096 of 8, 12 heads, 25 / 31, up to 24 sequences the same).
template <int NT>
__device__ __forceinline__ int first_key(const PackedK& a, int b0, int b) {
  __shared__ int tops[NT / 64];
  const int tid = threadIdx.x, lane = tid & 63;
  auto end = [&](int i) { return end_within(a.cu_k[i], a.N); };
  const int at = end(b0), own = b < a.B ? end(b) : 0;
  int top = 0;
  for (int i = tid; i < b0; i += NT) top = max(top, end(i));
  top = __any(top > at) ? wave_max(top) : 0;
  if (lane == 0) tops[tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) top = max(top, tops[w]);
  for (int i0 = b0; i0 < b; i0 += 64) {
    const int x = i0 + lane < b ? end(i0 + lane) : 0;
    if (__any(x > own)) top = max(top, wave_max(x));
  }
  return max(top, own);
}

}  // namespace

// The first workgroups make the plan (that of the keys only where a backward may follow), the others the sums of a (sequence, head) each; with NT = 64 of sixteen.
template <int NT>
__global__ __launch_bounds__(1024) void packed_scan_kernel(const PackedK a) {
  constexpr int THREADS = 1024;
  __shared__ PlanMemory mem;
  const int plans = a.lse ? 2 : 1;
  if (blockIdx.x == 0) return make_plan<THREADS, false>(a, mem);
  if (blockIdx.x < plans) return make_plan<THREADS, true>(a, mem);
  const int row0 = (blockIdx.x - plans) * (THREADS / NT), row = row0 + threadIdx.x / NT;
  const int b = divide(row, a.by_heads), h = row - b * a.H;
  const int k0 = first_key<THREADS>(a, divide(row0, a.by_heads), min(b, a.B));
  if (row >= a.B * a.H) return;
  const int n = max(end_within(a.cu_k[b + 1], a.N), k0) - k0;
  const float* g = a.g + (int64_t)k0 * a.g_st + h * a.g_sh;
  double* c = a.c + (int64_t)h * a.N + k0;
  sum_row<NT, false>(n, [&](int j) { return bounded_gate(g[j * a.g_st]); }, [&](int j, double sum) { c[j] = sum; });
}

// The backward's counters of arrived parts: its own, since two of one forward may run at once.  (Those of the forward are cleared next to its plan.)
__global__ __launch_bounds__(256) void packed_clear_kernel(const PackedK a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < a.q_extra * a.H) a.q_arrived[i] = 0;
  if (i < a.k_extra * a.Hk) a.k_arrived[i] = 0;
}

// dg of a (sequence, head) from dc.  The first gate of a sequence moves all its sums alike: an exact zero, as in the rows that belong to none, but NaN where one of the sums is.
template <int NT>
__global__ __launch_bounds__(1024) void packed_gate_grad_kernel(const PackedK a) {
  constexpr int THREADS = 1024;
  const int row = blockIdx.x * (THREADS / NT) + threadIdx.x / NT;
  if (row >= (a.B + kPackedOuter) * a.H) return;
  const int b = divide(row, a.by_heads), h = row - b * a.H;
  const int4 s = a.plan.seqs[b];
  const float* dc = a.dc + (int64_t)h * a.N + s.z;
  float* dg = a.dg + (int64_t)s.z * a.dg_st + h * a.dg_sh;
  const bool none = b >= a.B;
  sum_row<NT, true>(s.w, [&](int j) { return dc[j]; }, [&](int j, double sum) { dg[j * a.dg_st] = none || (j == 0 && sum == sum) ? 0.f : (float)sum; });
}

namespace {

// Item and head of a workgroup: the heads of an XCD are next to each other where 8 divides them, so that those of a group, which read the same keys, share
// its L2, and all tiles of a head follow each other there.  `heads` is fixed for a launch, by_heads and by_xcd_heads are its divisors.
__device__ __forceinline__ void packed_block(const PackedK& a, int heads, int& item, int& head) {
  const uint32_t id = blockIdx.x;
  if (heads % kXcds == 0) {
    const int r = (int)(id / kXcds), per = heads / kXcds;
    item = divide(r, a.by_xcd_heads);
    head = (int)(id % kXcds) * per + r - item * per;
  } else {
    item = divide((int)id, a.by_heads);
    head = (int)id - item * heads;
  }
}

}  // namespace

// ---------------------------------------------------------------------------
// Tiles at the diagonal: scores with the biases as differences of pairs, masked (the others: fox_tiles.hpp)
// ---------------------------------------------------------------------------
namespace {

// A 64-bit number of log2 units as two of 32 bits.
struct Pair {
  float hi, lo;
};
__device__ __forceinline__ Pair pair_of(double x) {
  const float hi = (float)x;
  return {hi, (float)(x - (double)hi)};
}
constexpr double kLog2eD = 1.4426950408889634074;

// x[r] = s[r] scale + (row - column) with the pairs of rows (or columns) c_row(r, g) in LDS; sign -1: LDS holds the columns.
template <int SIGN>
__device__ __forceinline__ void add_pairs(f32x16& s, const float* hi_s, const float* lo_s, int at, int g, Pair own, float scale) {
#pragma unroll
  for (int q4 = 0; q4 < 4; ++q4) {   // (four at a time: all of them at once do not fit the registers of dQ at head dim 128)
    const f32x4 hi = *reinterpret_cast<const f32x4*>(&hi_s[at + 8 * q4 + 4 * g]), lo = *reinterpret_cast<const f32x4*>(&lo_s[at + 8 * q4 + 4 * g]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      s[4 * q4 + e] = fmaf(s[4 * q4 + e], scale, SIGN > 0 ? (hi[e] - own.hi) + (lo[e] - own.lo) : (own.hi - hi[e]) + (own.lo - lo[e]));
    __builtin_amdgcn_sched_barrier(0);
  }
}
template <typename Tr, int D>
__device__ __forceinline__ f32x16 dots(const char* tile, int row0, const u32x4 (&reg)[D / 16], f32x16 s, int lane) {
  const int g = lane >> 5, i = lane & 31;
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) s = Tr::mfma32(lds_row_operand<D>(tile, row0 + i, 2 * kk + g), reg[kk], s);
  return s;
}
__device__ __forceinline__ f32x16 splat(float x) {
  f32x16 v;
#pragma unroll
  for (int r = 0; r < 16; ++r) v[r] = x;
  return v;
}

// A running maximum and sum for every 32 keys: those above the rows of the wave cost nothing, and only those at the diagonal are masked.
template <typename Tr, int D>
__device__ __forceinline__ void packed_fwd_tile(const char* k_tile, const char* v_tile, const float* hi_s, const float* lo_s, const u32x4 (&qreg)[D / 16],
                                                f32x16 (&oacc)[(D + 31) / 32], float& m_i, float& l_i, int n0, int a_m, int a_w0, Pair row, float qk_scale, int lane) {
  constexpr int BN = kFwdBN, DB = (D + 31) / 32, NB = BN / 32;
  const int g = lane >> 5;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int nb0 = n0 + 32 * nb;
    if (nb0 > a_w0 + 31) continue;
    f32x16 s = dots<Tr, D>(k_tile, 32 * nb, qreg, splat(0.f), lane);
    add_pairs<-1>(s, hi_s, lo_s, 32 * nb, g, row, qk_scale);
    if (nb0 + 31 > a_w0) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = nb0 + c_row(r, g) > a_m ? -INFINITY : s[r];
    }
    float mloc = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mloc = fmaxf(mloc, s[r]);
    mloc = half_max(mloc);
    const bool raise = mloc > m_i + kLazyMaxLog2;
    if (__any(raise)) {
      const float m_new = raise ? mloc : m_i, alpha = __builtin_amdgcn_exp2f(m_i - m_new);
      m_i = m_new;
      l_i *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[db][r] *= alpha;
    }
    float rsum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = __builtin_amdgcn_exp2f(s[r] - m_i);
      rsum += s[r];
    }
    l_i += rsum;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const u32x4 pb = pack8<Tr>(s, 8 * hh);
#pragma unroll
      for (int db = 0; db < DB; ++db) oacc[db] = Tr::mfma32(lds_col_operand<D>(v_tile, 32 * nb + 16 * hh, db, lane), pb, oacc[db]);
    }
  }
}

// Off the diagonal of a tile that every row of the wave sees: cn_s holds the start values of the score accumulators, rowc the row's term.  (dq_tile without its causal
// part, whose row positions the registers of head dim 128 have no room for.)
template <typename Tr, int D>
__device__ __forceinline__ void packed_dq_interior(const char* k_tile, const char* v_tile, const float* cn_s, const u32x4 (&qreg)[D / 16], const u32x4 (&doreg)[D / 16],
                                                   f32x16 (&dqacc)[(D + 31) / 32], float& rows, float qk_scale, float rowc, float delta, int lane) {
  constexpr int BN = kFwdBN, DB = (D + 31) / 32, NB = BN / 32;
  const int g = lane >> 5;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    f32x16 s = dots<Tr, D>(k_tile, 32 * nb, qreg, acc_init(cn_s, 32 * nb, g), lane);
    f32x16 dp = dots<Tr, D>(v_tile, 32 * nb, doreg, splat(-delta), lane);
    float rsum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      dp[r] *= __builtin_amdgcn_exp2f(fmaf(s[r], qk_scale, rowc));
      rsum += dp[r];
    }
    rows += rsum;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const u32x4 dsb = pack8<Tr>(dp, 8 * hh);
#pragma unroll
      for (int db = 0; db < DB; ++db) dqacc[db] = Tr::mfma32(lds_col_operand<D>(k_tile, 32 * nb + 16 * hh, db, lane), dsb, dqacc[db]);
    }
  }
}

// `row`: of the query, its log-normaliser taken off.  `all`: the wave's rows see these 32 keys at most, so that what is missing of delta is known in time for dq too (sequences of 2 tokens,
// D 64: dq off by 3.7e-3, now 2.4e-3; on longer walks it averages out).
template <typename Tr, int D>
__device__ __forceinline__ void packed_dq_tile(const char* k_tile, const char* v_tile, const float* hi_s, const float* lo_s,
                                               const u32x4 (&qreg)[D / 16], const u32x4 (&doreg)[D / 16], f32x16 (&dqacc)[(D + 31) / 32], float& rows, int n0, int a_m, int a_w0, Pair row,
                                               float qk_scale, float delta, bool all, int lane) {
  constexpr int BN = kFwdBN, DB = (D + 31) / 32, NB = BN / 32;
  const int g = lane >> 5;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int nb0 = n0 + 32 * nb;
    if (nb0 > a_w0 + 31) continue;   // entirely above this wave's rows
    f32x16 s = dots<Tr, D>(k_tile, 32 * nb, qreg, splat(0.f), lane);
    add_pairs<-1>(s, hi_s, lo_s, 32 * nb, g, row, qk_scale);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r]);
    if (nb0 + 31 > a_w0) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = nb0 + c_row(r, g) > a_m ? 0.f : s[r];
    }
    f32x16 dp = dots<Tr, D>(v_tile, 32 * nb, doreg, splat(-delta), lane);
    float rsum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      dp[r] *= s[r];
      rsum += dp[r];
    }
    rows += rsum;
    if (all) {
      const float missing = half_sum(rsum);
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] = fmaf(-s[r], missing, dp[r]);
    }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const u32x4 dsb = pack8<Tr>(dp, 8 * hh);
#pragma unroll
      for (int db = 0; db < DB; ++db) dqacc[db] = Tr::mfma32(lds_col_operand<D>(k_tile, 32 * nb + 16 * hh, db, lane), dsb, dqacc[db]);
    }
  }
}

struct Rows {                          // of a step of dK/dV in LDS, log-normalisers taken off
  alignas(16) float rc[kKvBM];         // start values of the score accumulators
  alignas(16) float hi[kKvBM];         // at the diagonal: pairs
  alignas(16) float lo[kKvBM];
  alignas(16) float dl[kKvBM];         // -delta
};

template <typename Tr, int D>
__device__ __forceinline__ void packed_dkdv_step(const char* q_tile, const char* do_tile, const Rows& rows, bool diagonal, const u32x4 (&kreg)[D / 16], const u32x4 (&vreg)[D / 16],
                                                 f32x16 (&dkacc)[(D + 31) / 32], f32x16 (&dvacc)[(D + 31) / 32], float& csum, int a_s0, int n, int n_w0, Pair col,
                                                 float qk_scale, int lane) {
  constexpr int DB = (D + 31) / 32, MB = kKvBM / 32;
  const int g = lane >> 5;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int a_b0 = a_s0 + 32 * mb;
    if (a_b0 + 31 < n_w0) continue;   // entirely above the diagonal for this wave
    f32x16 s;
    if (diagonal) {
      s = dots<Tr, D>(q_tile, 32 * mb, kreg, splat(0.f), lane);
      add_pairs<1>(s, rows.hi, rows.lo, 32 * mb, g, col, qk_scale);
    } else {
      s = dots<Tr, D>(q_tile, 32 * mb, kreg, acc_init(rows.rc, 32 * mb, g), lane);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], qk_scale, -col.hi);
    }
    f32x16 dp = dots<Tr, D>(do_tile, 32 * mb, vreg, acc_init(rows.dl, 32 * mb, g), lane);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r]);
    if (a_b0 < n_w0 + 31) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = n > a_b0 + c_row(r, g) ? 0.f : s[r];
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      dp[r] *= s[r];
      csum += dp[r];
    }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const u32x4 pb = pack8<Tr>(s, 8 * hh), dsb = pack8<Tr>(dp, 8 * hh);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        dvacc[db] = Tr::mfma32(lds_col_operand<D>(do_tile, 32 * mb + 16 * hh, db, lane), pb, dvacc[db]);
        dkacc[db] = Tr::mfma32(lds_col_operand<D>(q_tile, 32 * mb + 16 * hh, db, lane), dsb, dkacc[db]);
      }
    }
  }
}

}  // namespace

// ---------------------------------------------------------------------------
// Parts of a walk: accumulators of 128 rows as the waves hold them, then two numbers a row; read and written past the L2 of an XCD (fox_common.hpp)
// ---------------------------------------------------------------------------
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
template <int D> constexpr int kAccFloats = (D + 31) / 32 * 32 * kPackedTile;
template <int D> constexpr int kQueryPartFloats = kAccFloats<D> + 2 * kPackedTile;       // forward: maximum and sum; dQ: row sum of dS
template <int D> constexpr int kKeyPartFloats = 2 * kAccFloats<D> + kPackedTile;         // dK, dV; dc

template <int DB>
__device__ __forceinline__ void store_part(float* part, const f32x16 (&acc)[DB], int wave, int lane) {
  double* at = reinterpret_cast<double*>(part) + wave * DB * 512 + lane;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; r += 2) store_agent(at + db * 512 + r * 32, __builtin_bit_cast(double, f32x2{acc[db][r], acc[db][r + 1]}));
}
template <int DB>
__device__ __forceinline__ void add_part(const float* part, f32x16 (&acc)[DB], float weight, int wave, int lane) {
  const double* at = reinterpret_cast<const double*>(part) + wave * DB * 512 + lane;
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    double x[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) x[r] = load_agent(at + db * 512 + r * 64);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const f32x2 y = __builtin_bit_cast(f32x2, x[r]);
      acc[db][2 * r] = fmaf(y[0], weight, acc[db][2 * r]);
      acc[db][2 * r + 1] = fmaf(y[1], weight, acc[db][2 * r + 1]);
    }
  }
}
template <int DB>
__device__ __forceinline__ void clear(f32x16 (&acc)[DB]) {
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = splat(0.f);
}
// Whether this workgroup is the last of a tile's parts to arrive.  Every thread calls it, behind its stores.
__device__ __forceinline__ bool last_part(uint32_t* arrived, int parts) {
  __shared__ bool last;
  stores_complete();
  __syncthreads();
  if (threadIdx.x == 0) last = arrive(arrived) == (uint32_t)parts - 1u;
  __syncthreads();
  return last;
}
// The tiles of keys [begin, end) of a part, those of the last keys in part 0.
struct Walk {
  int begin, end;
};
__device__ __forceinline__ Walk walk_of(const PackedItem& it) {
  const int tiles = key_tiles(it.m, it.n, it.tile);
  if (it.parts == 1) return {0, tiles};
  const int span = (tiles + it.parts - 1) / it.parts, end = tiles - it.part * span;
  return {max(end - span, 0), end};
}

}  // namespace

// ---------------------------------------------------------------------------
// Forward: four waves, 32 query rows each, K and V tiles of 64 keys in two alternating LDS buffers, the tiles at the diagonal one by one and
// the others software-pipelined (the tile code and its reasons: fox_tiles.hpp, fox_fwd.hip).
// Bound by the matrix units and, at head dim 64 and below, by the exponentials as much.  One sequence of 16384 tokens, 12 heads, D 64 855 TFLOP/s; 8 of about 3000, 16 heads, D 128 890 to 1040
// (by the box); 8 of 2048, 12 heads, D 64 88 us, 590 TFLOP/s, where starts and the last workgroups weigh.
// ---------------------------------------------------------------------------
template <typename Tr, int D>
__global__ __launch_bounds__(256, D <= 64 ? 3 : 2) void packed_fwd_kernel(const PackedK a) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int BM = kFwdBM, BN = kFwdBN, KK = D / 16, DB = (D + 31) / 32, NB = BN / 32;
  __shared__ __align__(16) char k_tile0[Tile<D>::bytes(BN)];
  __shared__ __align__(16) char k_tile1[Tile<D>::bytes(BN)];
  __shared__ __align__(16) char v_tile0[Tile<D>::bytes(BN)];
  __shared__ __align__(16) char v_tile1[Tile<D>::bytes(BN)];
  __shared__ __align__(16) float cn_s0[BN];
  __shared__ __align__(16) float cn_s1[BN];
  __shared__ __align__(16) float lo_s0[BN];
  __shared__ __align__(16) float lo_s1[BN];
  int item, h;
  packed_block(a, a.H, item, h);
  const PackedItem it = a.plan.q_items[item];   // (next to their count: there is memory for as many as the launch has)
  if (item >= a.plan.counts[0]) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5, i = lane & 31;
  const int M = it.m, N = it.n, p_seq = N - M, m0 = it.tile * BM;
  const int hk = h / a.group;
  const double* c_row = a.c + (int64_t)h * a.N + it.k0;
  const uint16_t* qp = a.q.ptr + (int64_t)it.q0 * a.q.st + h * a.q.sh;
  const uint16_t* kp = a.k.ptr + (int64_t)it.k0 * a.k.st + hk * a.k.sh;
  const uint16_t* vp = a.v.ptr + (int64_t)it.k0 * a.v.st + hk * a.v.sh;
  uint16_t* op = const_cast<uint16_t*>(a.o.ptr) + (int64_t)it.q0 * a.o.st + h * a.o.sh;
  const int a0 = p_seq + m0;   // key position of the first row
  const int m = m0 + 32 * wave + i, a_m = p_seq + m, a_w0 = a0 + 32 * wave;
  const float qk_scale = nonzero_scale(a.sm_scale * kLog2e), inv_scale = 1.0f / qk_scale;
  const bool wave_has_rows = m0 + 32 * wave < M;

  const DirectTileLoader<D, BN, 4, 0> kld(a.k.st, wave, lane), vld(a.v.st, wave, lane);
  const Walk walk = walk_of(it);   // from the last tile down
  const int n_tiles = walk.end, t_begin = walk.begin;
  f32x16 oacc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) oacc[db][r] = 0.f;
  float m_i = -3.0e38f, l_i = 0.f;   // (finite: a row that has seen no key yet yields exp2(-inf) = 0)
  if (n_tiles > 0) {
    kld.issue(kp, a.k.st, (n_tiles - 1) * BN, N, k_tile0);
    vld.issue(vp, a.v.st, (n_tiles - 1) * BN, N, v_tile0);
    u32x4 qreg[KK];
    load_row_operand_regs<D>(qreg, qp, a.q.st, m, M, g);
    const double c_ref = c_row[min(max(a0, 0), N - 1)];
    // the key terms of a tile: requested here, worked out where they go to LDS, a tile later
    double cn_raw = 0.0;
    bool cn_ok = false;
    auto issue_cn = [&](int n0) {
      if (tid < BN) {
        cn_ok = n0 + tid < N;
        cn_raw = c_row[min(n0 + tid, N - 1)];
      }
    };
    // at the diagonal a pair, elsewhere the start value of the score accumulators; keys past the last one get a probability of zero
    auto store_pair = [&](float* hi, float* lo) {
      const Pair c = pair_of((cn_raw - c_ref) * kLog2eD);
      hi[tid] = cn_ok ? c.hi : INFINITY;
      lo[tid] = cn_ok ? c.lo : 0.f;
    };
    auto cn_term = [&]() { return cn_ok ? (float)(c_ref - cn_raw) * kLog2e * inv_scale : -INFINITY; };   // (the scale is positive where it is used)
    auto issue = [&](int n0, char* kt, char* vt) {
      issue_cn(n0);   // small load first: the counter of loads retires in order
      kld.issue(kp, a.k.st, n0, N, kt);
      vld.issue(vp, a.v.st, n0, N, vt);
    };
    issue_cn((n_tiles - 1) * BN);
    const Pair row = pair_of((c_row[min(max(a_m, 0), N - 1)] - c_ref) * kLog2eD);
    auto compute = [&](int n0, const char* kt, const char* vt, const float* hi, const float* lo) {
      if (n0 > a_w0 + 31 || !wave_has_rows) return;   // tile entirely above this wave's rows
      packed_fwd_tile<Tr, D>(kt, vt, hi, lo, qreg, oacc, m_i, l_i, n0, a_m, a_w0, row, qk_scale, lane);
    };
    // tiles at the diagonal; all of them where the pipelined code, which needs a positive scale and a few tiles, is not entered
    int n_diag = 0;
    while (n_diag < n_tiles - t_begin && (n_tiles - 1 - n_diag) * BN + BN - 1 > a0) ++n_diag;
    if (!(qk_scale > 0.f) || n_tiles - t_begin - n_diag < kMinPipelinedTiles) n_diag = n_tiles - t_begin;
    const int t_stop = n_tiles - n_diag, n_int = t_stop - t_begin;
    if (n_diag > 0 && tid < BN) store_pair(cn_s0, lo_s0);
    for (int t = n_tiles - 1; t >= t_stop; t -= 2) {
      wait_vmem_all();
      __syncthreads();
      if (t - 1 >= t_stop) issue((t - 1) * BN, k_tile1, v_tile1);
      compute(t * BN, k_tile0, v_tile0, cn_s0, lo_s0);
      if (t - 1 < t_stop) break;
      if (tid < BN) store_pair(cn_s1, lo_s1);
      wait_vmem_all();
      __syncthreads();
      if (t - 2 >= t_stop) issue((t - 2) * BN, k_tile0, v_tile0);
      compute((t - 1) * BN, k_tile1, v_tile1, cn_s1, lo_s1);
      if (t - 2 >= t_stop && tid < BN) store_pair(cn_s0, lo_s0);
    }
    if (n_int > 0) {   // K runs one tile ahead of V: iteration j computes S(j + 1) and P(j) V(j)
      auto int_n0 = [&](int j) { return (t_stop - 1 - j) * BN; };
      auto issue_k = [&](int j, char* kt) {
        issue_cn(int_n0(j));
        kld.issue(kp, a.k.st, int_n0(j), N, kt);
      };
      if (n_diag > 0) {
        __syncthreads();   // every wave is done with every buffer
        issue_k(0, k_tile0);
      }
      if (tid < BN) cn_s0[tid] = cn_term();
      wait_vmem_all();
      __syncthreads();
      if (n_int > 1) issue_k(1, k_tile1);
      vld.issue(vp, a.v.st, int_n0(0), N, v_tile0);
      f32x16 s_a[NB], s_b[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        if (!wave_has_rows) break;
        s_a[nb] = acc_init(cn_s0, 32 * nb, g);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) s_a[nb] = Tr::mfma32(lds_row_operand<D>(k_tile0, 32 * nb + i, 2 * kk + g), qreg[kk], s_a[nb]);
      }
      auto pipelined_tile = [&](int j, const char* k_nx, const char* v_cur, const float* cn_nx, char* k_fill, char* v_fill, f32x16 (&s_cur)[NB],
                                f32x16 (&s_nx)[NB]) {
        const bool more_k = j + 2 < n_int, more_v = j + 1 < n_int;
        const int nk = more_k ? int_n0(j + 2) : 0, nv = more_v ? int_n0(j + 1) : 0;
        if (more_k) issue_cn(nk);
        const uint16_t *k_src = kp + (int64_t)nk * a.k.st, *v_src = vp + (int64_t)nv * a.v.st;
        const int k_bytes = kld.extent(a.k.st, nk, more_k ? N : nk), v_bytes = vld.extent(a.v.st, nv, more_v ? N : nv);
        const TileDma<D, 0> dma{kld, vld, k_src, v_src, k_bytes, v_bytes, k_fill, v_fill};
        if (wave_has_rows) fwd_tile_pipelined<Tr, D, true>(k_nx, v_cur, cn_nx, qreg, oacc, m_i, l_i, qk_scale, lane, s_cur, s_nx, dma, row.hi);
        else dma.all();
      };
      for (int j = 0; j < n_int; j += 2) {
        wait_vmem_all();
        if (j + 1 < n_int && tid < BN) cn_s1[tid] = cn_term();
        __syncthreads();
        pipelined_tile(j, k_tile1, v_tile0, cn_s1, k_tile0, v_tile1, s_a, s_b);
        if (j + 1 >= n_int) break;
        wait_vmem_all();
        if (j + 2 < n_int && tid < BN) cn_s0[tid] = cn_term();
        __syncthreads();
        pipelined_tile(j + 1, k_tile0, v_tile1, cn_s0, k_tile1, v_tile0, s_b, s_a);
      }
    }
  }
  float l_tot = half_sum(l_i);
  if (it.parts > 1) {
    constexpr int ACC = kAccFloats<D>;
    const int row = wave * 32 + i;
    float* parts = a.q_parts + ((int64_t)it.slot * a.H + h) * kQueryPartFloats<D>;   // the tile's, H apart
    const int64_t step = (int64_t)a.H * kQueryPartFloats<D>;
    if (wave_has_rows) {
      float* own = parts + it.part * step;
      store_part<DB>(own, oacc, wave, lane);
      store_agent(own + ACC + g * BM + row, g ? l_tot : m_i);
    }
    if (!last_part(a.q_arrived + (int64_t)it.slot * a.H + h, it.parts)) return;
    if (wave_has_rows) {
      for (int p = 0; p < it.parts; ++p) m_i = fmaxf(m_i, load_agent(parts + p * step + ACC + row));
      clear(oacc);
      l_tot = 0.f;
      for (int p = 0; p < it.parts; ++p) {
        const float* part = parts + p * step;
        const float weight = __builtin_amdgcn_exp2f(load_agent(part + ACC + row) - m_i);
        l_tot = fmaf(load_agent(part + ACC + BM + row), weight, l_tot);
        add_part<DB>(part, oacc, weight, wave, lane);
      }
    }
  }
  const bool empty = a_m < 0 || n_tiles <= 0;
  const float inv = empty ? 0.f : 1.0f / l_tot;
  if (a.lse && m < M && g == 0) a.lse[(int64_t)h * a.T + it.q0 + m] = empty ? -INFINITY : m_i * kLn2 + __logf(l_tot);
  // o leaves through LDS, a tile buffer per wave, so that the global stores are whole rows
  static_assert(kStoreStageBytes<D> <= Tile<D>::bytes(BN), "one wave stages in one tile buffer");
  wait_vmem_all();
  __syncthreads();
  char* stage = wave == 0 ? k_tile0 : wave == 1 ? k_tile1 : wave == 2 ? v_tile0 : v_tile1;
  store_rows_via_lds<Tr, D>(stage, oacc, inv, op, a.o.st, m0 + 32 * wave, M, lane);
#endif
}

// ---------------------------------------------------------------------------
// dQ: the same walk with Q and dO in registers.  It leaves delta in full for the dK/dV kernel, which runs behind it.
// Bound by the matrix units: 8 sequences of about 3000 tokens, 16 heads, D 128 910 to 1090 TFLOP/s.  dS goes into its product in 16 bits, as P does in the forward: 2.4e-3 of dq next to the
// 1.7e-3 of its own rounding, 2.5e-3 with what delta is off on longer walks.
// ---------------------------------------------------------------------------
template <typename Tr, int D>
__global__ __launch_bounds__(256, D <= 64 ? 3 : 2) void packed_dq_kernel(const PackedK a) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int BM = kFwdBM, BN = kFwdBN, KK = D / 16, DB = (D + 31) / 32;
  __shared__ __align__(16) char k_tile0[Tile<D>::bytes(BN)];
  __shared__ __align__(16) char k_tile1[Tile<D>::bytes(BN)];
  __shared__ __align__(16) char v_tile0[Tile<D>::bytes(BN)];
  __shared__ __align__(16) char v_tile1[Tile<D>::bytes(BN)];
  __shared__ __align__(16) float cn_s0[BN];
  __shared__ __align__(16) float cn_s1[BN];
  __shared__ __align__(16) float lo_s0[BN];
  __shared__ __align__(16) float lo_s1[BN];
  int item, h;
  packed_block(a, a.H, item, h);
  const PackedItem it = a.plan.q_items[item];   // (next to their count: there is memory for as many as the launch has)
  if (item >= a.plan.counts[0]) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5, i = lane & 31;
  const int M = it.m, N = it.n, p_seq = N - M, m0 = it.tile * BM;
  const int hk = h / a.group;
  const double* c_row = a.c + (int64_t)h * a.N + it.k0;
  const int64_t row0 = (int64_t)h * a.T + it.q0;
  const uint16_t* qp = a.q.ptr + (int64_t)it.q0 * a.q.st + h * a.q.sh;
  const uint16_t* dop = a.d_o.ptr + (int64_t)it.q0 * a.d_o.st + h * a.d_o.sh;
  const uint16_t* op = a.o.ptr + (int64_t)it.q0 * a.o.st + h * a.o.sh;
  const uint16_t* kp = a.k.ptr + (int64_t)it.k0 * a.k.st + hk * a.k.sh;
  const uint16_t* vp = a.v.ptr + (int64_t)it.k0 * a.v.st + hk * a.v.sh;
  uint16_t* dqp = const_cast<uint16_t*>(a.dq.ptr) + (int64_t)it.q0 * a.dq.st + h * a.dq.sh;
  const int a0 = p_seq + m0;
  const int m = m0 + 32 * wave + i, a_m = p_seq + m, a_w0 = a0 + 32 * wave;
  const float qk_scale = nonzero_scale(a.sm_scale * kLog2e), inv_scale = 1.0f / qk_scale;
  const bool wave_has_rows = m0 + 32 * wave < M;
  const Walk walk = walk_of(it);
  const int n_tiles = walk.end, t_begin = walk.begin;

  f32x16 dqacc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) dqacc[db][r] = 0.f;
  float delta = 0.f;
  float rsum = 0.f;   // (of sums of tiles: thousands of terms of either sign one by one are only good to 1e-6 of them)
  if (n_tiles > 0) {
    const DirectTileLoader<D, BN> kld(a.k.st, wave, lane), vld(a.v.st, wave, lane);
    kld.issue(kp, a.k.st, (n_tiles - 1) * BN, N, k_tile0);
    vld.issue(vp, a.v.st, (n_tiles - 1) * BN, N, v_tile0);
    u32x4 qreg[KK], doreg[KK], oreg[KK];
    load_row_operand_regs<D>(qreg, qp, a.q.st, m, M, g);
    load_row_operand_regs<D>(doreg, dop, a.d_o.st, m, M, g);
    load_row_operand_regs<D>(oreg, op, a.o.st, m, M, g);
    const double c_ref = c_row[min(max(a0, 0), N - 1)], c_m = c_row[min(max(a_m, 0), N - 1)];
    const float l = a.lse[row0 + min(m, M - 1)];
    double cn_raw = 0.0;
    bool cn_ok = false;
    auto issue_cn = [&](int n0) {
      if (tid < BN) {
        cn_ok = n0 + tid < N;
        cn_raw = c_row[min(n0 + tid, N - 1)];
      }
    };
    auto store_pair = [&](float* hi, float* lo) {
      const Pair c = pair_of((cn_raw - c_ref) * kLog2eD);
      hi[tid] = cn_ok ? c.hi : INFINITY;
      lo[tid] = cn_ok ? c.lo : 0.f;
    };
    auto cn_term = [&]() { return (float)(c_ref - cn_raw) * kLog2e * inv_scale; };   // (off the diagonal every key is one)
    auto issue = [&](int n0, char* kt, char* vt) {
      issue_cn(n0);
      kld.issue(kp, a.k.st, n0, N, kt);
      vld.issue(vp, a.v.st, n0, N, vt);
    };
    issue_cn((n_tiles - 1) * BN);
    // rows past M and rows that see no key (lse = -inf) get -inf
    const bool row_ok = m < M && l != -INFINITY;   // (NaN stays)
    Pair row = pair_of((c_m - c_ref) * kLog2eD);
    const float rowc = row_ok ? row.hi - l * kLog2e : -INFINITY;
    const bool few_keys = min(N, a_w0 + 32) <= 32;
    row = row_ok ? Pair{row.hi, row.lo - l * kLog2e} : Pair{-INFINITY, 0.f};
    {
      float part = 0.f;   // each half of the wave holds half of the row
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int e = 0; e < 4; ++e) part += delta_term<Tr>(oreg[kk][e], doreg[kk][e]);
      delta = half_sum(part);
    }
    // the tiles at the diagonal, an even number of them so that the others find the same buffers free (or all tiles)
    int n_diag = 0;
    while (n_diag < n_tiles - t_begin && (n_tiles - 1 - n_diag) * BN + BN - 1 > a0) ++n_diag;
    n_diag = min(n_diag + (n_diag & 1), n_tiles - t_begin);
    const int t_stop = n_tiles - n_diag;
    if (tid < BN) {
      if (n_diag > 0) store_pair(cn_s0, lo_s0);
      else cn_s0[tid] = cn_term();
    }
    auto next_terms = [&](int t, float* cn, float* lo) {   // of tile t, which has been requested
      if (tid < BN) {
        if (t >= t_stop) store_pair(cn, lo);
        else cn[tid] = cn_term();
      }
    };
    for (int t = n_tiles - 1; t >= t_stop; t -= 2) {
      wait_vmem_all();
      __syncthreads();
      if (t > t_begin) issue((t - 1) * BN, k_tile1, v_tile1);
      if (wave_has_rows) packed_dq_tile<Tr, D>(k_tile0, v_tile0, cn_s0, lo_s0, qreg, doreg, dqacc, rsum, t * BN, a_m, a_w0, row, qk_scale, delta, few_keys, lane);
      if (t <= t_begin) break;
      next_terms(t - 1, cn_s1, lo_s1);
      wait_vmem_all();
      __syncthreads();
      if (t - 1 > t_begin) issue((t - 2) * BN, k_tile0, v_tile0);
      if (wave_has_rows) packed_dq_tile<Tr, D>(k_tile1, v_tile1, cn_s1, lo_s1, qreg, doreg, dqacc, rsum, (t - 1) * BN, a_m, a_w0, row, qk_scale, delta, few_keys, lane);
      if (t - 1 > t_begin) next_terms(t - 2, cn_s0, lo_s0);
    }
    for (int t = t_stop - 1; t >= t_begin; t -= 2) {
      wait_vmem_all();
      __syncthreads();
      if (t > t_begin) issue((t - 1) * BN, k_tile1, v_tile1);
      if (wave_has_rows) packed_dq_interior<Tr, D>(k_tile0, v_tile0, cn_s0, qreg, doreg, dqacc, rsum, qk_scale, rowc, delta, lane);
      if (t <= t_begin) break;
      if (tid < BN) cn_s1[tid] = cn_term();
      wait_vmem_all();
      __syncthreads();
      if (t - 1 > t_begin) issue((t - 2) * BN, k_tile0, v_tile0);
      if (wave_has_rows) packed_dq_interior<Tr, D>(k_tile1, v_tile1, cn_s1, qreg, doreg, dqacc, rsum, qk_scale, rowc, delta, lane);
      if (t - 1 > t_begin && tid < BN) cn_s0[tid] = cn_term();
    }
  }
  float rtot = half_sum(rsum);
  if (it.parts > 1) {
    constexpr int ACC = kAccFloats<D>;
    const int row = wave * 32 + i;
    float* parts = a.q_parts + ((int64_t)it.slot * a.H + h) * kQueryPartFloats<D>;
    const int64_t step = (int64_t)a.H * kQueryPartFloats<D>;
    if (wave_has_rows) {
      float* own = parts + it.part * step;
      store_part<DB>(own, dqacc, wave, lane);
      if (g == 0) store_agent(own + ACC + row, rtot);
    }
    if (!last_part(a.q_arrived + (int64_t)it.slot * a.H + h, it.parts)) return;
    if (wave_has_rows) {
      clear(dqacc);
      rtot = 0.f;
      for (int p = 0; p < it.parts; ++p) {
        const float* part = parts + p * step;
        rtot += load_agent(part + ACC + row);
        add_part<DB>(part, dqacc, 1.f, wave, lane);
      }
    }
  }
  if (m < M && g == 0) a.delta[row0 + m] = delta + rtot;
  __syncthreads();
  char* stage = wave == 0 ? k_tile0 : wave == 1 ? k_tile1 : wave == 2 ? v_tile0 : v_tile1;
  store_rows_via_lds<Tr, D>(stage, dqacc, a.sm_scale, dqp, a.dq.st, m0 + 32 * wave, M, lane);
#endif
}

// ---------------------------------------------------------------------------
// dK/dV: one workgroup keeps 128 keys of a key head (K, V and the accumulators in registers) and walks the query rows that see them in steps of 128, for
// one query head of the group after the other: the sums over the group never leave the registers.
// Bound by the matrix units: 8 sequences of about 3000 tokens, 16 heads on 4, D 128 827 to 1000 TFLOP/s, one workgroup a CU whose waves have no other to hide behind.  (There 56 scalar
// registers are kept in a vector register; none goes to memory.)
// ---------------------------------------------------------------------------
template <typename Tr, int D>
__global__ __launch_bounds__(256, D <= 64 ? 2 : 1) void packed_dkdv_kernel(const PackedK a) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int BN = kKvBN, BMQ = kKvBM, KK = D / 16, DB = (D + 31) / 32;
  __shared__ __align__(16) char q_tile0[Tile<D>::bytes(BMQ)];
  __shared__ __align__(16) char q_tile1[Tile<D>::bytes(BMQ)];
  __shared__ __align__(16) char do_tile0[Tile<D>::bytes(BMQ)];
  __shared__ __align__(16) char do_tile1[Tile<D>::bytes(BMQ)];
  __shared__ Rows rows_s0;
  __shared__ Rows rows_s1;
  int item, hk;
  packed_block(a, a.Hk, item, hk);
  const PackedItem it = a.plan.k_items[item];
  if (item >= a.plan.counts[1]) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5, i = lane & 31;
  const int M = it.m, N = it.n, p_seq = N - M, n0 = it.tile * BN;
  const uint16_t* kp = a.k.ptr + (int64_t)it.k0 * a.k.st + hk * a.k.sh;
  const uint16_t* vp = a.v.ptr + (int64_t)it.k0 * a.v.st + hk * a.v.sh;
  uint16_t* dkp = const_cast<uint16_t*>(a.dk.ptr) + (int64_t)it.k0 * a.dk.st + hk * a.dk.sh;
  uint16_t* dvp = const_cast<uint16_t*>(a.dv.ptr) + (int64_t)it.k0 * a.dv.st + hk * a.dv.sh;
  // rows whose key position reaches this tile; a step may begin above them, and all that lies left of key 0 or above a key is masked
  int m_lo = first_row(M, N, it.tile), n_steps = row_steps(M, N, it.tile), j0 = 0, j1 = a.group;
  KeyParts cut{1, 1, 0, 0};
  if (it.parts > 1) {
    cut = key_parts(n_steps, a.group, it.parts);
    const int hp = it.part / cut.rows, first = (it.part - hp * cut.rows) * cut.row_span;
    j0 = hp * cut.head_span;
    j1 = min(j0 + cut.head_span, a.group);
    m_lo += first * BMQ;
    n_steps = min(n_steps - first, cut.row_span);
  }
  int n_diag = 0;
  while (n_diag < n_steps && p_seq + m_lo + n_diag * BMQ < n0 + BN - 1) ++n_diag;
  const int n_int = n_steps - n_diag, m_top = m_lo + (n_steps - 1) * BMQ;
  const int n_w0 = n0 + 32 * wave, n = n_w0 + i;
  const float qk_scale = nonzero_scale(a.sm_scale * kLog2e), inv_scale = 1.0f / qk_scale;
  const DirectTileLoader<D, BMQ> qld(a.q.st, wave, lane), dold(a.d_o.st, wave, lane);

  f32x16 dkacc[DB], dvacc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) { dkacc[db][r] = 0.f; dvacc[db][r] = 0.f; }
  u32x4 kreg[KK], vreg[KK];
  if (n_steps > 0) {
    load_row_operand_regs<D>(kreg, kp, a.k.st, n, N, g);
    load_row_operand_regs<D>(vreg, vp, a.v.st, n, N, g);
  }

  // A step is a (query head, first row).  Its tiles and its rows' terms are requested while the step before it is computed, across the heads as well; the terms
  // are worked out where they go to LDS, a quarter of the rows a wave, and so is the key's own term of a new head.
  struct Step {
    int j, ms;   // head within the group, first row
  };
  const bool row_lane = lane < BMQ / 4;
  const int row_slot = wave * (BMQ / 4) + lane;
  float l_raw = 0.f, d_raw = 0.f;
  double c_raw = 0.0, c_ref = 0.0, c_key = 0.0;   // of the step requested last
  bool row_ok = false;
  auto head_of = [&](int j) { return hk * a.group + j; };
  auto issue_rows = [&](Step s) {
    const int h = head_of(s.j);
    const double* c_row = a.c + (int64_t)h * a.N + it.k0;
    const int64_t rows = (int64_t)h * a.T + it.q0;
    c_ref = c_row[min(n0 + BN, N) - 1];   // the tile's last key: between its keys and the rows below the diagonal
    c_key = c_row[min(n, N - 1)];
    if (row_lane) {
      const int mm = s.ms + row_slot, mc = min(mm, M - 1);
      row_ok = mm < M;
      l_raw = a.lse[rows + mc];
      c_raw = c_row[min(max(p_seq + mc, 0), N - 1)];
      d_raw = a.delta[rows + mc];
    }
  };
  // the start values of the score accumulators, at the diagonal pairs as well; rows past M and those that see no key get a probability of zero
  auto on_diagonal = [&](Step s) { return p_seq + s.ms < n0 + BN - 1; };
  auto store_rows = [&](Step s, Rows& to) {
    const bool ok = row_ok && l_raw != -INFINITY;   // (NaN stays)
    if (row_lane) {
      to.rc[row_slot] = ok ? ((float)(c_raw - c_ref) - l_raw) * kLog2e * inv_scale : copysignf(INFINITY, -inv_scale);
      to.dl[row_slot] = ok ? -d_raw : 0.f;
    }
    if (on_diagonal(s)) {
      const Pair c = pair_of((c_raw - c_ref) * kLog2eD);
      if (row_lane) {
        to.hi[row_slot] = ok ? c.hi : -INFINITY;
        to.lo[row_slot] = ok ? c.lo - l_raw * kLog2e : 0.f;
      }
    }
  };
  auto q_at = [&](Step s) { return a.q.ptr + head_of(s.j) * a.q.sh + (int64_t)(it.q0 + s.ms) * a.q.st; };
  auto do_at = [&](Step s) { return a.d_o.ptr + head_of(s.j) * a.d_o.sh + (int64_t)(it.q0 + s.ms) * a.d_o.st; };
  constexpr int PER = DirectTileLoader<D, BMQ>::PER;
  auto issue = [&](Step s, char* qt, char* dot) {
    issue_rows(s);   // small loads first: the counter of loads retires in order
    const uint16_t *qs = q_at(s), *ds = do_at(s);
    const int q_bytes = qld.extent(a.q.st, s.ms, M), do_bytes = dold.extent(a.d_o.st, s.ms, M);
#pragma unroll
    for (int e = 0; e < PER; ++e) qld.issue_one(e, qs, q_bytes, qt);
#pragma unroll
    for (int e = 0; e < PER; ++e) dold.issue_one(e, ds, do_bytes, dot);
  };
  Pair col{0.f, 0.f};   // of the lane's key, for the head that is being computed
  auto new_key_term = [&]() {
    col = pair_of((c_key - c_ref) * kLog2eD);
    if (n >= N) col = {INFINITY, 0.f};
  };
  double csum = 0.0;   // (steps in 32 bits, their sum in 64, as in dQ)
  // dc of a head's keys; `more`: its other steps have left their part there
  float dc_part = 0.f;   // where the rows are cut the part has one head
  auto store_dc = [&](int j, bool more) {
    const float ctot = half_sum((float)csum);
    if (cut.rows > 1) {
      dc_part -= ctot;
      csum = 0.0;
      return;
    }
    float* dc = a.dc + (int64_t)head_of(j) * a.N + it.k0 + n;
    if (n < N && g == 0) *dc = (more ? *dc : 0.f) - ctot;
    csum = 0.0;
  };

  if (n_steps == 0) {
    for (int j = 0; j < a.group; ++j) store_dc(j, false);
  } else if constexpr (D <= 64) {
    // every head's steps, those at the diagonal first, in turn from two sets of buffers
    auto next = [&](Step s) {
      const int idx = s.ms < m_lo + n_diag * BMQ ? (s.ms - m_lo) / BMQ : n_diag + (m_top - s.ms) / BMQ, up = idx + 1;
      if (up == n_steps) return Step{s.j + 1, n_diag > 0 ? m_lo : m_top};
      return Step{s.j, up < n_diag ? m_lo + up * BMQ : m_top - (up - n_diag) * BMQ};
    };
    Step cur{j0, n_diag > 0 ? m_lo : m_top};
    issue(cur, q_tile1, do_tile1);
    store_rows(cur, rows_s1);
    new_key_term();
    wait_vmem_all();
    for (int t = 0;; ++t) {
      const bool odd = t & 1;
      const Step nx = next(cur);
      const bool more = nx.j < j1;
      __syncthreads();
      if (more) issue(nx, odd ? q_tile1 : q_tile0, odd ? do_tile1 : do_tile0);
      const char *qt = odd ? q_tile0 : q_tile1, *dot = odd ? do_tile0 : do_tile1;
      const Rows& rows = odd ? rows_s0 : rows_s1;
      float sum = 0.f;
      packed_dkdv_step<Tr, D>(qt, dot, rows, on_diagonal(cur), kreg, vreg, dkacc, dvacc, sum, p_seq + cur.ms, n, n_w0, col, qk_scale, lane);
      csum += (double)sum;
      if (nx.j != cur.j) store_dc(cur.j, false);
      if (!more) break;
      store_rows(nx, odd ? rows_s1 : rows_s0);
      if (nx.j != cur.j) new_key_term();
      wait_vmem_all();
      cur = nx;
    }
  } else {
    // First the steps at the diagonal of all heads, then the others, pipelined: one wave per SIMD, whose registers hold one kind of step at a time.
    const int diag_steps = n_diag * (j1 - j0), int_steps = n_int * (j1 - j0);
    for (int j = j0, d = 0, t = 0; t < diag_steps; ++t) {
      const Step s{j, m_lo + d * BMQ};
      if (t > 0) __syncthreads();   // buffers 1 are free again
      issue(s, q_tile1, do_tile1);
      store_rows(s, rows_s1);
      new_key_term();
      wait_vmem_all();
      __syncthreads();
      if (t == diag_steps - 1 && n_int > 0) issue(Step{j0, m_top}, q_tile0, do_tile0);
      float sum = 0.f;
      packed_dkdv_step<Tr, D>(q_tile1, do_tile1, rows_s1, true, kreg, vreg, dkacc, dvacc, sum, p_seq + s.ms, n, n_w0, col, qk_scale, lane);
      csum += (double)sum;
      if (++d == n_diag) {
        store_dc(j++, false);
        d = 0;
      }
    }
    if (n_int > 0) {
      if (n_diag == 0) issue(Step{j0, m_top}, q_tile0, do_tile0);
      store_rows(Step{j0, m_top}, rows_s0);
      new_key_term();
    }
    Step cur{j0, m_top};
    const int m_int = m_lo + n_diag * BMQ;   // first row of the interior steps
    // a step from one set of buffers, the next one's tiles into the other; an empty extent where there is none (zeros into the free buffers)
    auto interior = [&](const char* qt, const char* dot, const Rows& rows, char* qf, char* dof, Rows& to, bool more) {
      const bool last = cur.ms == m_int;   // of its head
      const Step nx = last ? Step{cur.j + 1, m_top} : Step{cur.j, cur.ms - BMQ};
      if (more) issue_rows(nx);
      const uint16_t *qs = q_at(more ? nx : cur), *ds = do_at(more ? nx : cur);
      const int q_bytes = more ? qld.extent(a.q.st, nx.ms, M) : 0, do_bytes = more ? dold.extent(a.d_o.st, nx.ms, M) : 0;
      float sum = 0.f;
      dkdv_step_interior<Tr, D, 2 * PER>(qt, dot, rows.rc, rows.dl, kreg, vreg, dkacc, dvacc, sum, qk_scale, col.hi, lane, [&](auto k) {
        constexpr int K = decltype(k)::value;
        if constexpr (K < PER) qld.issue_one(K, qs, q_bytes, qf);
        else dold.issue_one(K - PER, ds, do_bytes, dof);
      });
      csum += (double)sum;
      if (last) store_dc(cur.j, n_diag > 0);
      if (more) {
        store_rows(nx, to);
        if (last) new_key_term();
      }
      cur = nx;
    };
    for (int t = 0; t < int_steps; t += 2) {
      wait_vmem_all();
      __syncthreads();
      interior(q_tile0, do_tile0, rows_s0, q_tile1, do_tile1, rows_s1, t + 1 < int_steps);
      if (t + 1 >= int_steps) break;
      wait_vmem_all();
      __syncthreads();
      interior(q_tile1, do_tile1, rows_s1, q_tile0, do_tile0, rows_s0, t + 2 < int_steps);
    }
    wait_vmem_all();   // (the last interior step requested empty tiles)
  }
  if (it.parts > 1) {
    constexpr int ACC = kAccFloats<D>;
    const int key = wave * 32 + i;
    float* parts = a.k_parts + ((int64_t)it.slot * a.Hk + hk) * kKeyPartFloats<D>;
    const int64_t step = (int64_t)a.Hk * kKeyPartFloats<D>;
    if (n_w0 < N) {
      float* own = parts + it.part * step;
      store_part<DB>(own, dkacc, wave, lane);
      store_part<DB>(own + ACC, dvacc, wave, lane);
      if (g == 0) store_agent(own + 2 * ACC + key, dc_part);
    }
    if (!last_part(a.k_arrived + (int64_t)it.slot * a.Hk + hk, it.parts)) return;
    if (n_w0 < N) {
      clear(dkacc);
      clear(dvacc);
      for (int p = 0; p < it.parts; ++p) {
        add_part<DB>(parts + p * step, dkacc, 1.f, wave, lane);
        add_part<DB>(parts + p * step + ACC, dvacc, 1.f, wave, lane);
      }
      for (int hp = 0; cut.rows > 1 && hp < cut.heads; ++hp) {
        float sum = 0.f;
        for (int r = 0; r < cut.rows; ++r) sum += load_agent(parts + (hp * cut.rows + r) * step + 2 * ACC + key);
        if (n < N && g == 0) a.dc[(int64_t)head_of(hp) * a.N + it.k0 + n] = sum;
      }
    }
  }
  static_assert(2 * kStoreStageBytes<D> <= Tile<D>::bytes(BMQ), "two waves stage in one tile buffer");
  __syncthreads();
  char* stage = (wave < 2 ? q_tile0 : do_tile0) + (wave & 1) * kStoreStageBytes<D>;
  store_rows_via_lds<Tr, D>(stage, dkacc, a.sm_scale, dkp, a.dk.st, n_w0, N, lane);
  store_rows_via_lds<Tr, D>(stage, dvacc, 1.0f, dvp, a.dv.st, n_w0, N, lane);
#endif
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
namespace {

// Tiles of `rows` rows in B sequences and the two ends outside them, at most: each of the sequences that are not empty may have a partial one.
int tile_bound(int B, int rows) {
  const int64_t partial = (int64_t)B + 2 < rows ? (int64_t)B + 2 : rows;
  return (int)(rows / kPackedTile + partial);
}
int64_t up(int64_t bytes) { return (bytes + 255) / 256 * 256; }
// (Parts of a half or a third of that length, us: documents of 150 to 2048 tokens, forward 42, 44 for 36, prompts of up to 2048 117, 125 for 110.)
// Parts of cut walks, at most: `over` halves as many as workgroups run at once for a head (each walk's last part may be a short one), or as come of walks of `longest` units, and of `units` in all, in
// shares of at least `least`; none where the longest walk there can be stays whole.  Each costs a workgroup that may find nothing to do.
int extra_parts(int at_once, int heads, int over, int64_t tiles, int64_t longest, double units, int least) {
  const int64_t target = at_once / heads;
  if (target < 2 || longest <= least) return 0;
  return (int)std::min({(double)(over * target / 2), std::floor((double)tiles * std::sqrt((double)longest)), std::floor(over * units / (2.0 * least)) + 1.0});
}

}  // namespace

// Groups of a launch over `tokens` of which an XCD reads `bytes` each: the walks of a group share its L2 as far as 8 MiB of them do (fox_kernels.hpp, order_groups).
static int order_groups_of(int64_t tokens, int64_t bytes) {
  return (int)std::min<int64_t>(kOrderGroups, std::max<int64_t>(1, tokens * bytes >> 23));
}
PackedShape packed_shape(int B, int T, int N, int H, int Hk, int D) {
  PackedShape s;
  s.q_bound = tile_bound(B, T);
  s.k_bound = tile_bound(B, N);
  const int64_t q_tiles = ((int64_t)T + kPackedTile - 1) / kPackedTile, k_tiles = ((int64_t)N + kPackedTile - 1) / kPackedTile, k_steps = ((int64_t)N + kFwdBN - 1) / kFwdBN;
  // (a sequence has at most all whole tiles, and the others' keys add up to all)
  s.q_extra = extra_parts((D <= 64 ? 3 : 2) * kCus, H, kQueryOver, s.q_bound, k_steps, (double)(q_tiles + 1) * (double)(k_steps + B), kQueryShare);
  s.k_extra = extra_parts((D <= 64 ? 2 : 1) * kCus, Hk, kKeyOver, s.k_bound, q_tiles * (H / Hk), (double)(k_tiles + 1) * (double)(q_tiles + B) * (H / Hk), kKeyShare);
  s.q_groups = order_groups_of(N, ((int64_t)Hk + kXcds - 1) / kXcds * D * 4);
  s.k_groups = order_groups_of(T, ((int64_t)H + kXcds - 1) / kXcds * D * 4);
  s.seqs_at = 256;
  const int64_t seqs = (int64_t)B + kPackedOuter;   // once for the queries, once for the keys
  s.items_at = s.seqs_at + up(2 * seqs * sizeof(int4));
  s.plan_bytes = s.items_at + ((int64_t)s.q_bound + s.q_extra + s.k_bound + s.k_extra) * (int64_t)sizeof(PackedItem);
  const int64_t acc = (int64_t)(D + 31) / 32 * 32 * kPackedTile, q_rows = (int64_t)s.q_extra * H, k_rows = (int64_t)s.k_extra * Hk;
  s.q_arrived_at = up(q_rows * (acc + 2 * kPackedTile) * 4);
  s.fwd_bytes = s.k_parts_at = s.q_arrived_at + up(q_rows * 4);
  s.k_arrived_at = s.k_parts_at + up(k_rows * (2 * acc + kPackedTile) * 4);
  s.bwd_bytes = s.k_arrived_at + up(k_rows * 4);
  return s;
}
void packed_memory(PackedK& a, const PackedShape& s, void* plan, void* workspace) {
  char *at = (char*)plan, *ws = (char*)workspace;
  a.q_bound = s.q_bound;
  a.k_bound = s.k_bound;
  a.q_extra = s.q_extra;
  a.q_groups = s.q_groups;
  a.k_groups = s.k_groups;
  a.k_extra = s.k_extra;
  a.plan.counts = (int32_t*)at;
  a.plan.seqs = (int4*)(at + s.seqs_at);
  a.plan.q_items = (PackedItem*)(at + s.items_at);
  a.plan.k_items = a.plan.q_items + s.q_bound + s.q_extra;
  a.q_parts = (float*)ws;
  a.q_arrived = (uint32_t*)(ws + s.q_arrived_at);
  a.k_parts = (float*)(ws + s.k_parts_at);
  a.k_arrived = (uint32_t*)(ws + s.k_arrived_at);
}

// Whether a row of the scans is a wave's rather than a workgroup's of 1024.  A wave is done after some 5 + 0.008 us for each of the longest row's elements, workgroups
// after 6 + 0.01 for each row.  (A wave / a workgroup, 16 heads, us: 64 rows of 100 elements 8.6 / 16.2, 64 of 800 11.2 / 18.6, 256 of 500 12.2 / 57.7, 32 of 500 9.1 / 10.6, 24 of 800
// 10.2 / 9.2, 32 of 1500 16.2 / 12.9, 20 of 4000 36.2 / 14.4.)  The host knows the rows and all their elements, not the longest of them, so the rule takes rows to be alike.  Where they are not, one
// long row makes its wave the last by far: 63 of 100 and one of 16384 136 / 28 and, in the gradient, 152 / 24; 31 of 401 and one of 8512 73 / 18 and 80 / 15; 255 of 301 and one of 4064, 8 heads, 22 / 33.
static bool short_rows(int64_t elements, int64_t rows, int heads) { return 2 * elements <= 3 * rows * rows * heads; }

template <typename Tr, int D>
static hipError_t packed_fwd_d(const PackedK& args, hipStream_t s) {
  PackedK a = args;
  a.by_heads = divisor(a.H);
  a.by_xcd_heads = divisor(a.H % kXcds ? 1 : a.H / kXcds);
  const int rows = a.B * a.H, plans = a.lse ? 2 : 1;
  if (short_rows(a.N, a.B, a.H)) hipLaunchKernelGGL(packed_scan_kernel<64>, dim3((unsigned)(plans + (rows + 15) / 16)), dim3(1024), 0, s, a);
  else hipLaunchKernelGGL(packed_scan_kernel<1024>, dim3((unsigned)(plans + rows)), dim3(1024), 0, s, a);
  hipLaunchKernelGGL((packed_fwd_kernel<Tr, D>), dim3((unsigned)(((int64_t)a.q_bound + a.q_extra) * a.H)), dim3(256), 0, s, a);
  return hipGetLastError();
}
template <typename Tr, int D>
static hipError_t packed_bwd_d(const PackedK& args, hipStream_t s) {
  PackedK a = args;
  a.by_heads = divisor(a.H);
  a.by_xcd_heads = divisor(a.H % kXcds ? 1 : a.H / kXcds);
  const int counters = std::max(a.q_extra * a.H, a.k_extra * a.Hk);
  if (counters > 0) hipLaunchKernelGGL(packed_clear_kernel, dim3((unsigned)((counters + 255) / 256)), dim3(256), 0, s, a);
  hipLaunchKernelGGL((packed_dq_kernel<Tr, D>), dim3((unsigned)(((int64_t)a.q_bound + a.q_extra) * a.H)), dim3(256), 0, s, a);
  PackedK k = a;
  k.by_heads = divisor(a.Hk);
  k.by_xcd_heads = divisor(a.Hk % kXcds ? 1 : a.Hk / kXcds);
  hipLaunchKernelGGL((packed_dkdv_kernel<Tr, D>), dim3((unsigned)(((int64_t)a.k_bound + a.k_extra) * a.Hk)), dim3(256), 0, s, k);
  const int rows = (a.B + kPackedOuter) * a.H;
  if (short_rows(a.N, a.B, a.H)) hipLaunchKernelGGL(packed_gate_grad_kernel<64>, dim3((unsigned)((rows + 15) / 16)), dim3(1024), 0, s, a);
  else hipLaunchKernelGGL(packed_gate_grad_kernel<1024>, dim3((unsigned)rows), dim3(1024), 0, s, a);
  return hipGetLastError();
}

template <typename Tr>
static hipError_t packed_t(const PackedK& a, int D, bool bwd, hipStream_t s) {
  switch (D) {
    case 16: return bwd ? packed_bwd_d<Tr, 16>(a, s) : packed_fwd_d<Tr, 16>(a, s);
    case 32: return bwd ? packed_bwd_d<Tr, 32>(a, s) : packed_fwd_d<Tr, 32>(a, s);
    case 64: return bwd ? packed_bwd_d<Tr, 64>(a, s) : packed_fwd_d<Tr, 64>(a, s);
    case 128: return bwd ? packed_bwd_d<Tr, 128>(a, s) : packed_fwd_d<Tr, 128>(a, s);
    default: return hipErrorInvalidValue;
  }
}
hipError_t launch_packed_fwd(const PackedK& a, int D, int dtype, hipStream_t s) {
  return dtype == 0 ? packed_t<Bf16>(a, D, false, s) : packed_t<Fp16>(a, D, false, s);
}
hipError_t launch_packed_bwd(const PackedK& a, int D, int dtype, hipStream_t s) {
  return dtype == 0 ? packed_t<Bf16>(a, D, true, s) : packed_t<Fp16>(a, D, true, s);
}

}  // namespace fox
