// How the attention of new tokens over their requests' pages is cut: the plan that every workgroup works out from the lengths or finds in the workspace
// (fox_paged.hip, fox_paged8.hip).
#pragma once
#include "fox_common.hpp"
#include "fox_kernels.hpp"

namespace fox {

namespace {

// Sums of x and y over the threads 0 .. own of a workgroup of 1024, exact for integers below 2^53.  Every thread calls it.
struct Sums {
  double x, y, all_x, all_y;   // up to this thread, of all
};
__device__ __forceinline__ Sums block_scan(double x, double y, double (&waves)[2][16]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  x = wave_scan(x);
  y = wave_scan(y);
  __syncthreads();   // (the sums of an earlier call have been read)
  if (lane == 63) {
    waves[0][wave] = x;
    waves[1][wave] = y;
  }
  __syncthreads();
  const double wx = wave_scan(lane < 16 ? waves[0][lane] : 0.0), wy = wave_scan(lane < 16 ? waves[1][lane] : 0.0);
  if (wave > 0) {
    x += of_lane(wx, wave - 1);
    y += of_lane(wy, wave - 1);
  }
  return Sums{x, y, of_lane(wx, 15), of_lane(wy, 15)};
}

// Keys a row may see, 0 where its request is none of the table's.
__device__ __forceinline__ int keys_of(const PagedDecodeK& a, int b) {
  if (a.requests && (uint32_t)a.requests[b] >= (uint32_t)a.R) return 0;
  return min(max(a.lengths[b], 0), a.max_keys);
}

__host__ __device__ constexpr int paged_batch(int D) { return 4 * 4096 / D; }   // keys of a batch: of the four waves of a workgroup

struct PagedShare {    // of a row: its keys and how they are cut
  int keys, batches;   // batches a piece
  int pieces;          // at least one
};
template <int D>
__device__ __forceinline__ PagedShare share_of(const PagedDecodeK& a, int b, int per_piece) {
  PagedShare s;
  s.keys = b < a.B ? keys_of(a, b) : 0;
  const int nb = (s.keys + paged_batch(D) - 1) / paged_batch(D);
  s.batches = max(max(per_piece, (nb + kDecodeMaxSplits - 1) / kDecodeMaxSplits), 1);
  s.pieces = max((nb + s.batches - 1) / s.batches, 1);
  return s;
}

// Batches a piece.  All rows and heads together fill at most kPagedPieces pieces; short rows stay whole where splitting
// them brings no more than a merge and starts of workgroups.  Both ways in us, from the batches that each of the 1024
// workgroups that run at once gets (`load`): batch_us, 10, for the bytes of one batch each at 6.5 TB/s (half in 8 bits) or 1.8 for each of a run's round
// trips, 3 for every 1024 workgroups that start, 1.5 for the merge, 3 a batch for the longest rows' tail.  Pages of 16, us,
// split / as it is: D 64, 1024 requests and heads of 300 keys 25.4 / 19.0, 512 of 700 23.6 / 20.4, D 128, 1024 of 300 39.7 / 32.4.
template <int D>
__device__ __forceinline__ int choose_batches(const PagedDecodeK& a, double total, int most) {
  const int c = max((int)fmin(ceil(total * a.H * a.per_piece), a.max_keys / paged_batch(D) + 1), 1);   // (no row has more batches)
  if (most <= c || most > 8) return c;
  const float load = (float)total * a.H / 1024.f, rows = (float)a.B * a.H / 1024.f, full = (float)total / ((float)a.B * most);
  const float split = fmaxf(a.batch_us * load, 1.8f * c) + 3.f * fmaxf(load / c, 1.f) + 1.5f;
  const float whole = fmaxf(a.batch_us * load, 1.8f * most) + 3.f * fmaxf(rows, 1.f) + 3.f * (most - 1) * (1.f - full);
  return whole < split ? most : c;
}
template <int D>
__device__ __forceinline__ int batches_of(const PagedDecodeK& a, int b) {
  return (keys_of(a, b) + paged_batch(D) - 1) / paged_batch(D);
}
// The same from the lengths themselves.  Executed by whole waves.
template <int D>
__device__ __forceinline__ int batches_per_piece(const PagedDecodeK& a, int lane) {
  double sum = 0;
  int most = 0;
  for (int b = lane; b < a.B; b += 64) {
    const int nb = batches_of<D>(a, b);
    sum += nb;
    most = max(most, nb);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) most = max(most, __shfl_xor(most, off));
  return __builtin_amdgcn_readfirstlane(choose_batches<D>(a, of_lane(wave_scan(sum), 63), most));
}

struct PagedPiece {
  int b, piece, first;   // row, its piece, and the row's first piece among all (of one head)
  PagedShare share;
};
// The row that piece number p (of one head) belongs to; b < 0: there is none.  The result is the same in all lanes, and in
// all workgroups, which run this same code.
template <int D>
__device__ __forceinline__ PagedPiece find_piece(const PagedDecodeK& a, int p, int lane) {
  PagedPiece r;
  r.b = -1;
  if (!a.ws_row) {   // no row can be more than one piece
    if (p >= a.B) return r;
    r.b = r.first = p;
    r.piece = 0;
    r.share = PagedShare{keys_of(a, p), 1, 1};
    return r;
  }
  if (a.planned) {   // the rows' first pieces are there, sorted: 64 of them compared at a time
    const PagedRow all = a.ws_row[a.B];
    if (p >= all.first) return r;
    int lo = 0, n = a.B;
    while (n > 1) {
      const int step = (n + 63) / 64, at = lane * step;
      const uint64_t before = __ballot(at < n && a.ws_row[lo + min(at, n - 1)].first <= p);   // (the first always is)
      const int k = (__popcll(before) - 1) * step;
      lo += k;
      n = min(step, n - k);
    }
    const PagedRow row = a.ws_row[lo];
    r.b = lo;
    r.first = row.first;
    r.piece = p - row.first;
    r.share = share_of<D>(a, lo, all.pieces);
    return r;
  }
  const int per_piece = batches_per_piece<D>(a, lane);
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const PagedShare s = share_of<D>(a, b0 + lane, per_piece);
    const int pieces = b0 + lane < a.B ? s.pieces : 0, end = before + (int)wave_scan(pieces), first = end - pieces;
    const uint64_t hit = __ballot(first <= p && p < end);
    if (hit) {
      const int from = __ffsll((unsigned long long)hit) - 1;
      r.b = b0 + from;
      r.first = __builtin_amdgcn_readlane(first, from);
      r.piece = p - r.first;
      r.share.keys = __builtin_amdgcn_readlane(s.keys, from);
      r.share.batches = __builtin_amdgcn_readlane(s.batches, from);
      r.share.pieces = __builtin_amdgcn_readlane(s.pieces, from);
      return r;
    }
    before = __builtin_amdgcn_readlane(end, 63);
  }
  return r;
}

}  // namespace

// Full pieces of all rows and heads together, at most: eight workgroups a CU.  4, 6, 12 and 16 instead of 8: geomean of 36
// shapes 1.014, 1.010, 1.004, 1.011 of the time.
constexpr int kPagedPieces = 8 * kCus;

inline int64_t most_pieces(int max_keys, int D) {   // of a row
  const int64_t batches = ((int64_t)max_keys + paged_batch(D) - 1) / paged_batch(D);
  return batches < 1 ? 1 : batches < kDecodeMaxSplits ? batches : kDecodeMaxSplits;
}
// Workgroups: no row makes more pieces than its share of `pieces` and one for what is left over.
inline int64_t paged_decode_workgroups(int B, int H, int max_keys, int D) {
  const int64_t by_row = (int64_t)B * H * most_pieces(max_keys, D), shared = kPagedPieces + (int64_t)B * H;
  return by_row < shared ? by_row : shared;
}
// Whether a launch in front makes the plan.  Up to 255 rows every wave works it out from the lengths, 64 at a time, which a launch of its own would not make
// up for (300 keys, H8 D64, us, waves / launch: 256 rows 41.0 / 40.4, 384 64.5 / 55.6, 1024 216 / 142; 64 rows take 12.2).
inline bool plan_ahead(const PagedDecodeK& a) { return a.ws_row && a.B >= 256; }

}  // namespace fox
