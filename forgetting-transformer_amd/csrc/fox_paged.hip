// Serving from pages for gfx950: slots of new tokens in a pool of pages, the append into them, and Forgetting Attention of one new
// token per request over its pages.
//
// The pool holds P pages of S = 2^shift tokens: keys and values (P, H, S, D), log forget gates (P, H, S).  Row b of the block table names
// the pages of request b in order, lengths[b] tokens are cached.  Token i of a request lives in slot page * S + i % S, page = table[b][i / S].
// The free pages are a stack, so who gets which page depends on the order of the requests alone.
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

struct Request {   // of a page_slots, in LDS
  int32_t end;     // new tokens up to and including this request's
  int32_t begin;
  int32_t length;  // cached tokens
  int32_t held;    // pages of those; negative (-1 - held): refused
  int32_t place;   // of its first new page in the stack; the others lie below
};

}  // namespace

// Every workgroup scans the requests (8 bytes each, from the L2) and serves 1024 tokens; the first one writes the requests'
// new state.  Bound by latency: the state's round trip, a scan, a binary search in LDS and the round trip of the page; 3.8 us for 256
// requests' next tokens, 5.2 for 16384 tokens of 64 requests, where a copy of as much takes 2.2.
__global__ __launch_bounds__(1024) void page_slots_kernel(const PageSlotsK a) {
  __shared__ Request req[kPageRequests];
  __shared__ double waves[2][16];
  __shared__ int used_s;
  const int tid = threadIdx.x, S = 1 << a.shift;
  const bool state = a.state && blockIdx.x == 0;
  const int count = min(max(*a.free_count, 0), a.P);
  const int64_t room = (int64_t)a.W << a.shift;
  double tokens = 0, pages = 0;   // of the requests before this chunk
  int used = 0;                   // pages handed out, up to this thread's last
  if (tid == 0) used_s = 0;
  for (int b0 = 0; b0 < a.B; b0 += 1024) {
    const int b = b0 + tid;
    int len = 0, fresh = 0;
    if (b < a.B) {
      len = (int)min((int64_t)max(a.lengths[b], 0), room);
      fresh = max(a.new_tokens[b], 0);
    }
    const int held = (int)(((int64_t)len + S - 1) >> a.shift);
    const int64_t wanted = ((int64_t)len + fresh + S - 1) >> a.shift, need = wanted - held;
    // A request that fits no row of the table takes no pages.  One whose tokens end behind the last place takes none either,
    // but all behind it end there as well, so that nobody who is served counts on it.
    const Sums sum = block_scan(fresh, wanted <= a.W ? (double)need : 0.0, waves);
    const double end = tokens + sum.x, taken = pages + sum.y;
    tokens += sum.all_x;
    pages += sum.all_y;
    // pages in request order while they last: beyond the first that cannot be served the sums only grow
    const bool ok = wanted <= a.W && end <= a.T && (need == 0 || taken <= count);
    if (ok && need > 0) used = (int)taken;
    if (b < a.B) {
      const int32_t e = (int32_t)min(end, 2147483647.0);
      req[b] = Request{e, (int32_t)min(end - fresh, 2147483647.0), len, ok ? held : -1 - held, ok ? (int32_t)(count - 1 - (taken - need)) : 0};
      if (state) {
        a.lengths_out[b] = ok ? len + fresh : len;
        a.granted[b] = ok;
      }
    }
  }
  if (state && used > 0) atomicMax(&used_s, used);   // (the barriers of the scan lie behind the zero)
  __syncthreads();
  if (state && tid == 0) *a.free_out = count - used_s;   // what is left below the last page handed out
  if (!a.tokens) return;
  for (int64_t t = (int64_t)blockIdx.x * 1024 + tid; t < a.T; t += (int64_t)gridDim.x * 1024) {
    int lo = 0, hi = a.B;   // the first request whose tokens end behind t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (req[mid].end > t) hi = mid;
      else lo = mid + 1;
    }
    int64_t slot = -1, pos = 0;
    int who = -1;
    if (lo < a.B) {
      const Request r = req[lo];
      pos = r.length + (t - r.begin);
      if (r.held >= 0) {
        const int idx = (int)(pos >> a.shift);
        int32_t* entry = a.table + lo * a.table_sb + idx;
        const int page = idx < r.held ? *entry : a.free_pages[r.place - (idx - r.held)];
        if (idx >= r.held && (pos & (S - 1)) == 0) *entry = page;   // one token is the first of a new page
        who = lo;
        if (page >= 0) slot = ((int64_t)page << a.shift) + (pos & (S - 1));
      }
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
    a.requests[t] = who;
    a.keys[t] = who < 0 ? 0 : (int)pos + 1;
  }
}

hipError_t launch_page_slots(const PageSlotsK& a, hipStream_t s) {
  const unsigned wgs = a.T > 1024 ? (unsigned)((a.T + 1023) / 1024) : 1u;
  const bool in_place = a.lengths_out == a.lengths || a.free_out == a.free_count;
  if (wgs == 1 || !in_place) {
    PageSlotsK k = a;
    k.tokens = k.state = true;
    hipLaunchKernelGGL(page_slots_kernel, dim3(wgs), dim3(1024), 0, s, k);
    return hipGetLastError();
  }
  // several workgroups read the state that one would overwrite: it is written by a launch of its own
  PageSlotsK k = a;
  k.tokens = true;
  k.state = false;
  hipLaunchKernelGGL(page_slots_kernel, dim3(wgs), dim3(1024), 0, s, k);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  k.tokens = false;
  k.state = true;
  hipLaunchKernelGGL(page_slots_kernel, dim3(1), dim3(1024), 0, s, k);
  return hipGetLastError();
}

// The pages of finished requests back on the stack, request by request, a wave each (a quarter of 512 requests with 62 pages
// each 6.6 us; a page a thread, which looks its request up as page_slots_kernel's tokens do, 7.9).
__global__ __launch_bounds__(1024) void page_release_kernel(const PageReleaseK a) {
  __shared__ int32_t place[kPageRequests], held_s[kPageRequests];
  __shared__ double waves[2][16];
  const int tid = threadIdx.x, lane = tid & 63, S = 1 << a.shift;
  const int count = min(max(*a.free_count, 0), a.P);
  double pages = count;
  for (int b0 = 0; b0 < a.B; b0 += 1024) {
    const int b = b0 + tid;
    int len = 0;
    bool done = false;
    if (b < a.B) {
      len = (int)min((int64_t)max(a.lengths[b], 0), (int64_t)a.W << a.shift);
      done = a.done[b] != 0;
    }
    const int held = done ? (int)(((int64_t)len + S - 1) >> a.shift) : 0;
    const Sums sum = block_scan(held, 0, waves);
    if (b < a.B) {
      place[b] = (int32_t)min(pages + sum.x - held, (double)a.P);
      held_s[b] = held;
      a.lengths_out[b] = done ? 0 : len;
    }
    pages += sum.all_x;
  }
  __syncthreads();
  if (tid == 0) *a.free_out = (int)min(pages, (double)a.P);
  for (int b = tid >> 6; b < a.B; b += 16) {
    const int n = min(held_s[b], a.P - place[b]);   // (a stack that is full takes no more)
    for (int i = lane; i < n; i += 64) a.free_pages[place[b] + i] = a.table[b * a.table_sb + i];
  }
}

hipError_t launch_page_release(const PageReleaseK& a, hipStream_t s) {
  hipLaunchKernelGGL(page_release_kernel, dim3(1), dim3(1024), 0, s, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// New tokens' keys, values and log gates into their slots: one 16-byte piece of k and the same piece of v per thread, the thread with a row's
// first piece also moves its gate.  A plain stream, read through the caches (the projections have just written it) and
// written past them (the attention reads all of the cache before it comes back to these rows; both past them / as it is,
// H16 D128, 2048 tokens 8.2 / 7.2 us).  16384 tokens take 49 us (5.5 TB/s), 48 of H12 D64 3.2.  Slots outside the pool are left out.
template <int D>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendK a) {
  constexpr int CH = D / 8;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= a.total) return;
  const int ch = (int)(idx % CH), row = (int)(idx / CH), t = divide(row, a.by_heads), h = row - t * a.H;
  const int64_t slot = a.slots[t];
  const u32x4 kx = *reinterpret_cast<const u32x4*>(a.k + t * a.k_st + h * a.k_sh + ch * 8);
  const u32x4 vx = *reinterpret_cast<const u32x4*>(a.v + t * a.v_st + h * a.v_sh + ch * 8);
  float gx = 0.f;
  if (ch == 0) gx = a.g[t * a.g_st + h * a.g_sh];
  if (slot < 0 || slot >= (int64_t)a.pages.P << a.pages.shift) return;
  const int64_t page = slot >> a.pages.shift, at = slot & ((1 << a.pages.shift) - 1);
  const View &k = a.pages.k, &v = a.pages.v;
  __builtin_nontemporal_store(kx, reinterpret_cast<u32x4*>(const_cast<uint16_t*>(k.ptr) + page * k.sb + h * k.sh + at * k.st + ch * 8));
  __builtin_nontemporal_store(vx, reinterpret_cast<u32x4*>(const_cast<uint16_t*>(v.ptr) + page * v.sb + h * v.sh + at * v.st + ch * 8));
  if (ch == 0) a.pages.g[page * a.pages.g_sp + h * a.pages.g_sh + at * a.pages.g_ss] = gx;
}

hipError_t launch_paged_append(const PagedAppendK& a, int D, hipStream_t s) {
  const dim3 grid((unsigned)((a.total + 255) / 256));
  switch (D) {
    case 16: hipLaunchKernelGGL(paged_append_kernel<16>, grid, dim3(256), 0, s, a); break;
    case 32: hipLaunchKernelGGL(paged_append_kernel<32>, grid, dim3(256), 0, s, a); break;
    case 64: hipLaunchKernelGGL(paged_append_kernel<64>, grid, dim3(256), 0, s, a); break;
    case 128: hipLaunchKernelGGL(paged_append_kernel<128>, grid, dim3(256), 0, s, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Forgetting Attention of one token per row over the pages of its request:
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(q.k_j sm_scale + sum of the log gates behind j up to the row's last key).
//
// One pass over the pages, 4*D flops per 4*D + 4 bytes: a key row of D elements is spread over D/8 lanes, every lane holds eight 16-byte loads of K
// and of V in flight, each row group runs its own online softmax.  A wave walks its run of keys from the end and carries the sum of the
// gates behind it (fp64, rounded once per key) relative to the end of the run; where runs are merged their totals shift the maxima of those in front,
// so every gate is read once.
//
// How long the requests are only the device knows.  Every wave works out the same plan from the lengths: batches of four
// waves' loads, pieces of c batches, with c chosen so that all rows and heads together fill at most kPagedPieces of them: requests of
// very different lengths still give the workgroups the same share.  Every (row, head) may add a piece that is not full, so there are up to
// kPagedPieces + B * H pieces, which is what the grid and the workspace are sized for; a workgroup past the last one ends.
// For many rows a launch in front makes the plan once.
//
// 16 requests of 24576 to 32768 tokens, H16 D128, 572 us: 6.4 TB/s, where a stream that is only read reaches 7.1; 48
// requests of up to 8192 tokens, H12 D64, 42.1 us and 4.6 of the merge (5.3 TB/s); one request of 1500 tokens, H12 D64, 6.9 us, a
// chain of four round trips (lengths, table, rows, partials), and 3.7 of the merge.
//
// A lane holds the table's entry for one of 64 consecutive pages and takes a row's page from the lane that has it; the
// entries are read again every 64 pages.  Entries outside the pool name no page: their keys are left out and their gates count as 0.
namespace {

template <typename Tr>
__device__ __forceinline__ void unpack8p(const u32x4& v, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = Tr::lo(v[e]);
    f[2 * e + 1] = Tr::hi(v[e]);
  }
}

// merge the online-softmax state (m2, l2, acc2) into (m, l, acc)
__device__ __forceinline__ void merge_runs(float& m, float& l, float (&acc)[8], float m2, float l2, const float (&acc2)[8]) {
  const float mx = fmaxf(m, m2);
  const float w1 = __builtin_amdgcn_exp2f(m - mx), w2 = __builtin_amdgcn_exp2f(m2 - mx);
  l = l * w1 + l2 * w2;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = acc[e] * w1 + acc2[e] * w2;
  m = mx;
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
// workgroups that run at once gets (`load`): 10 for the bytes of one batch each at 6.5 TB/s or 1.8 for each of a run's round
// trips, 3 for every 1024 workgroups that start, 1.5 for the merge, 3 a batch for the longest rows' tail.  Pages of 16, us,
// split / as it is: D 64, 1024 requests and heads of 300 keys 25.4 / 19.0, 512 of 700 23.6 / 20.4, D 128, 1024 of 300 39.7 / 32.4.
template <int D>
__device__ __forceinline__ int choose_batches(const PagedDecodeK& a, double total, int most) {
  const int c = max((int)fmin(ceil(total * a.H * a.per_piece), a.max_keys / paged_batch(D) + 1), 1);   // (no row has more batches)
  if (most <= c || most > 8) return c;
  const float load = (float)total * a.H / 1024.f, rows = (float)a.B * a.H / 1024.f, full = (float)total / ((float)a.B * most);
  const float split = fmaxf(10.f * load, 1.8f * c) + 3.f * fmaxf(load / c, 1.f) + 1.5f;
  const float whole = fmaxf(10.f * load, 1.8f * most) + 3.f * fmaxf(rows, 1.f) + 3.f * (most - 1) * (1.f - full);
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

// The plan of many rows in a launch of its own: every row's pieces, and behind them the number of all pieces and the batches a piece.
template <int D>
__global__ __launch_bounds__(1024) void paged_plan_kernel(const PagedDecodeK a) {
  __shared__ double waves[2][16];
  __shared__ int longest;
  const int tid = threadIdx.x;
  if (tid == 0) longest = 0;
  double total = 0;
  int most = 0;
  for (int b = tid; b < a.B; b += 1024) {
    const int nb = batches_of<D>(a, b);
    total += nb;
    most = max(most, nb);
  }
  total = block_scan(total, 0, waves).all_x;   // (its barriers lie between the zero and the maxima)
  atomicMax(&longest, most);
  __syncthreads();
  const int per_piece = choose_batches<D>(a, total, longest);
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 1024) {
    const int b = b0 + tid, pieces = b < a.B ? share_of<D>(a, b, per_piece).pieces : 0;
    const Sums sum = block_scan(pieces, 0, waves);
    const int end = before + (int)sum.x;
    if (b < a.B) a.ws_row[b] = PagedRow{end - pieces, pieces};
    before += (int)sum.all_x;
  }
  if (tid == 0) a.ws_row[a.B] = PagedRow{before, per_piece};
}

template <typename Tr, int D>
__global__ __launch_bounds__(256) void paged_decode_kernel(const PagedDecodeK a) {
  constexpr int LPR = D / 8;      // lanes per key row
  constexpr int KPL = 64 / LPR;   // keys per wave load instruction
  constexpr int U = 8;            // loads of K and of V in flight per lane
  constexpr int KPB = KPL * U;    // keys per wave and batch
  constexpr int GB = (KPB + 63) / 64;   // gates per lane and batch
  static_assert(4 * KPB == paged_batch(D), "the plan counts batches with the same size");
  __shared__ float part_m[4], part_l[4];
  __shared__ double part_g[4];
  __shared__ __align__(16) float part_acc[4][D];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ch = lane % LPR, r = lane / LPR;
  const int number = divide(blockIdx.x, a.by_heads), h = blockIdx.x - number * a.H;
  const PagedPiece at = find_piece<D>(a, number, lane);
  if (at.b < 0) return;   // (the same in all waves)
  if (a.ws_row && !a.planned && at.piece == 0 && h == 0 && tid == 0) a.ws_row[at.b] = PagedRow{at.first, at.share.pieces};   // for the merge
  const int b = at.b;
  const PagesK& pg = a.pages;
  const int32_t* table = a.table + (a.requests ? a.requests[b] : b) * a.table_sb;
  const uint16_t* kp = pg.k.ptr + h * pg.k.sh + ch * 8;
  const uint16_t* vp = pg.v.ptr + h * pg.v.sh + ch * 8;
  const float* gp = pg.g + h * pg.g_sh;
  const int in_page = (1 << pg.shift) - 1;

  // run of this wave, counted from the last key: whole batches, the first one excepted
  const int per = at.share.batches * KPB;
  const int64_t back = (int64_t)(at.piece * 4 + wave) * per;
  const int k1 = back < at.share.keys ? at.share.keys - (int)back : 0, k0 = max(k1 - per, 0);

  float qf[8];
  {
    const float qk_scale = a.sm_scale * kLog2e;
    unpack8p<Tr>(*reinterpret_cast<const u32x4*>(a.q + b * a.q_sb + h * a.q_sh + ch * 8), qf);
#pragma unroll
    for (int e = 0; e < 8; ++e) qf[e] *= qk_scale;
  }
  float m = -3.0e38f, l = 0.f;  // finite floor: a group that has seen no key yet yields exp2(-inf) = 0
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  double behind = 0.0;          // sum of the run's gates behind the batch
  int page0 = INT32_MAX, entry = -1;   // this lane has the table's entry for page page0 + lane

  for (int end = k1; end > k0; end -= KPB) {   // keys end - KPB .. end - 1, those left of k0 masked
    const int first = max(end - KPB, k0);
    if ((first >> pg.shift) < page0) {
      page0 = max(((end - 1) >> pg.shift) - 63, 0);
      entry = table[min(page0 + lane, a.W - 1)];
      if ((uint32_t)entry >= (uint32_t)pg.P) entry = -1;
    }
    auto page_of = [&](int n) { return __builtin_amdgcn_ds_bpermute(((n >> pg.shift) - page0) << 2, entry); };
    float gx[GB];
#pragma unroll
    for (int s = 0; s < GB; ++s) {             // lane j of group s holds the gate of key end - 1 - 64 s - j
      const int j = 64 * s + lane, n = max(end - 1 - j, first), page = page_of(n);
      gx[s] = gp[max(page, 0) * pg.g_sp + (n & in_page) * pg.g_ss];
      if (j >= KPB || end - 1 - j < first || page < 0) gx[s] = 0.f;
    }
    // The fences keep one row's addresses in registers at a time: 119 to 127 registers, four workgroups a CU (without them 131
    // to 135 and three at head dims 32 and 64, 36 shapes geomean 1.036 of the time; all rows' pages asked for first, since a
    // page takes as long as an LDS read).
    u32x4 kx[U], vx[U];
    uint32_t ok = 0;
    int pages[U];
#pragma unroll
    for (int u = 0; u < U; ++u) pages[u] = page_of(max(end - KPB + u * KPL + r, first));   // keys left of the run read its first row and are masked below
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int n0 = end - KPB + u * KPL + r;
      ok |= (uint32_t)(n0 >= first && pages[u] >= 0) << u;
      const int64_t from = max(pages[u], 0);
      const int row = max(n0, first) & in_page;
      kx[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp + from * pg.k.sb + row * pg.k.st));
      vx[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vp + from * pg.v.sb + row * pg.v.st));
      __builtin_amdgcn_sched_barrier(0);
    }
    if (__ballot(ok != (1u << U) - 1)) {   // what is masked may hold anything, NaN among it
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (!(ok >> u & 1)) vx[u] = u32x4{0u, 0u, 0u, 0u};
    }
    float bias[GB];   // log2e * sum of the gates behind the key whose gate this lane holds
#pragma unroll
    for (int s = 0; s < GB; ++s) {
      const double incl = wave_scan((double)gx[s]), excl = lane_before(incl);   // (not incl - gate: a gate may be -inf)
      bias[s] = (float)(behind + excl) * kLog2e;
      behind += of_lane(incl, 63);
    }
    float sc[U];
    float bmax = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float kf[8];
      unpack8p<Tr>(kx[u], kf);
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) dot = fmaf(qf[e], kf[e], dot);
      dot = row_sum<LPR>(dot);
      const int j = KPB - 1 - u * KPL;   // key u * KPL + r of the batch sits j - r keys before its end
      const float x = dot + __shfl(bias[j / 64], (j - r) & 63);
      sc[u] = ok >> u & 1 ? x : -INFINITY;
      bmax = fmaxf(bmax, sc[u]);
    }
    const float m_new = fmaxf(m, bmax);
    const float alpha = __builtin_amdgcn_exp2f(m - m_new);
    m = m_new;
    l *= alpha;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= alpha;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float p = __builtin_amdgcn_exp2f(sc[u] - m);
      l += p;
      float vf[8];
      unpack8p<Tr>(vx[u], vf);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(p, vf[e], acc[e]);
    }
  }

  // merge the KPL row groups of the wave, then the waves, each shifted by the gates of the runs behind its own
#pragma unroll
  for (int off = LPR; off < 64; off <<= 1) {
    const float m2 = __shfl_xor(m, off), l2 = __shfl_xor(l, off);
    float acc2[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc2[e] = __shfl_xor(acc[e], off);
    merge_runs(m, l, acc, m2, l2, acc2);
  }
  if (r == 0) {
    if (ch == 0) { part_m[wave] = m; part_l[wave] = l; part_g[wave] = behind; }
#pragma unroll
    for (int e = 0; e < 8; ++e) part_acc[wave][ch * 8 + e] = acc[e];
  }
  __syncthreads();
  if (tid >= LPR) return;
  m = part_m[0];
  l = part_l[0];
  double shift = part_g[0];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = part_acc[0][ch * 8 + e];
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    float acc2[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc2[e] = part_acc[w][ch * 8 + e];
    merge_runs(m, l, acc, part_m[w] + (float)shift * kLog2e, part_l[w], acc2);
    shift += part_g[w];
  }
  if (at.share.pieces > 1) {   // accumulator, maximum and sum relative to the piece's last key, sum of its gates
    const int64_t row = (int64_t)number * a.H + h;
    float* wo = a.ws_o + row * D + ch * 8;
    const f32x4 w0 = {acc[0], acc[1], acc[2], acc[3]}, w1 = {acc[4], acc[5], acc[6], acc[7]};
    *reinterpret_cast<f32x4*>(wo) = w0;
    *reinterpret_cast<f32x4*>(wo + 4) = w1;
    if (ch == 0) a.ws_p[row] = DecodePartial{shift, m, l};
    return;
  }
  const float inv = l > 0.f ? 1.0f / l : 0.f;   // no key at all: o = 0
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = Tr::pack2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  *reinterpret_cast<u32x4*>(a.o + b * a.o_sb + h * a.o_sh + ch * 8) = w;
}

// Merge of the pieces of a (row, head) by 256 threads, every partial in flight at once.
template <typename Tr, int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(const PagedDecodeK a) {
  constexpr int TPR = D / 4, GROUPS = 256 / TPR, PER = (kDecodeMaxSplits + GROUPS - 1) / GROUPS;
  __shared__ float weight[kDecodeMaxSplits];
  __shared__ float l_tot;
  __shared__ __align__(16) float part[GROUPS][D];
  const int tid = threadIdx.x, b = divide(blockIdx.x, a.by_heads), h = blockIdx.x - b * a.H;
  const PagedRow at = a.ws_row[b];   // (written there, not worked out again: another kernel's arithmetic need not round alike)
  const int pieces = at.pieces;
  if (pieces <= 1) return;   // written where it was computed
  const int grp = tid / TPR, d = (tid % TPR) * 4;
  const int64_t row0 = (int64_t)at.first * a.H + h;
  f32x4 x[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i)
    x[i] = *reinterpret_cast<const f32x4*>(a.ws_o + (row0 + (int64_t)min(grp + i * GROUPS, pieces - 1) * a.H) * D + d);
  if (tid < kWave) {   // one lane per piece (counted from the last keys): its maximum moves by the gates of the pieces behind it
    const DecodePartial p = a.ws_p[row0 + (int64_t)min(tid, pieces - 1) * a.H];
    const double excl = lane_before(wave_scan(tid < pieces ? p.g : 0.0));
    const float m = tid < pieces ? p.m + (float)excl * kLog2e : -INFINITY;
    float mx = m;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
    const float w = __builtin_amdgcn_exp2f(m - mx);
    float l = p.l * w;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off);
    weight[tid] = w;
    if (tid == 0) l_tot = l;
  }
  __syncthreads();
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (grp + i * GROUPS < pieces) acc += x[i] * weight[grp + i * GROUPS];
  *reinterpret_cast<f32x4*>(&part[grp][d]) = acc;
  __syncthreads();
  if (tid >= TPR) return;
  acc = *reinterpret_cast<const f32x4*>(&part[0][d]);
  const int used = min(GROUPS, pieces);
  for (int i = 1; i < used; ++i) acc += *reinterpret_cast<const f32x4*>(&part[i][d]);
  const float inv = l_tot > 0.f ? 1.0f / l_tot : 0.f;
  u32x2 w;
  w[0] = Tr::pack2(acc[0] * inv, acc[1] * inv);
  w[1] = Tr::pack2(acc[2] * inv, acc[3] * inv);
  *reinterpret_cast<u32x2*>(a.o + b * a.o_sb + h * a.o_sh + d) = w;
}

// Full pieces of all rows and heads together, at most: eight workgroups a CU.  4, 6, 12 and 16 instead of 8: geomean of 36
// shapes 1.014, 1.010, 1.004, 1.011 of the time.
constexpr int kPagedPieces = 8 * kCus;

static int64_t most_pieces(int max_keys, int D) {   // of a row
  const int64_t batches = ((int64_t)max_keys + paged_batch(D) - 1) / paged_batch(D);
  return batches < 1 ? 1 : batches < kDecodeMaxSplits ? batches : kDecodeMaxSplits;
}
// Workgroups: no row makes more pieces than its share of `pieces` and one for what is left over.
static int64_t paged_decode_workgroups(int B, int H, int max_keys, int D) {
  const int64_t by_row = (int64_t)B * H * most_pieces(max_keys, D), shared = kPagedPieces + (int64_t)B * H;
  return by_row < shared ? by_row : shared;
}
int64_t paged_decode_rows(int B, int H, int max_keys, int D) { return most_pieces(max_keys, D) > 1 ? paged_decode_workgroups(B, H, max_keys, D) : 0; }

template <typename Tr, int D>
static hipError_t launch_paged_decode_d(const PagedDecodeK& args, hipStream_t s) {
  PagedDecodeK a = args;
  a.per_piece = 1.0 / kPagedPieces;
  // Up to 255 rows every wave works the plan out from the lengths, 64 at a time, which a launch of its own would not make
  // up for (300 keys, H8 D64, us, waves / launch: 256 rows 41.0 / 40.4, 384 64.5 / 55.6, 1024 216 / 142; 64 rows take 12.2).
  a.planned = a.ws_row && a.B >= 256;
  if (a.planned) hipLaunchKernelGGL(paged_plan_kernel<D>, dim3(1), dim3(1024), 0, s, a);
  hipLaunchKernelGGL((paged_decode_kernel<Tr, D>), dim3((unsigned)paged_decode_workgroups(a.B, a.H, a.max_keys, D)), dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || most_pieces(a.max_keys, D) <= 1) return e;
  hipLaunchKernelGGL((paged_merge_kernel<Tr, D>), dim3((unsigned)((int64_t)a.B * a.H)), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <typename Tr>
static hipError_t launch_paged_decode_t(const PagedDecodeK& a, int D, hipStream_t s) {
  switch (D) {
    case 16: return launch_paged_decode_d<Tr, 16>(a, s);
    case 32: return launch_paged_decode_d<Tr, 32>(a, s);
    case 64: return launch_paged_decode_d<Tr, 64>(a, s);
    case 128: return launch_paged_decode_d<Tr, 128>(a, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_paged_decode(const PagedDecodeK& a, int D, int dtype, hipStream_t s) {
  return dtype == 0 ? launch_paged_decode_t<Bf16>(a, D, s) : launch_paged_decode_t<Fp16>(a, D, s);
}

}  // namespace fox
