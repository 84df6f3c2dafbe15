// Position rotation of queries and keys for gfx950, alone or in the pass of their per-head RMS norms:
//   n[t,h,:] = x[t,h,:] * rstd[t,h] * w[h,:],  rstd = 1 / sqrt(mean_d x^2 + eps)        (without weights n = x)
//   theta[t,i] = position[t] * inv_freq[i],  (a, b) = the i-th pair of the first R elements of n[t,h,:]
//   y = (a cos theta - b sin theta, a sin theta + b cos theta),  the rest of the head as it is.
// A pair is (i, i + R/2), or (2i, 2i+1) interleaved.  The rotation is orthogonal, so its gradient is the rotation by
// -theta; behind it the norm's backward, with dn the gradient turned back,
//   dw[h,:] = sum_t dn * xhat,  dx = rstd * (dn * w - xhat * mean_d(dn * w * xhat)),  xhat = x * rstd.
// The backward forms rstd again from the x that it reads anyway.
//
// All are streams over HBM.  A lane holds sixteen elements of a head, two 16-byte vectors chosen so that both halves of
// every pair are in the lane: vectors c and c + R/16 of the rotated part (2c and 2c+1 interleaved, and beyond the rotated
// part).  Row sums are DPP adds over the D/16 lanes of a head.  The angles are the same for all heads of a token: a workgroup
// forms them once per token, in 64 bits up to the fraction of a turn (a position of 2^20 would leave 32-bit angles 4 digits),
// and keeps cosine and sine in LDS.  A thread owns one column (tensor, head, sixteen elements).  Forward it takes one token:
// four, with all their rows in flight, keep fewer waves busy (30 shapes geomean 1.06 of the time).  Backward it walks
// tokens, so the weights are loaded once and their gradient stays in registers; partial gradients leave once per workgroup
// and are added in a fixed order.
//
// Rows are read through the caches, in which what the projections wrote a moment ago may still be, and written past them
// (norm and rotation B4 T512 H16 D128, us, both past them / as it is: forward 10.1 / 7.9, backward 24.7 / 21.3; long calls alike).
// B4 T16384 H16 D128, norm and rotation of q and k: 167 us forward, 296 backward (6.4 and 5.4 TB/s; a copy runs at 5.0 to 5.2).
#include "fox_common.hpp"
#include "fox_kernels.hpp"

namespace fox {

namespace {

template <typename Tr>
__device__ __forceinline__ void unpack8r(const u32x4& v, float* f) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = Tr::lo(v[e]);
    f[2 * e + 1] = Tr::hi(v[e]);
  }
}
template <typename Tr>
__device__ __forceinline__ u32x4 pack8r(const float* f) {
  u32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = Tr::pack2(f[2 * e], f[2 * e + 1]);
  return r;
}

// A thread's column: which tensor, head and vectors.
template <int D, bool INTERLEAVED>
struct Column {
  static constexpr int L = D / 16;   // lanes per head
  int side, h, c, v0, v1;
  __device__ __forceinline__ Column(const RotaryK& a, int col) {
    const int q_cols = a.side[0].H * L;
    side = col >= q_cols;
    const int in = col - (side ? q_cols : 0);
    h = in / L;
    c = in % L;
    const int half_vectors = a.R / 16;
    const bool apart = !INTERLEAVED && c < half_vectors;
    v0 = apart ? c : 2 * c;
    v1 = apart ? c + half_vectors : 2 * c + 1;
  }
};

// A thread's row lane and column.  In memory order, so that a wave reads whole lines: the lanes of a head, then the heads
// of a token or, where a head's tokens lie next to each other, the tokens of a head (norm and rotation with gradients of
// (B, H, T, D) memory, B4 T8192 H16 D32, us, heads / tokens first: 163 / 98; D64, two tokens a workgroup, 140 / 141).
template <int D>
__device__ __forceinline__ void place(const RotaryK& a, int& rl, int& col) {
  constexpr int L = D / 16;
  const int tid = threadIdx.x;
  if (a.cols > kRotaryThreads) {
    rl = 0;
    col = blockIdx.y * kRotaryThreads + tid;
  } else if (a.tokens_first) {
    const int unit = tid / L, head = divide(unit, a.by_lanes);
    rl = unit - head * a.lanes;
    col = head * L + tid % L;
  } else {
    rl = divide(tid, a.by_cols);
    col = tid - rl * a.cols;
  }
}

// Cosine and sine of a number of turns, to 2^-22 of their own magnitude: the hardware's are off by up to 1.25e-7, which is a thousandth of the sine
// that a low frequency has at its first positions, more than fp16's rounding.  The nearest quarter turn is taken off in 64
// bits; Taylor polynomials in the rest, x of at most pi / 4: the first terms left out are x^11 / 11! and x^12 / 12!, below
// 2^-28 of the values (us, the hardware's / these: rotation B8 T16000 H1 D64 12.0 / 13.5; from twelve heads on the same).
__device__ __forceinline__ float2 cos_sin_of_turns(double turns) {
#pragma clang fp contract(off)
  const double quarters = (turns - rint(turns)) * 4.0, nearest = rint(quarters);
  const float x = (float)((quarters - nearest) * 1.5707963267948966), z = x * x;
  const float s = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
  const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const int q = (int)nearest;   // -2 .. 2
  const float a = q & 1 ? s : c, b = q & 1 ? c : s;
  return float2{(q + 1) & 2 ? -a : a, q & 2 ? -b : b};
}

// cos and sin of the tile's tokens, pair by pair.  Executed by the whole workgroup.
template <int D>
__device__ __forceinline__ void make_angles(const RotaryK& a, int64_t n0, int tokens, float2 (*cs)[D / 2]) {
  const int half = a.R / 2;
  for (int i = threadIdx.x; i < tokens * half; i += blockDim.x) {
    const int tok = divide(i, a.by_half), pair = i - tok * half;
    const int64_t n = n0 + tok;
    if (n < a.N) {
      const int b = divide((int)n, a.by_T), t = (int)n - b * a.T;
      const int64_t pos = a.positions ? a.positions[b * a.p_sb + t * a.p_st] : a.first + t;
      const double turns = (double)pos * a.inv_freq[pair] * 0.15915494309189535;   // 1 / (2 pi)
      const float2 angle = cos_sin_of_turns(turns);
      cs[tok][pair] = float2{angle.x, a.sign < 0 ? -angle.y : angle.y};
    }
  }
}

// The lane's sixteen elements turned by the angles of its eight pairs; pairs outside the rotated part stay as they are
// (not turned by zero: an infinite element would make its neighbour NaN).  Halves: all of the lane's pairs or none.
template <bool INTERLEAVED>
__device__ __forceinline__ void turn(float (&f)[16], const float2* cs, int first_pair, int half) {
#pragma clang fp contract(off)
  if (first_pair >= half) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int ia = INTERLEAVED ? 2 * e : e, ib = INTERLEAVED ? 2 * e + 1 : 8 + e;
    const float2 t = cs[first_pair + e];
    const float x = f[ia], y = f[ib], a = fmaf(x, t.x, -(y * t.y)), b = fmaf(x, t.y, y * t.x);
    const bool in = !INTERLEAVED || first_pair + e < half;
    f[ia] = in ? a : x;
    f[ib] = in ? b : y;
  }
}

template <int L>
__device__ __forceinline__ float head_sum(float x) {
  if constexpr (L > 1) return row_sum<L>(x);
  return x;
}

}  // namespace

template <typename Tr, int D, bool NORM, bool INTERLEAVED>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(const RotaryK a) {
  constexpr int L = D / 16;
  __shared__ float2 cs[kRotaryLanes<D>][D / 2];
  int rl, col;
  place<D>(a, rl, col);
  const bool live = rl < a.lanes && col < a.cols;
  const Column<D, INTERLEAVED> at(a, live ? col : 0);
  const View in = at.side ? a.side[1].in : a.side[0].in, out = at.side ? a.side[1].out : a.side[0].out;
  const int64_t n0 = (int64_t)blockIdx.x * a.tile;
  float w[16];
  if constexpr (NORM) {
    const float* wp = (at.side ? a.side[1].w : a.side[0].w) + at.h * a.w_sh;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = wp[at.v0 * 8 + e];
      w[8 + e] = wp[at.v1 * 8 + e];
    }
  }
  const int n = (int)min(n0 + rl, (int64_t)a.N - 1);   // a token past the end reads the last one and is not stored
  const int b = divide(n, a.by_T), t = n - b * a.T;
  const uint16_t* from = in.ptr + b * in.sb + t * in.st + at.h * in.sh;
  const u32x4 x0 = *reinterpret_cast<const u32x4*>(from + at.v0 * 8), x1 = *reinterpret_cast<const u32x4*>(from + at.v1 * 8);
  make_angles<D>(a, n0, a.tile, cs);
  __syncthreads();
  float f[16];
  unpack8r<Tr>(x0, f);
  unpack8r<Tr>(x1, f + 8);
  if constexpr (NORM) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) ss += f[e] * f[e];
    const float rstd = 1.0f / sqrtf(head_sum<L>(ss) * (1.0f / D) + a.eps);
#pragma unroll
    for (int e = 0; e < 16; ++e) f[e] = f[e] * rstd * w[e];
  }
  if (live && n0 + rl < a.N) {
    turn<INTERLEAVED>(f, cs[rl], at.c * 8, a.R / 2);
    uint16_t* p = const_cast<uint16_t*>(out.ptr) + b * out.sb + t * out.st + at.h * out.sh;
    __builtin_nontemporal_store(pack8r<Tr>(f), reinterpret_cast<u32x4*>(p + at.v0 * 8));
    __builtin_nontemporal_store(pack8r<Tr>(f + 8), reinterpret_cast<u32x4*>(p + at.v1 * 8));
  }
}

// Gradient of the norm and the rotation behind it.  A workgroup walks a strip of `tiles` tiles, kRotaryRows tokens of a thread
// each: a barrier and new angles per tile, and always the rows of the next token on their way while those of one are used.
template <typename Tr, int D, bool INTERLEAVED>
__global__ __launch_bounds__(kRotaryThreads, 2) void qk_norm_rotary_bwd_kernel(const RotaryK a) {
  constexpr int L = D / 16;
  __shared__ float2 cs[2][kRotaryRows * kRotaryLanes<D>][D / 2];
  __shared__ __align__(16) float dw_s[kRotaryThreads * 16];
  const int tid = threadIdx.x;
  int rl, col;
  place<D>(a, rl, col);
  const bool live = rl < a.lanes && col < a.cols;
  const Column<D, INTERLEAVED> at(a, live ? col : 0);
  const View xv = at.side ? a.side[1].x : a.side[0].x, in = at.side ? a.side[1].in : a.side[0].in;
  const View out = at.side ? a.side[1].out : a.side[0].out;
  float w[16], dw[16];
  {
    const float* wp = (at.side ? a.side[1].w : a.side[0].w) + at.h * a.w_sh;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = wp[at.v0 * 8 + e];
      w[8 + e] = wp[at.v1 * 8 + e];
    }
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) dw[e] = 0.f;

  struct Row {
    u32x4 x0, x1, g0, g1;
  };
  auto load = [&](Row& r, int n) {   // tokens past the end read the last one and count for nothing
    n = min(n, a.N - 1);
    const int b = divide(n, a.by_T), t = n - b * a.T;
    const uint16_t* p = xv.ptr + b * xv.sb + t * xv.st + at.h * xv.sh;
    const uint16_t* g = in.ptr + b * in.sb + t * in.st + at.h * in.sh;
    r.x0 = *reinterpret_cast<const u32x4*>(p + at.v0 * 8);
    r.x1 = *reinterpret_cast<const u32x4*>(p + at.v1 * 8);
    r.g0 = *reinterpret_cast<const u32x4*>(g + at.v0 * 8);
    r.g1 = *reinterpret_cast<const u32x4*>(g + at.v1 * 8);
  };
  // Which products are fused into sums is written out: the compiler's choice differed between the copies of this code, so
  // that a token's place in the strip showed in its last bit.
  auto use = [&](const Row& r, int n, const float2* angles) {
#pragma clang fp contract(off)
    float x[16], g[16];
    unpack8r<Tr>(r.x0, x);
    unpack8r<Tr>(r.x1, x + 8);
    unpack8r<Tr>(r.g0, g);
    unpack8r<Tr>(r.g1, g + 8);
    turn<INTERLEAVED>(g, angles, at.c * 8, a.R / 2);
    float ss = 0.f, s1 = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      ss = fmaf(x[e], x[e], ss);
      s1 = fmaf(g[e] * w[e], x[e], s1);
    }
    const float rstd = 1.0f / sqrtf(fmaf(head_sum<L>(ss), 1.0f / D, a.eps));
    const float c1 = head_sum<L>(s1) * rstd * (1.0f / D);
    if (live && n < a.N) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float xhat = x[e] * rstd;
        dw[e] = fmaf(g[e], xhat, dw[e]);
        g[e] = fmaf(g[e], w[e], -(xhat * c1)) * rstd;
      }
      const int b = divide(n, a.by_T), t = n - b * a.T;
      uint16_t* p = const_cast<uint16_t*>(out.ptr) + b * out.sb + t * out.st + at.h * out.sh;
      __builtin_nontemporal_store(pack8r<Tr>(g), reinterpret_cast<u32x4*>(p + at.v0 * 8));
      __builtin_nontemporal_store(pack8r<Tr>(g + 8), reinterpret_cast<u32x4*>(p + at.v1 * 8));
    }
  };

  const int start = blockIdx.x * a.tiles * a.tile, stop = min(start + a.tiles * a.tile, a.N);   // (N is at most 2^30)
  Row even, odd;
  load(even, start + rl);
  make_angles<D>(a, start, a.tile, cs[0]);
  __syncthreads();
  int buf = 0;
  for (int n0 = start; n0 < stop; n0 += a.tile, buf ^= 1) {   // (the same steps in the whole workgroup)
    if (n0 + a.tile < stop) make_angles<D>(a, n0 + a.tile, a.tile, cs[buf ^ 1]);
#pragma unroll
    for (int u = 0; u < kRotaryRows; u += 2) {
      const int tok = rl + u * a.lanes;
      const float2* angles = cs[buf][live ? tok : 0];
      load(odd, n0 + tok + a.lanes);
      use(even, n0 + tok, angles);
      load(even, n0 + tok + 2 * a.lanes);   // (of the next tile behind this one's last)
      use(odd, n0 + tok + a.lanes, cs[buf][live ? tok + a.lanes : 0]);
    }
    __syncthreads();
  }

  // the workgroup's sums in element order: row lanes, and with shared weights heads, one after the other
  const bool wide = a.cols > kRotaryThreads;
  const int cols = wide ? min(kRotaryThreads, a.cols - (int)blockIdx.y * kRotaryThreads) : a.cols, col0 = wide ? blockIdx.y * kRotaryThreads : 0;
  if (live) {
    float* p = dw_s + rl * cols * 16 + (col - col0) / L * D;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[at.v0 * 8 + e] = dw[e];
      p[at.v1 * 8 + e] = dw[8 + e];
    }
  }
  __syncthreads();
  const int width = cols * 16;
  if (a.w_sh != 0) {
    float* dst = a.dw_partial + (int64_t)blockIdx.x * a.dw_width + col0 * 16;
    for (int j = tid; j < width; j += blockDim.x) {
      float sum = dw_s[j];
      for (int r = 1; r < a.lanes; ++r) sum += dw_s[r * width + j];
      dst[j] = sum;
    }
  } else {
    float* dst = a.dw_partial + ((int64_t)blockIdx.x * gridDim.y + blockIdx.y) * a.dw_width;
    const int q_elems = min(max(a.side[0].H * D - col0 * 16, 0), width);   // of this workgroup's columns
    for (int j = tid; j < a.dw_width; j += blockDim.x) {   // (2 * D, or D of one side alone)
      const int k0 = j < D ? j : q_elems + j - D, k1 = j < D ? q_elems : width;
      float sum = 0.f;
      for (int r = 0; r < a.lanes; ++r)
        for (int k = k0; k < k1; k += D) sum += dw_s[r * width + k];
      dst[j] = sum;
    }
  }
}

namespace {
// How a call over `tokens` tokens is cut: columns, workgroups' worth of them, row lanes of a workgroup, tokens a tile,
// tiles a workgroup.
struct RotaryPlan {
  int cols, chunks, lanes, tile, tiles;
  int64_t strips;
};
RotaryPlan rotary_plan(int64_t tokens, int heads, int D, bool bwd) {
  RotaryPlan p;
  p.cols = heads * (D / 16);
  p.chunks = (p.cols + kRotaryThreads - 1) / kRotaryThreads;
  p.lanes = p.cols > kRotaryThreads ? 1 : kRotaryThreads / p.cols;
  // as many as LDS holds the angles of: two workgroups a CU in the backward.  With a quarter of them few heads would leave workgroups of one
  // or two waves (norm and rotation with gradients B8 T4096 H1 D128, us, a quarter / as it is: 43.2 / 28.9; B33 T9954 H3 D32 29.4 / 31.7)
  if (p.lanes > 2048 / D) p.lanes = 2048 / D;   // kRotaryLanes
  p.tile = p.lanes * (bwd ? kRotaryRows : 1);
  // backward: strips for two workgroups a CU, at once.  Heads of several workgroups (chunks) that share weights can make
  // up to 512 + chunks partial gradients, more than one launch of the reduction adds.
  const int64_t tiles = (tokens + p.tile - 1) / p.tile, per = bwd ? (tiles * p.chunks + 2 * kCus - 1) / (2 * kCus) : 1;
  p.tiles = (int)per;
  p.strips = (tiles + per - 1) / per;
  return p;
}
}  // namespace

int64_t rotary_workspace_floats(int64_t tokens, int heads, int D, bool shared) {
  const RotaryPlan p = rotary_plan(tokens, heads, D, true);
  const int64_t width = shared ? 2 * D : (int64_t)heads * D;
  return reduce_rows_floats(shared ? p.strips * p.chunks : p.strips, width);
}

template <typename Tr, int D>
static hipError_t launch_rotary_d(const RotaryK& args, bool norm, bool interleaved, bool bwd, hipStream_t s) {
  RotaryK a = args;
  const int heads = a.side[0].H + a.side[1].H;
  const RotaryPlan p = rotary_plan(a.N, heads, D, bwd);
  a.cols = p.cols;
  a.lanes = p.lanes;
  a.tile = p.tile;
  a.tiles = p.tiles;
  a.dw_width = a.w_sh != 0 ? heads * D : a.side[1].H > 0 ? 2 * D : D;   // what the caller's buffer holds: no more is written
  a.by_T = divisor(a.T);
  a.by_half = divisor(a.R / 2);
  a.by_cols = divisor(p.cols);
  a.by_lanes = divisor(p.lanes);
  a.tokens_first = a.side[0].in.st < a.side[0].in.sh;
  const unsigned threads = p.cols > kRotaryThreads ? kRotaryThreads : (p.cols * p.lanes + 63) / 64 * 64;
  const dim3 grid((unsigned)p.strips, (unsigned)p.chunks), block(threads);
  if (!bwd) {
    if (norm && interleaved) hipLaunchKernelGGL((rotary_kernel<Tr, D, true, true>), grid, block, 0, s, a);
    else if (norm) hipLaunchKernelGGL((rotary_kernel<Tr, D, true, false>), grid, block, 0, s, a);
    else if (interleaved) hipLaunchKernelGGL((rotary_kernel<Tr, D, false, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((rotary_kernel<Tr, D, false, false>), grid, block, 0, s, a);
    return hipGetLastError();
  }
  if (interleaved) hipLaunchKernelGGL((qk_norm_rotary_bwd_kernel<Tr, D, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((qk_norm_rotary_bwd_kernel<Tr, D, false>), grid, block, 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  return launch_reduce_rows(a.dw_partial, a.dw, a.w_sh == 0 ? p.strips * p.chunks : p.strips, a.dw_width, s);
}

template <typename Tr>
static hipError_t launch_rotary_t(const RotaryK& a, int D, bool norm, bool interleaved, bool bwd, hipStream_t s) {
  switch (D) {
    case 16: return launch_rotary_d<Tr, 16>(a, norm, interleaved, bwd, s);
    case 32: return launch_rotary_d<Tr, 32>(a, norm, interleaved, bwd, s);
    case 64: return launch_rotary_d<Tr, 64>(a, norm, interleaved, bwd, s);
    case 128: return launch_rotary_d<Tr, 128>(a, norm, interleaved, bwd, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_rotary(const RotaryK& a, int D, int dtype, bool norm, bool interleaved, bool bwd, hipStream_t s) {
  return dtype == 0 ? launch_rotary_t<Bf16>(a, D, norm, interleaved, bwd, s) : launch_rotary_t<Fp16>(a, D, norm, interleaved, bwd, s);
}

}  // namespace fox
