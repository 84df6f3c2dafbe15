// Pages of 8-bit keys and values for gfx950: the append that quantises, the gather that reads back, and Forgetting Attention of one new token per request.
//
// A page of S tokens holds the codes of every key head's keys and values (P, Hk, S, D) and one fp32 scale for each block of G = min(S, 16) tokens and head; an
// element stands for code * scale.  The log gates, one for every query head, stay in 32 bits.  Codes are e4m3 (largest 448) or whole numbers (largest 127).
//
// The scales that the append gives are powers of two.  x / scale is exact then, so the code of a new element is one rounding of it (to the nearest, ties to the even one).  A block
// whose scale has to grow is rounded again from its codes: e4m3 keeps a code's bits at any scale down to its subnormals; those, and whole numbers, lose up to half a step of the new scale each time, and with
// the steps in front of it half as large or less, an element is off by less than one step of the last scale in all, where one rounding takes half of it.  Whole numbers lose half a bit on average against
// the scale that just fits.  The readers take any scales.
#include <algorithm>

#include "fox_common.hpp"
#include "fox_kernels.hpp"
#include "fox_paged_plan.hpp"

namespace fox {

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));

struct E4m3 {
  static constexpr float kLargest = 448.f;
  // exponent field of the smallest power of two by which a magnitude fits: 448 is 1.75 * 2^8
  static __device__ __forceinline__ int scale_exponent(uint32_t amax_bits) { return (int)((amax_bits + 0x1fffffu) >> 23) - 8; }
  static __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {   // of values within the largest, or NaN
    uint32_t w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  }
  static __device__ __forceinline__ void decode4(uint32_t w, float (&f)[4]) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    f[0] = lo[0]; f[1] = lo[1]; f[2] = hi[0]; f[3] = hi[1];
  }
  static __device__ __forceinline__ float clamped(float x) { return x == x ? fminf(fmaxf(x, -kLargest), kLargest) : x; }   // NaN stays one
  // four codes as bf16, which holds every one of them
  static __device__ __forceinline__ u32x2 bf16x4(uint32_t w) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))};
  }
  static __device__ __forceinline__ u32x2 f16x4(uint32_t w) {   // as fp16, which does as well
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))};
  }
};
struct Int8 {
  static constexpr float kLargest = 127.f;
  static __device__ __forceinline__ int scale_exponent(uint32_t amax_bits) { return (int)((amax_bits + 0x1ffffu) >> 23) - 6; }   // 127 is 1.984375 * 2^6
  static __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    auto one = [](float x) { return (uint32_t)(int)__builtin_rintf(x) & 0xffu; };
    return one(a) | one(b) << 8 | one(c) << 16 | one(d) << 24;
  }
  static __device__ __forceinline__ void decode4(uint32_t w, float (&f)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = (float)(int8_t)(w >> (8 * e));
  }
  static __device__ __forceinline__ float clamped(float x) { return x == x ? fminf(fmaxf(x, -kLargest), kLargest) : 0.f; }   // NaN becomes zero
  static __device__ __forceinline__ u32x2 bf16x4(uint32_t w) {
    float f[4];
    decode4(w, f);
    return u32x2{Bf16::pack2(f[0], f[1]), Bf16::pack2(f[2], f[3])};
  }
  static __device__ __forceinline__ u32x2 f16x4(uint32_t w) {
    float f[4];
    decode4(w, f);
    return u32x2{Fp16::pack2(f[0], f[1]), Fp16::pack2(f[2], f[3])};
  }
};

template <typename Tr>
__device__ __forceinline__ void unpack8(const u32x4& v, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = Tr::lo(v[e]);
    f[2 * e + 1] = Tr::hi(v[e]);
  }
}

}  // namespace

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
namespace {

// One tensor's rows of a run: `len` consecutive tokens into rows row0 .. of a block, whose rows in front of row0 stay.  Executed by a whole wave; lane / LPR is the row of a
// load, LPR lanes of eight elements each.
template <typename Tr, typename C, int D>
__device__ __forceinline__ void append_rows(const u32x4 (&x)[(16 * (D / 8) + 63) / 64], uint8_t* block, int64_t st, float* scale_at, int row0, int len, int lane) {
  constexpr int LPR = D / 8, R = 64 / LPR, NIT = (16 + R - 1) / R;
  const int r = lane / LPR, ch = lane % LPR;
  uint32_t amax = 0;   // bits of the largest finite magnitude
#pragma unroll
  for (int it = 0; it < NIT; ++it) {
    float f[8];
    unpack8<Tr>(x[it], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t m = __float_as_uint(f[e]) & 0x7fffffffu;
      if (it * R + r < len && m < 0x7f800000u) amax = max(amax, m);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, off));
  float scale = __uint_as_float((uint32_t)max(C::scale_exponent(amax), 1) << 23);
  const float old = row0 > 0 ? *scale_at : 0.f;
  scale = fmaxf(scale, old);
  if (row0 > 0 && scale != old) {   // the rows in front, rounded again to the larger scale
    const float ratio = old / scale;
    u32x2 w[NIT];
#pragma unroll
    for (int it = 0; it < NIT; ++it) w[it] = *reinterpret_cast<const u32x2*>(block + min(it * R + r, row0 - 1) * st + 8 * ch);
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      u32x2 y;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float f[4];
        C::decode4(w[it][i], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = C::clamped(f[e] * ratio);
        y[i] = C::encode4(f[0], f[1], f[2], f[3]);
      }
      if (it * R + r < row0) *reinterpret_cast<u32x2*>(block + (it * R + r) * st + 8 * ch) = y;
    }
  }
  const float inv = 1.0f / scale;
#pragma unroll
  for (int it = 0; it < NIT; ++it) {
    float f[8];
    unpack8<Tr>(x[it], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = C::clamped(f[e] * inv);
    const u32x2 y = {C::encode4(f[0], f[1], f[2], f[3]), C::encode4(f[4], f[5], f[6], f[7])};
    if (it * R + r < len) *reinterpret_cast<u32x2*>(block + (row0 + it * R + r) * st + 8 * ch) = y;
  }
  if (lane == 0 && scale != old) *scale_at = scale;
}

}  // namespace

// A run is what lies in one block of consecutive slots of consecutive tokens; its first token's wave of a key head takes it whole, so that the block's scale is known before
// a code is written and nobody waits for anybody.  A wave looks at CHUNK tokens of a head for the beginnings of runs: one token each where there are few (the next tokens
// of a step are runs of their own), sixteen where prompts fill whole blocks, so that few waves find nothing to do.  Few tokens are bound by their chain of loads: slots, scale, codes.
// In us for 1 / 4 / 8 / 16 tokens a wave: runs of one token, 48 of 12 heads, D 64 4.8 / 10.5 / 17.6 / 31.9, 1024 of 4 heads, D 128 8.1 / 13.1 / 22.8 / 43.4, 4096 22.9 / 21.5 / 26.7 / 43.7; whole
// blocks, 1024 tokens 8.8 / 6.2 / 5.9 / 5.8, 4096 27.2 / 11.4 / 6.3 / 6.3, 16384 95 / 29.5 / 17.4 / 11.4: repeated, its 52 MB in the last-level cache.
// Inputs that no cache holds take 18.8 us there, 2.8 TB/s.
template <typename Tr, typename C, int D, int CHUNK>
__global__ __launch_bounds__(256) void paged8_append_kernel(const Paged8AppendK a) {
  constexpr int LPR = D / 8, R = 64 / LPR, NIT = (16 + R - 1) / R;
  const int lane = threadIdx.x & 63, unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunk = divide(unit, a.by_heads), hk = unit - chunk * a.Hk, t0 = chunk * CHUNK;
  if (t0 >= a.T) return;
  const Pages8K& pg = a.pages;
  const int64_t slots = (int64_t)pg.P << pg.shift;
  const int block_rows = 1 << pg.block_shift;
  // lane i has the slot of token t0 - 1 + i
  int64_t slot = -2;
  if (lane <= CHUNK + 15) {
    const int t = t0 - 1 + lane;
    if (t >= 0 && t < a.T) slot = a.slots[t];
  }
  if (slot < 0 || slot >= slots) slot = -2;
  const int64_t before = __shfl_up(slot, 1);
  const bool follows = lane > 0 && slot >= 0 && before == slot - 1 && (slot & (block_rows - 1)) != 0;
  uint64_t starts = __ballot(lane > 0 && lane <= CHUNK && slot >= 0 && !follows);
  const uint64_t rest = __ballot(follows);
  const int r = lane / LPR, ch = lane % LPR;
  while (starts) {
    const int i = __ffsll((unsigned long long)starts) - 1;
    starts &= starts - 1;
    const int len = 1 + (__ffsll((unsigned long long)~(rest >> (i + 1))) - 1);   // (the run ends within the lanes that have a slot)
    const int64_t first = ((int64_t)__builtin_amdgcn_readlane((int)(slot >> 32), i) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)slot, i);
    const int t = t0 - 1 + i;
    u32x4 kx[NIT], vx[NIT];
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int64_t row = t + min(it * R + r, len - 1);
      kx[it] = *reinterpret_cast<const u32x4*>(a.k + row * a.k_st + hk * a.k_sh + 8 * ch);
      vx[it] = *reinterpret_cast<const u32x4*>(a.v + row * a.v_st + hk * a.v_sh + 8 * ch);
    }
    const int64_t page = first >> pg.shift;
    const int at = (int)(first & ((1 << pg.shift) - 1)), block = at >> pg.block_shift, row0 = at & (block_rows - 1);
    // the gates of the group's query heads: a token each of sixteen lanes
    const int tok = lane & 15;
    if (tok < len) {
      for (int j = lane >> 4; j < a.group; j += 4) {
        const int h = hk * a.group + j;
        pg.g[page * pg.g_sp + h * pg.g_sh + (at + tok) * pg.g_ss] = a.g[(int64_t)(t + tok) * a.g_st + h * a.g_sh];
      }
    }
    append_rows<Tr, C, D>(kx, pg.k.ptr + page * pg.k.sp + hk * pg.k.sh + (at - row0) * pg.k.st, pg.k.st, pg.k.scale + page * pg.k.s_sp + hk * pg.k.s_sh + block * pg.k.s_st, row0, len, lane);
    append_rows<Tr, C, D>(vx, pg.v.ptr + page * pg.v.sp + hk * pg.v.sh + (at - row0) * pg.v.st, pg.v.st, pg.v.scale + page * pg.v.s_sp + hk * pg.v.s_sh + block * pg.v.s_st, row0, len, lane);
  }
}

// ---------------------------------------------------------------------------
// Gather: the first tokens of requests out of their pages, one request after the other, in 16 bits.  A workgroup takes eight places: their requests from a search
// in the ends, their pages from the table, then rows of eight elements a lane, head by head, so that the codes of neighbouring tokens are read as they lie.
// Memory bounds it where there are many tokens; few need many workgroups.  In us for 4 / 8 / 16 / 32 places: 1600 tokens, 12 heads, D 64 4.8 / 4.7 / 5.8 / 7.8, 16384 tokens, 4 key heads, D 128
// 11.3 / 10.3 / 9.5 / 11.6, 80000 of those 40.3 / 37.5 / 37.1 / 36.7 (repeated; 40.9 for 37.5, 5.5 TB/s, on inputs that no cache holds).  Every workgroup reads all ends: 32768 tokens of 12 heads, D 64, of 64 requests
// 19.4, of 1024 22.4, of 4096 29.2.
// ---------------------------------------------------------------------------
constexpr int kGatherTokens = 8;

template <typename Tr, int CODES, int D>
__global__ __launch_bounds__(256) void paged_gather_kernel(const PagedGatherK a, const Divisor by_heads) {
  constexpr int LPR = D / 8, TOK = kGatherTokens, PER_HEAD = TOK * LPR;
  __shared__ int32_t ends[kPageRequests + 1];
  __shared__ int64_t slot_s[TOK];   // -1: zeros
  const int tid = threadIdx.x;
  const Pages8K& pg = a.pages;
  for (int i = tid; i <= a.B; i += 256) ends[i] = a.ends[i];
  for (int64_t t0 = (int64_t)blockIdx.x * TOK; t0 < a.T; t0 += (int64_t)gridDim.x * TOK) {
    __syncthreads();
    if (tid < TOK) {
      const int64_t t = t0 + tid;
      int lo = 0, hi = a.B;   // the first request whose tokens end behind t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid + 1] > t) hi = mid;
        else lo = mid + 1;
      }
      int64_t slot = -1;
      if (lo < a.B && t >= ends[lo]) {
        const int64_t pos = t - ends[lo], idx = pos >> pg.shift;
        const int who = a.requests ? a.requests[lo] : lo;
        if ((uint32_t)who < (uint32_t)a.R && idx < a.W) {
          const int page = a.table[who * a.table_sb + idx];
          if ((uint32_t)page < (uint32_t)pg.P) slot = ((int64_t)page << pg.shift) + (pos & ((1 << pg.shift) - 1));
        }
      }
      slot_s[tid] = slot;
    }
    __syncthreads();
    const int count = (int)min((int64_t)TOK, a.T - t0);
    for (int idx = tid; idx < PER_HEAD * a.Hk; idx += 256) {
      const int hk = idx / PER_HEAD, in = idx % PER_HEAD, tok = in / LPR, ch = in % LPR;
      if (tok >= count) continue;
      const int64_t slot = slot_s[tok], from = slot < 0 ? 0 : slot;
      const int64_t page = from >> pg.shift;
      const int at = (int)(from & ((1 << pg.shift) - 1));
      u32x4 out[2];
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const Pages8K::Codes& c = side ? pg.v : pg.k;
        if constexpr (CODES == kCodesNone) {
          out[side] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(c.ptr) + page * c.sp + hk * c.sh + at * c.st + 8 * ch);
        } else {
          const u32x2 w = *reinterpret_cast<const u32x2*>(c.ptr + page * c.sp + hk * c.sh + at * c.st + 8 * ch);
          const float scale = c.scale[page * c.s_sp + hk * c.s_sh + (at >> pg.block_shift) * c.s_st];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float f[4];
            if constexpr (CODES == kCodesE4m3) E4m3::decode4(w[i], f);
            else Int8::decode4(w[i], f);
            out[side][2 * i] = Tr::pack2(f[0] * scale, f[1] * scale);
            out[side][2 * i + 1] = Tr::pack2(f[2] * scale, f[3] * scale);
          }
        }
        if (slot < 0) out[side] = u32x4{0u, 0u, 0u, 0u};
      }
      const int64_t to = ((t0 + tok) * a.Hk + hk) * D + 8 * ch;
      *reinterpret_cast<u32x4*>(a.k + to) = out[0];
      *reinterpret_cast<u32x4*>(a.v + to) = out[1];
    }
    for (int idx = tid; idx < count * a.H; idx += 256) {
      const int tok = divide(idx, by_heads), h = idx - tok * a.H;
      const int64_t slot = slot_s[tok], from = slot < 0 ? 0 : slot;
      const float g = pg.g[(from >> pg.shift) * pg.g_sp + h * pg.g_sh + (from & ((1 << pg.shift) - 1)) * pg.g_ss];
      a.g[t0 * a.H + idx] = slot < 0 ? 0.f : g;
    }
  }
}

// ---------------------------------------------------------------------------
// Attention of one token per row over the 8-bit pages of its request, the query heads of a group together:
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(q.k_j sm_scale + sum of the log gates behind j up to the row's last key),  k = code * scale.
//
// 2*D bytes of codes a key and key head, 4*D flops for each of its query heads, so the group's heads share what is read: they are the sixteen columns of the matrix
// instructions (a group of one wastes fifteen, which costs nothing here: a CU's matrix units could take twelve times what memory brings).  Codes become 16-bit numbers on their
// way, exactly: those of K in the type of q, those of V in bf16, whose range has room for p times any scale, with p in two bf16 parts.  The products are as good as 32 bits.
//
//   S (16 keys x heads) = K Q^T: a lane holds 16 consecutive codes of a key, the contraction runs over the lanes' own order of the elements.  Rows of 128 codes are loaded as whole
//     lines and come to their lanes through LDS: in the operand's own order a load touches half of every line, and memory gives 5.0 TB/s in place of 6.4.
//   O^T (16 elements x heads) += V^T P^T: S leaves a lane four keys of one head, which are its part of P^T as they are; V goes through LDS and comes back transposed.
//
// Bound by HBM where caches are long: 32 requests of some 29000 tokens, 4 key heads, D 128, 985 MB of codes and gates in 158 to 165 us, 6.0 to 6.2 TB/s (the same loads alone 154 us); one request of
// 1500 tokens is a chain of round trips, 7.2 us, and the merge behind it another, 3.8.
//
// A wave walks whole batches of keys from the last one on, its sum of the gates behind it in 64 bits; runs, pieces, plan and merge are those of the 16-bit pages
// (fox_paged.hip).  Runs begin at multiples of a batch, so that sixteen keys lie in one block and four gates behind each other.
// ---------------------------------------------------------------------------
namespace {

__device__ __forceinline__ f32x4 mfma16(const u32x4& x, const u32x4& y, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
}
// of codes of K (8 of each lane) and q
template <typename Tr, typename C>
__device__ __forceinline__ f32x4 score16(uint32_t w0, uint32_t w1, const u32x4& q, const f32x4& c) {
  if constexpr (std::is_same_v<Tr, Fp16>) {
    const u32x2 x0 = C::f16x4(w0), x1 = C::f16x4(w1);
    const u32x4 k = {x0[0], x0[1], x1[0], x1[1]};
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
  } else {
    const u32x2 x0 = C::bf16x4(w0), x1 = C::bf16x4(w1);
    return mfma16(u32x4{x0[0], x0[1], x1[0], x1[1]}, q, c);
  }
}
// Two bf16 whose sum is x to 16 bits
struct Split {
  uint32_t hi, lo;   // of two numbers
};
__device__ __forceinline__ Split split2(float x, float y) {
  Split s;
  s.hi = Bf16::pack2(x, y);
  s.lo = Bf16::pack2(x - Bf16::lo(s.hi), y - Bf16::hi(s.hi));
  return s;
}

}  // namespace

// Keys that a wave has in registers at once, and waves a SIMD that the registers are held to (head dim 64 with 64 keys and three waves: 48 ragged requests 30.4 us, 28.9 so).
template <int D> constexpr int kPaged8Keys = D >= 64 ? 32 : 64;
template <int D> constexpr int kPaged8Waves = D >= 128 ? 3 : 4;

// VECTORS: four gates of consecutive tokens are read at once.  (Where the kernel chooses at run time nobody knows how many loads are on their way, and every step waits for all.)
// WAVES: four with runs of whole batches, pieces of a row for several workgroups; or one workgroup for a row, of as many waves as the registers allow, each with its share of the steps.
template <int D> constexpr int kPaged8RowWaves = D >= 128 ? 8 : 16;
template <typename Tr, typename C, int D, bool VECTORS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 4 ? kPaged8Waves<D> : WAVES / 4) void paged8_decode_kernel(const Paged8DecodeK a8) {
  constexpr int KEYS = kPaged8Keys<D>, NT = KEYS / 16;   // tiles of sixteen keys
  constexpr int STEPS = paged_batch(D) / 4 / KEYS;       // of a wave's batch
  constexpr int LB = D >= 64 ? 16 : 8;         // codes a lane loads at once
  constexpr int NL = D >= 64 ? D / 64 : 1;     // loads of a tile
  constexpr bool LINES = D == 128;             // a load takes eight whole rows of 128 bytes, else all sixteen rows
  constexpr int KS = D >= 32 ? D / 32 : 1;     // k-steps of a score
  constexpr int RS = 2 * D + (D >= 64 ? 32 : 16);   // bytes from one key to the next in LDS
  typedef std::conditional_t<LB == 16, u32x4, u32x2> Load;
  constexpr int AS = D + 4;                    // floats of a head's accumulator at the merge, where it takes the place of V
  static_assert(16 * AS * 4 <= 32 * RS, "a wave's accumulators fit where its V was");
  constexpr int KRS = D + 16;                  // bytes from one key to the next where K goes through LDS
  __shared__ __align__(16) char v_s[WAVES][32 * RS];
  static_assert(!LINES || KEYS * KRS <= 32 * RS, "K passes through the place of V, before V");
  __shared__ float part_m[WAVES][16], part_l[WAVES][16];
  __shared__ double part_g[WAVES][16];

  const PagedDecodeK& a = a8.row;
  const Pages8K& pg = a8.pages;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane & 15, g = lane >> 4;
  const int number = divide(blockIdx.x, a.by_heads), hp = blockIdx.x - number * a.H;
  const PagedPiece at = find_piece<D>(a, number, lane);
  if (at.b < 0) return;   // (the same in all waves)
  if (a.ws_row && !a.planned && at.piece == 0 && hp == 0 && tid == 0) a.ws_row[at.b] = PagedRow{at.first, at.share.pieces};   // for the merge
  const int b = at.b, hk = divide(hp, a8.by_parts), part = hp - hk * a8.parts;
  const int heads = min(a8.group - part * kPaged8Heads, kPaged8Heads), h0 = hk * a8.group + part * kPaged8Heads;   // of this workgroup
  const int32_t* table = a.table + (a.requests ? a.requests[b] : b) * a.table_sb;
  const uint8_t *kp = pg.k.ptr + hk * pg.k.sh, *vp = pg.v.ptr + hk * pg.v.sh;
  const float *ks = pg.k.scale + hk * pg.k.s_sh, *vs = pg.v.scale + hk * pg.v.s_sh;
  const float* gp = pg.g + (h0 + min(i16, heads - 1)) * pg.g_sh;   // (columns without a head repeat the last one's)
  const int in_page = (1 << pg.shift) - 1;
  // (strides in 32 bits: an address is one multiplication of 32 bits by 32)
  const uint32_t k_sp = (uint32_t)pg.k.sp, k_st = (uint32_t)pg.k.st, v_sp = (uint32_t)pg.v.sp, v_st = (uint32_t)pg.v.st, g_sp = (uint32_t)pg.g_sp, g_ss = (uint32_t)pg.g_ss;
  const uint32_t ks_sp = (uint32_t)pg.k.s_sp, ks_st = (uint32_t)pg.k.s_st, vs_sp = (uint32_t)pg.v.s_sp, vs_st = (uint32_t)pg.v.s_st;

  // run of this wave in steps, from the last
  const int keys = at.share.keys, steps = (keys + KEYS - 1) / KEYS;
  int s0, s1;
  if constexpr (WAVES == 4) {
    const int all = (keys + KEYS * STEPS - 1) / (KEYS * STEPS), per = at.share.batches, b1 = max(all - (at.piece * 4 + wave) * per, 0);
    s0 = max(b1 - per, 0) * STEPS;
    s1 = min(b1 * STEPS, steps);
  } else {
    const int per = (steps + WAVES - 1) / WAVES;
    s1 = max(steps - wave * per, 0);
    s0 = max(s1 - per, 0);
  }

  // element e of k-step s of a lane is number elem0(s) + e of its row
  auto elem0 = [&](int s) { return D >= 64 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 8 * g; };
  u32x4 q[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const bool there = D >= 32 || g < 2;
    q[s] = *reinterpret_cast<const u32x4*>(a.q + b * a.q_sb + (h0 + min(i16, heads - 1)) * a.q_sh + (there ? elem0(s) : 0));
    if (!there || i16 >= heads) q[s] = u32x4{0u, 0u, 0u, 0u};
  }
  const float qk_scale = a.sm_scale * kLog2e;
  float m = -3.0e38f, l = 0.f;   // of this lane's head; finite floor: what has seen no key yet yields exp2(-inf) = 0
  f32x4 acc[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  double behind = 0.0;           // sum of the run's gates behind the step, of this lane's head
  int page0 = INT32_MAX, entry = -1;   // this lane has the table's entry for page page0 + lane
  char* const v_tile = v_s[wave];

  // What a step needs, each part requested for the next step as soon as this one has used it: the codes and gates of K before the weights are worked out, those of V when they
  // are in LDS.  A step's loads are in flight during most of the one before, without a second set of registers.
  Load kx[NT][NL], vx[NT][NL];   // codes of this lane's keys of every tile
  f32x4 gate[NT];                // of the four keys of every tile whose scores this lane will have,
  float ksc[NT], vsc[NT];        // their scales
  int page[2 * NT];              // of every eight keys
  bool whole = true;             // every key of the step counts; else
  uint32_t ok = 0;               // bit NL t + c: this lane's key of load c of tile t does, bit 8 + 4 t + r: its r-th score
  // A tile begins at a multiple of sixteen tokens: a lane's row in its page is the tile's and its own, both fixed, and the blocks of its keys are the tile's.  Rows past the
  // last key lie on the last key's page.
  const uint32_t lane_row = LINES ? lane >> 3 : i16 & in_page, lane_off = LINES ? 16 * (lane & 7) : LB == 16 ? 16 * g : D == 32 ? 8 * g : 8 * (g & 1);
  const uint32_t k_lane = lane_row * k_st + lane_off, v_lane = lane_row * v_st + lane_off, g_lane = (4 * g & in_page) * g_ss;
  // address of load c of tile t, in codes from the beginning of the head's
  auto code_at = [&](int n0, int t, int c, uint32_t sp, uint32_t st, uint32_t own) {
    const int first = n0 + 16 * t + (LINES ? 8 * c : 0);
    const uint32_t p = LINES ? page[2 * t + c] : i16 < 8 ? page[2 * t] : page[2 * t + 1];
    return (uint64_t)p * sp + ((first & in_page) * st + own + (LINES ? 0 : 64 * c));
  };
  auto page_of_scores = [&](int t) { return (uint32_t)(g < 2 ? page[2 * t] : page[2 * t + 1]); };
  auto fetch_k = [&](int step) {
    const int n0 = step * KEYS;
    if ((n0 >> pg.shift) < page0) {
      page0 = max(((min(n0 + KEYS, keys) - 1) >> pg.shift) - 63, 0);
      entry = table[min(page0 + lane, a.W - 1)];
      if ((uint32_t)entry >= (uint32_t)pg.P) entry = -1;
      asm volatile("" : "+v"(entry));   // (waited for here: behind the branch every step would wait for all that is on its way)
    }
    whole = n0 + KEYS <= keys;
#pragma unroll
    for (int e = 0; e < 2 * NT; ++e) {
      page[e] = __builtin_amdgcn_readlane(entry, (min(n0 + 8 * e, keys - 1) >> pg.shift) - page0);
      whole &= page[e] >= 0;
    }
    if (!whole) {
      ok = 0;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int c = 0; c < NL; ++c) {
          const int n = n0 + 16 * t + (LINES ? 8 * c + (lane >> 3) : i16), p = LINES ? page[2 * t + c] : i16 < 8 ? page[2 * t] : page[2 * t + 1];
          ok |= (uint32_t)(n < keys && p >= 0) << (NL * t + c);
        }
        if ((int)page_of_scores(t) >= 0) ok |= ((1u << min(max(keys - (n0 + 16 * t + 4 * g), 0), 4)) - 1) << (8 + 4 * t);
      }
#pragma unroll
      for (int e = 0; e < 2 * NT; ++e) page[e] = max(page[e], 0);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < NL; ++c) kx[t][c] = __builtin_nontemporal_load(reinterpret_cast<const Load*>(kp + code_at(n0, t, c, k_sp, k_st, k_lane)));
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint32_t row = (n0 + 16 * t) & in_page, p = page_of_scores(t);
      const float* at = gp + ((uint64_t)p * g_sp + (row * g_ss + g_lane));
      if constexpr (VECTORS) {
        gate[t] = *reinterpret_cast<const f32x4*>(at);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) gate[t][r] = at[r * g_ss];
      }
      ksc[t] = ks[(uint64_t)p * ks_sp + (row >> pg.block_shift) * ks_st];
    }
  };
  auto fetch_v = [&](int step, int t) {   // behind fetch_k of the same step
    const int n0 = step * KEYS;
#pragma unroll
    for (int c = 0; c < NL; ++c) vx[t][c] = __builtin_nontemporal_load(reinterpret_cast<const Load*>(vp + code_at(n0, t, c, v_sp, v_st, v_lane)));
    vsc[t] = vs[(uint64_t)page_of_scores(t) * vs_sp + (((n0 + 16 * t) & in_page) >> pg.block_shift) * vs_st];
  };
  auto work = [&](int step, auto more) {   // more: there is a step in front of this one
    constexpr bool kMore = decltype(more)::value;
    f32x4 s[NT];
    if constexpr (LINES) {   // whole rows: a lane's part of the operand lies with other lanes
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < NL; ++c) *reinterpret_cast<Load*>(v_tile + (16 * t + 8 * c + (lane >> 3)) * KRS + 16 * (lane & 7)) = kx[t][c];
      staged_rows_visible();
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < NL; ++c) kx[t][c] = *reinterpret_cast<const Load*>(v_tile + (16 * t + i16) * KRS + 64 * c + 16 * g);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const Load& w = kx[t][LB == 16 ? i >> 1 : 0];
        const int o = LB == 16 ? 2 * (i & 1) : 0;
        s[t] = score16<Tr, C>(w[o], w[o + 1], q[i], s[t]);
      }
    }
    // What is masked may hold anything, NaN among it; in most steps nothing is.
    const bool whole_now = whole;
    const uint32_t ok_now = ok;
    if (!whole_now) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) gate[t][r] = ok >> (8 + 4 * t + r) & 1 ? gate[t][r] : 0.f;
    }
    // biases, from the last tile on, and the maximum
    float top = -INFINITY;
#pragma unroll
    for (int t = NT - 1; t >= 0; --t) {
      float own[4], sum = 0.f;   // own[r]: gates of the lane's keys behind key r
#pragma unroll
      for (int r = 3; r >= 0; --r) {
        own[r] = sum;
        sum += gate[t][r];
      }
      const float next = __shfl_xor(sum, 16), pair = sum + next, other = __shfl_xor(pair, 32);
      const float after = (float)behind + ((g & 1 ? 0.f : next) + (g & 2 ? 0.f : other));   // with those of the lanes whose keys lie behind
      const float scale = ksc[t] * qk_scale;
#pragma unroll
      for (int r = 0; r < 4; ++r) s[t][r] = fmaf(s[t][r], scale, (own[r] + after) * kLog2e);
      behind += (double)(pair + other);
    }
    if (!whole_now) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[t][r] = ok_now >> (8 + 4 * t + r) & 1 ? s[t][r] : -INFINITY;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[t][r]);
    if constexpr (kMore) fetch_k(step - 1);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    // The maximum is raised when a step exceeds it by more than 2^8, which is rare behind the first ones.
    const bool raise = top > m + 8.f;
    if (__any(raise)) {
      const float m_new = raise ? top : m, alpha = __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) acc[d] *= alpha;
    }
    // O^T += V^T P^T, 32 keys at a time
#pragma unroll
    for (int u = 0; u < NT / 2; ++u) {
      if (!whole_now) {
#pragma unroll
        for (int t = 2 * u; t < 2 * u + 2; ++t) {
          if ((ok_now >> (8 + 4 * t) & 15) == 0) vsc[t] = 0.f;   // (a block that holds no key may have any scale)
#pragma unroll
          for (int c = 0; c < NL; ++c)
            if (!(ok_now >> (NL * t + c) & 1)) vx[t][c] = Load{};
        }
      }
      u32x4 ph, pl;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[r] = __builtin_amdgcn_exp2f(s[2 * u + t][r] - m);
          l += p[r];
          p[r] *= vsc[2 * u + t];
        }
        const Split y0 = split2(p[0], p[1]), y1 = split2(p[2], p[3]);
        ph[2 * t] = y0.hi; ph[2 * t + 1] = y1.hi;
        pl[2 * t] = y0.lo; pl[2 * t + 1] = y1.lo;
      }
      __builtin_amdgcn_wave_barrier();   // (the reads of the 32 keys before come first)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int c = 0; c < NL; ++c) {
          const Load w = vx[2 * u + t][c];
          char* row = v_tile + (LINES ? 16 * t + 8 * c + (lane >> 3) : 16 * t + i16) * RS;
#pragma unroll
          for (int half = 0; half < LB / 8; ++half) {
            const u32x2 x0 = C::bf16x4(w[2 * half]), x1 = C::bf16x4(w[2 * half + 1]);
            const int d = LINES ? 16 * (lane & 7) + 8 * half : LB == 16 ? 64 * c + 16 * g + 8 * half : 8 * g;
            if (D >= 32 || g < 2) *reinterpret_cast<u32x4*>(row + 2 * d) = u32x4{x0[0], x0[1], x1[0], x1[1]};
          }
        }
      }
      if constexpr (kMore) {
        fetch_v(step - 1, 2 * u);
        fetch_v(step - 1, 2 * u + 1);
      }
      staged_rows_visible();
      const char* src = v_tile + (4 * g + (i16 >> 2)) * RS + 8 * (i16 & 3);
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        const u32x2 lo = lds_tr_read(src + 32 * d), hi = lds_tr_read(src + 16 * RS + 32 * d);
        const u32x4 va = {lo[0], lo[1], hi[0], hi[1]};
        acc[d] = mfma16(va, ph, acc[d]);
        acc[d] = mfma16(va, pl, acc[d]);
      }
    }
  };
  if (s1 > s0) {
    fetch_k(s1 - 1);
#pragma unroll
    for (int t = 0; t < NT; ++t) fetch_v(s1 - 1, t);
    for (int step = s1 - 1; step > s0; --step) work(step, std::true_type{});
    work(s0, std::false_type{});
  }

  // merge the waves, each shifted by the gates of the runs behind its own
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (g == 0) {
    part_m[wave][i16] = m;
    part_l[wave][i16] = l;
    part_g[wave][i16] = behind;
  }
  __builtin_amdgcn_wave_barrier();   // (the last reads of V come first)
#pragma unroll
  for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f32x4*>(v_tile + (i16 * AS + 16 * d + 4 * g) * 4) = acc[d];
  __syncthreads();
  constexpr int CPH = D / 4;   // threads of a head, four elements each
  for (int idx = tid; idx < heads * CPH; idx += 64 * WAVES) {
    const int j = idx / CPH, d = idx % CPH * 4, h = h0 + j;
    float mw[WAVES], top = part_m[0][j];
    double shift = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      mw[w] = part_m[w][j] + (float)shift * kLog2e;
      shift += part_g[w][j];
      top = fmaxf(top, mw[w]);
    }
    float lt = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float weight = __builtin_amdgcn_exp2f(mw[w] - top);
      lt += part_l[w][j] * weight;
      o += *reinterpret_cast<const f32x4*>(v_s[w] + (j * AS + d) * 4) * weight;
    }
    if (at.share.pieces > 1) {   // accumulator, maximum and sum relative to the piece's last key, sum of its gates
      const int64_t row = (int64_t)number * a8.heads + h;
      *reinterpret_cast<f32x4*>(a.ws_o + row * D + d) = o;
      if (d == 0) a.ws_p[row] = DecodePartial{shift, top, lt};
    } else {
      const float inv = lt > 0.f ? 1.0f / lt : 0.f;   // no key at all: o = 0
      *reinterpret_cast<u32x2*>(a.o + b * a.o_sb + h * a.o_sh + d) = u32x2{Tr::pack2(o[0] * inv, o[1] * inv), Tr::pack2(o[2] * inv, o[3] * inv)};
    }
  }
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
template <typename Tr, typename C, int D>
static hipError_t append_d(const Paged8AppendK& a, hipStream_t s) {
  const auto grid = [&](int chunk) { return dim3((unsigned)(((int64_t)((a.T + chunk - 1) / chunk) * a.Hk + 3) / 4)); };
  const int64_t rows = (int64_t)a.T * a.Hk;
  if (rows <= 16 * kCus) hipLaunchKernelGGL((paged8_append_kernel<Tr, C, D, 1>), grid(1), dim3(256), 0, s, a);
  else if (rows <= 128 * kCus) hipLaunchKernelGGL((paged8_append_kernel<Tr, C, D, 8>), grid(8), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((paged8_append_kernel<Tr, C, D, 16>), grid(16), dim3(256), 0, s, a);
  return hipGetLastError();
}
// Whether rows stay whole, a large workgroup each and no merge behind.  That takes some 4.7 us and 0.07 us for each 1000 elements of a row's keys, while there are CUs for all rows; in pieces it is
// 11 us and what the bytes of all rows take.  (Whole / pieces, us: D 64, 12 rows of 500 keys 7.1 / 10.3, of 1500 11.9 / 10.9, 96 of 1500 12.4 / 13.3, 240 of 1500 13.2 / 20.8, 384 23.5 / 27.9, 576
// 34.4 / 33.4; D 128, 32 rows of 500 9.0 / 11.2, of 1000 12.6 / 11.1, 256 of 1500 20.5 / 28.6.)  What the host knows is the longest a row can be, so very long rows are left to pieces: others may be short.
static bool whole_rows(const Paged8DecodeK& a, int D) {
  const int64_t rows = (int64_t)a.row.B * a.row.H, elements = (int64_t)a.row.max_keys * D;
  return rows <= kCus && elements <= 1 << 18 && elements * (200 - rows) <= 17000000;
}
template <typename Tr, typename C, int D>
static hipError_t decode8_d(const Paged8DecodeK& args, hipStream_t s) {
  Paged8DecodeK a = args;
  if (whole_rows(a, D)) {
    a.row.ws_row = nullptr;
    constexpr int WAVES = kPaged8RowWaves<D>;
    const dim3 rows((unsigned)(a.row.B * a.row.H));
    if (a.gates_in_vectors) hipLaunchKernelGGL((paged8_decode_kernel<Tr, C, D, true, WAVES>), rows, dim3(64 * WAVES), 0, s, a);
    else hipLaunchKernelGGL((paged8_decode_kernel<Tr, C, D, false, WAVES>), rows, dim3(64 * WAVES), 0, s, a);
    return hipGetLastError();
  }
  a.row.per_piece = 1.0 / kPagedPieces;
  a.row.batch_us = 5.f;
  a.row.planned = plan_ahead(a.row);
  if (a.row.planned) {
    const hipError_t e = launch_paged_plan(a.row, D, s);
    if (e != hipSuccess) return e;
  }
  const dim3 grid((unsigned)paged_decode_workgroups(a.row.B, a.row.H, a.row.max_keys, D));
  if (a.gates_in_vectors) hipLaunchKernelGGL((paged8_decode_kernel<Tr, C, D, true, 4>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((paged8_decode_kernel<Tr, C, D, false, 4>), grid, dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || most_pieces(a.row.max_keys, D) <= 1) return e;
  PagedDecodeK m = a.row;   // the merge goes by query heads
  m.H = a.heads;
  m.by_heads = divisor(a.heads);
  return launch_paged_merge(m, D, std::is_same_v<Tr, Bf16> ? 0 : 1, s);
}

#define FOX_BY_HEAD_DIM(D, CALL)         \
  switch (D) {                           \
    case 16: return CALL(16);            \
    case 32: return CALL(32);            \
    case 64: return CALL(64);            \
    case 128: return CALL(128);          \
    default: return hipErrorInvalidValue; \
  }

template <typename Tr, typename C>
static hipError_t append_t(const Paged8AppendK& a, int D, hipStream_t s) {
#define FOX_CALL(N) append_d<Tr, C, N>(a, s)
  FOX_BY_HEAD_DIM(D, FOX_CALL)
#undef FOX_CALL
}
template <typename Tr, typename C>
static hipError_t decode8_t(const Paged8DecodeK& a, int D, hipStream_t s) {
#define FOX_CALL(N) decode8_d<Tr, C, N>(a, s)
  FOX_BY_HEAD_DIM(D, FOX_CALL)
#undef FOX_CALL
}
template <typename Tr, int CODES, int D>
static hipError_t gather_d(const PagedGatherK& a, hipStream_t s) {
  const int64_t groups = ((int64_t)a.T + kGatherTokens - 1) / kGatherTokens;
  hipLaunchKernelGGL((paged_gather_kernel<Tr, CODES, D>), dim3((unsigned)std::min<int64_t>(groups, 1 << 22)), dim3(256), 0, s, a, divisor(a.H));
  return hipGetLastError();
}
template <typename Tr, int CODES>
static hipError_t gather_t(const PagedGatherK& a, int D, hipStream_t s) {
#define FOX_CALL(N) gather_d<Tr, CODES, N>(a, s)
  FOX_BY_HEAD_DIM(D, FOX_CALL)
#undef FOX_CALL
}

hipError_t launch_paged8_append(const Paged8AppendK& a, int D, int dtype, int codes, hipStream_t s) {
  if (codes == kCodesE4m3) return dtype == 0 ? append_t<Bf16, E4m3>(a, D, s) : append_t<Fp16, E4m3>(a, D, s);
  return dtype == 0 ? append_t<Bf16, Int8>(a, D, s) : append_t<Fp16, Int8>(a, D, s);
}
hipError_t launch_paged_gather(const PagedGatherK& a, int D, int dtype, int codes, hipStream_t s) {
  if (codes == kCodesNone) return gather_t<Bf16, kCodesNone>(a, D, s);   // (copied: the type does not matter)
  if (codes == kCodesE4m3) return dtype == 0 ? gather_t<Bf16, kCodesE4m3>(a, D, s) : gather_t<Fp16, kCodesE4m3>(a, D, s);
  return dtype == 0 ? gather_t<Bf16, kCodesInt8>(a, D, s) : gather_t<Fp16, kCodesInt8>(a, D, s);
}
hipError_t launch_paged8_decode(const Paged8DecodeK& a, int D, int dtype, int codes, hipStream_t s) {
  if (codes == kCodesE4m3) return dtype == 0 ? decode8_t<Bf16, E4m3>(a, D, s) : decode8_t<Fp16, E4m3>(a, D, s);
  return dtype == 0 ? decode8_t<Bf16, Int8>(a, D, s) : decode8_t<Fp16, Int8>(a, D, s);
}

}  // namespace fox
