// kv8_cache.hip -- what goes into the paged 8-bit cache and comes back out of it
// (gfx950).
//
// A block of 64 slots of one head has one scale for K and one for V, the least 2^e with
// max|x| <= 448 * 2^e, so its values' maximum has to be known before the first code is: who
// encodes a block holds all its new tokens in registers meanwhile, and reads each once.  All
// of it moves bytes; nothing is bound by arithmetic.
#include <algorithm>

#include "dsa_launch.h"
#include "kv8.h"

namespace dsa {
namespace {

constexpr int kNT = 256;

// A pair (a, b) at position p becomes (a cos - b sin, b cos + a sin).  Products and
// sums are rounded one by one (no fma), as torch's elementary operations round them.
__device__ __forceinline__ float turn_a(float a, float b, float c, float s) {
#pragma clang fp contract(off)
  const float x = a * c, y = b * s;
  return x - y;
}
__device__ __forceinline__ float turn_b(float a, float b, float c, float s) {
#pragma clang fp contract(off)
  const float x = b * c, y = a * s;
  return x + y;
}

// A thread takes 16 elements of a row, unit u: elements lo .. lo+7 and hi .. hi+7, which are
// the pairs where halves turn; neighbouring units are neighbours in memory.
struct Unit {
  int lo, hi;
  bool turn_lo, turn_hi;
};
__device__ __forceinline__ Unit unit_of(int u, int D, int R, bool pairs) {
  if (!pairs && 16 * u < R) return {8 * u, 8 * u + R / 2, true, true};
  const int from = pairs ? 0 : R, lo = from + 8 * u - from / 2, hi = lo + (D - from) / 2;
  return {lo, hi, lo < R, hi < R};
}
struct Angles {
  float c[8], s[8];
};
__device__ __forceinline__ void load_angles(const Kv8Append& a, const Unit& un, int64_t at, Angles& g) {
  const int64_t row = at * (a.R / 2);
  if (!a.pairs) {
    if (!un.turn_lo) return;
    load_f32<8>(a.cos + row + un.lo, g.c);
    load_f32<8>(a.sin + row + un.lo, g.s);
    return;
  }
  if (un.turn_lo) {
    *reinterpret_cast<f32x4*>(g.c) = *reinterpret_cast<const f32x4*>(a.cos + row + un.lo / 2);
    *reinterpret_cast<f32x4*>(g.s) = *reinterpret_cast<const f32x4*>(a.sin + row + un.lo / 2);
  }
  if (un.turn_hi) {
    *reinterpret_cast<f32x4*>(g.c + 4) = *reinterpret_cast<const f32x4*>(a.cos + row + un.hi / 2);
    *reinterpret_cast<f32x4*>(g.s + 4) = *reinterpret_cast<const f32x4*>(a.sin + row + un.hi / 2);
  }
}
__device__ __forceinline__ void turn_pairs(float (&x)[8], const float* c, const float* s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = x[2 * i], b = x[2 * i + 1];
    x[2 * i] = turn_a(a, b, c[i], s[i]);
    x[2 * i + 1] = turn_b(a, b, c[i], s[i]);
  }
}
__device__ __forceinline__ void turn(float (&lo)[8], float (&hi)[8], const Angles& g, const Unit& un, bool pairs) {
  if (pairs) {
    if (un.turn_lo) turn_pairs(lo, g.c, g.s);
    if (un.turn_hi) turn_pairs(hi, g.c + 4, g.s + 4);
  } else if (un.turn_lo) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = lo[i], b = hi[i];
      lo[i] = turn_a(a, b, g.c[i], g.s[i]);
      hi[i] = turn_b(a, b, g.c[i], g.s[i]);
    }
  }
}

template <typename Tag>
__device__ __forceinline__ void store8(typename Tag::raw* p, const float (&x)[8]) {
  if constexpr (Tag::kBytes == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 v{x[2 * j], x[2 * j + 1]};
      if constexpr (__is_same(Tag, BF16)) w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
      else w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t m = __float_as_uint(x) & 0x7fffffffu;
  return m < 0x7f800000u ? m : 0u;
}
// x / scale to the nearest e4m3 (ties to even); Inf and NaN become NaN, e4m3 has no Inf.
__device__ __forceinline__ float scaled(float x, float inverse) {
  return (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u ? x * inverse : __builtin_nanf("");
}
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}
// Four codes at another scale: f = 2^(old - new) <= 1, exact up to the codes' own rounding.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float f) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  return encode4(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
}

__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) { return wave_extreme_u32<true>(v); }

// Where sequence b's new tokens go: slots [have, end) of those that the sequence has.
struct Span {
  int64_t have, end;
  int64_t many;
};
__device__ __forceinline__ Span span_of(const Kv8& c, const Kv8Append& a, int64_t b) {
  Span s;
  const int64_t S = c.slots();
  s.have = a.start ? max(int64_t{0}, min(static_cast<int64_t>(a.start[b]), S)) : kv8_length(c, b);
  s.many = a.count ? max(int64_t{0}, min(static_cast<int64_t>(a.count[b]), a.T)) : a.T;
  s.end = min(s.have + s.many, S);
  return s;
}

// Sequence b's counters, by one block: length, and the tokens past the last slot or
// on a page that is none.
__device__ __forceinline__ void update_counts(const Kv8& c, const Span& s, int64_t b) {
  __shared__ int32_t bad;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  const int shift = c.page_shift + 6;
  int32_t mine = 0;
  for (int64_t p = (s.have >> shift) + threadIdx.x; p << shift < s.end; p += blockDim.x) {
    const int32_t id = c.pages[b * c.max_pages + p];
    if (id < 0 || id >= c.NP)
      mine += static_cast<int32_t>(min(s.end, (p + 1) << shift) - max(s.have, p << shift));
  }
  if (mine) atomicAdd(&bad, mine);
  __syncthreads();
  if (threadIdx.x == 0) {
    c.length[b] = static_cast<int32_t>(s.end);
    c.lost[b] += bad + static_cast<int32_t>(s.many - (s.end - s.have));
  }
}

// f = 2^(old - new) for codes whose scale grows.
__device__ __forceinline__ float fall_of(uint32_t old_byte, uint32_t new_byte) {
  return new_byte - old_byte > 40 ? 0.0f : __uint_as_float((127u + old_byte - new_byte) << 23);
}
__device__ __forceinline__ uint2 encode8(const float (&x)[8], float inverse) {
  return make_uint2(encode4(scaled(x[0], inverse), scaled(x[1], inverse), scaled(x[2], inverse), scaled(x[3], inverse)),
                    encode4(scaled(x[4], inverse), scaled(x[5], inverse), scaled(x[6], inverse), scaled(x[7], inverse)));
}
__device__ __forceinline__ void make_nan(float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __builtin_nanf("");
}
// Of a dimension's 16 words of V, word w holds tokens t .. t + 3.
__device__ __forceinline__ int word_token(int w) { return (w & 3) * 16 + (w >> 2) * 4; }

// A block of threads takes a group of heads of one block of 64 slots, with the angles of
// its tokens in registers: K/V heads one after another (short ones two or four side by
// side), or query heads.  Of K a thread has one unit of some tokens; of V 4 tokens by 8
// dimensions, which it turns into words of 4 tokens (a word of the cache has one owner,
// so bytes that stay are merged without a barrier, and a wave writes whole rows of 64).
//
// Bound by memory: 2 x 16384 tokens of 32 and 8 heads of 128 in bf16 with rotated keys, 805 MB
// read and written, take 190 us, 4.2 TB/s where a large copy reaches 5.1.  (A block a head, which
// loads the angles anew for each, took 251.)  8 prompts of 1001 tokens of 8 heads of 64 in fp32:
// 17 us.  What a thread holds allows two blocks a compute unit,
// whose waves wait in 78 of 100 cycles.
template <typename Tag, int DK, int DV>
__global__ __launch_bounds__(kNT) void append_kernel(Kv8 c, Kv8Append a, int nblk, int kv_groups, int q_groups, int update) {
  using raw = typename Tag::raw;
  constexpr int kSide = DK >= 96 ? 1 : 128 / DK, kThreads = kNT / kSide, kWaves = kThreads / kWave;  // of one head
  constexpr int NU = DK / 16, kRows = kThreads / NU, kPasses = (kBlk + kRows - 1) / kRows;
  constexpr int kItems = 2 * DV, kTurns = (kItems + kThreads - 1) / kThreads;  // of V: 16 words by DV / 8 dimensions' eights
  __shared__ uint32_t tops[2][2][4];
  const int64_t S = c.slots();
  const uint32_t blocks = static_cast<uint32_t>(c.B) * nblk;
  const int grp = blockIdx.x / blocks;  // all of K and V first: they take longest
  const uint32_t rest = blockIdx.x % blocks;
  const int side = threadIdx.x / kThreads, tid = threadIdx.x % kThreads;
  const int64_t b = rest / nblk;
  const Span s = span_of(c, a, b);
  const int64_t blk = (s.have >> 6) + rest % nblk, first = blk * kBlk;
  // the call's tokens on this block: all, and those that are stored
  const int lo = static_cast<int>(max(s.have - first, int64_t{0}));
  const int all = static_cast<int>(min(s.have + a.T - first, int64_t{kBlk}));
  const int64_t row0 = b * a.T - s.have + first;  // the call's row of the block's token 0
  const bool pairs = a.pairs != 0;

  const int u = tid % NU, r0 = tid / NU;
  const Unit un = unit_of(u, DK, a.R, pairs);
  Angles ang[kPasses];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int t = r0 + p * kRows;
    if (r0 < kRows && t >= lo && t < all) load_angles(a, un, min(first + t, S - 1), ang[p]);
  }

  const int h0 = grp < kv_groups ? c.HKV * grp / kv_groups : 0, h1 = grp < kv_groups ? c.HKV * (grp + 1) / kv_groups : 0;
  for (int hh = h0, turn_no = 0; hh < h1; hh += kSide, ++turn_no) {
    const int h = min(hh + side, h1 - 1);
    const bool mine = hh + side < h1;  // the last head's threads may have neighbours without one
    const int64_t at = first < s.end ? kv8_block(c, b, blk, h) : -1;
    const int hi = at >= 0 ? static_cast<int>(min(s.end - first, int64_t{kBlk})) : lo;
    uint8_t* const codes = c.codes + at * c.block_bytes();
    uint8_t* const scale_at = c.scales + at * 2;
    uint32_t top_k = 0, top_v = 0, old_k = 0, old_v = 0;
    float k0[kPasses][8], k1[kPasses][8], v[kTurns][4][8];
    const raw* const ksrc = static_cast<const raw*>(a.K) + row0 * a.ldk + static_cast<int64_t>(h) * DK;
    const raw* const vsrc = static_cast<const raw*>(a.V) + row0 * a.ldv + static_cast<int64_t>(h) * DV;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int t = r0 + p * kRows;
      if (!mine || r0 >= kRows || t < lo || t >= (a.K_out ? all : hi)) continue;
      load_cvt<Tag, 8>(ksrc + t * a.ldk + un.lo, k0[p]);
      load_cvt<Tag, 8>(ksrc + t * a.ldk + un.hi, k1[p]);
    }
#pragma unroll
    for (int p = 0; p < kTurns; ++p) {
      const int i = tid + p * kThreads, d = (i >> 6) * 32 + (i & 3) * 8, t = word_token((i >> 2) & 15);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int x = 0; x < 8; ++x) v[p][e][x] = 0.0f;
        if (mine && i < kItems && t + e >= lo && t + e < hi) load_cvt<Tag, 8>(vsrc + (t + e) * a.ldv + d, v[p][e]);
      }
    }
    if (lo > 0 && lo < hi) {
      old_k = scale_at[0];
      old_v = scale_at[1];
    }
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int t = r0 + p * kRows;
      if (!mine || r0 >= kRows || t < lo || t >= (a.K_out ? all : hi)) continue;
      turn(k0[p], k1[p], ang[p], un, pairs);
      if (t < hi) {
#pragma unroll
        for (int i = 0; i < 8; ++i) top_k = max(top_k, max(finite_bits(k0[p][i]), finite_bits(k1[p][i])));
      }
      if (a.K_out) {
        raw* to = static_cast<raw*>(a.K_out) + ((row0 + t) * c.HKV + h) * DK;
        if (first + t >= S) {
          make_nan(k0[p]);
          make_nan(k1[p]);
        }
        store8<Tag>(to + un.lo, k0[p]);
        store8<Tag>(to + un.hi, k1[p]);
      }
    }
    if (lo >= hi) continue;  // the same for the whole block
#pragma unroll
    for (int p = 0; p < kTurns; ++p)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < 8; ++i) top_v = max(top_v, finite_bits(v[p][e][i]));
    top_k = wave_max_bits(top_k);
    top_v = wave_max_bits(top_v);
    uint32_t(&top)[2][4] = tops[turn_no & 1];
    if ((threadIdx.x & 63) == 0) {
      top[0][threadIdx.x >> 6] = top_k;
      top[1][threadIdx.x >> 6] = top_v;
    }
    __syncthreads();  // the old scales have been read; the next head writes the other tops
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      top_k = max(top_k, top[0][side * kWaves + w]);
      top_v = max(top_v, top[1][side * kWaves + w]);
    }
    if (!mine) continue;
    const uint32_t new_k = max(old_k, kv8_scale(top_k)), new_v = max(old_v, kv8_scale(top_v));
    if (tid == 0) *reinterpret_cast<uint16_t*>(scale_at) = static_cast<uint16_t>(new_k | new_v << 8);
    // Held tokens whose block's scale grows are rounded again, to the new one.
    if (lo > 0 && new_k > old_k) {
      const float f = fall_of(old_k, new_k);
      for (int i = tid; i < lo * DK / 4; i += kThreads) {
        uint32_t* w = reinterpret_cast<uint32_t*>(codes) + i;
        *w = rescale4(*w, f);
      }
    }
    {
      const float f = kv8_inverse(new_k);
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int t = r0 + p * kRows;
        if (r0 >= kRows || t < lo || t >= hi) continue;
        *reinterpret_cast<uint2*>(codes + t * DK + un.lo) = encode8(k0[p], f);
        *reinterpret_cast<uint2*>(codes + t * DK + un.hi) = encode8(k1[p], f);
      }
    }
    const float f = kv8_inverse(new_v), fall = fall_of(old_v, new_v);
    const bool grows = lo > 0 && new_v > old_v;
#pragma unroll
    for (int p = 0; p < kTurns; ++p) {
      const int i = tid + p * kThreads, d = (i >> 6) * 32 + (i & 3) * 8, w = (i >> 2) & 15, t = word_token(w);
      if (i >= kItems || t >= hi || (t + 4 <= lo && !grows)) continue;
      uint2 q[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e] = encode8(v[p][e], f);
      uint32_t* const to = reinterpret_cast<uint32_t*>(codes + kBlk * DK + d * kBlk) + w;
      uint32_t out[8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // 4 tokens by 4 dimensions change places
        const uint32_t q0 = half ? q[0].y : q[0].x, q1 = half ? q[1].y : q[1].x, q2 = half ? q[2].y : q[2].x, q3 = half ? q[3].y : q[3].x;
        const uint32_t a01 = __builtin_amdgcn_perm(q1, q0, 0x05010400u), a23 = __builtin_amdgcn_perm(q3, q2, 0x05010400u);
        const uint32_t b01 = __builtin_amdgcn_perm(q1, q0, 0x07030602u), b23 = __builtin_amdgcn_perm(q3, q2, 0x07030602u);
        out[4 * half] = __builtin_amdgcn_perm(a23, a01, 0x05040100u);
        out[4 * half + 1] = __builtin_amdgcn_perm(a23, a01, 0x07060302u);
        out[4 * half + 2] = __builtin_amdgcn_perm(b23, b01, 0x05040100u);
        out[4 * half + 3] = __builtin_amdgcn_perm(b23, b01, 0x07060302u);
      }
      if (t < lo || t + 4 > hi) {  // some bytes are others'
        uint32_t held = 0, fresh = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          held |= t + e < lo ? 0xffu << (8 * e) : 0u;
          fresh |= t + e >= lo && t + e < hi ? 0xffu << (8 * e) : 0u;
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const uint32_t was = to[x * (kBlk / 4)];
          const uint32_t kept = grows ? rescale4(was, fall) : was;
          out[x] = (out[x] & fresh) | (kept & held) | (was & ~(held | fresh));
        }
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) to[x * (kBlk / 4)] = out[x];
    }
  }

  if (grp >= kv_groups) {
    const int q0 = a.HQ * (grp - kv_groups) / q_groups, q1 = a.HQ * (grp - kv_groups + 1) / q_groups;
    const raw* __restrict__ const from = static_cast<const raw*>(a.Q);
    raw* __restrict__ const to = static_cast<raw*>(a.Q_out);
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int t = r0 + p * kRows;
      if (r0 >= kRows || t < lo || t >= all) continue;
      const raw* src = from + (row0 + t) * a.ldq;
      raw* dst = to + (row0 + t) * a.HQ * DK;
#pragma unroll 4
      for (int h = q0 + side; h < q1; h += kSide) {
        float x[8], y[8];
        load_cvt<Tag, 8>(src + static_cast<int64_t>(h) * DK + un.lo, x);
        load_cvt<Tag, 8>(src + static_cast<int64_t>(h) * DK + un.hi, y);
        turn(x, y, ang[p], un, pairs);
        if (first + t >= S) {
          make_nan(x);
          make_nan(y);
        }
        store8<Tag>(dst + static_cast<int64_t>(h) * DK + un.lo, x);
        store8<Tag>(dst + static_cast<int64_t>(h) * DK + un.hi, y);
      }
    }
  }
  if (update && grp == 0 && rest % nblk == 0) update_counts(c, s, b);
}

// Few tokens (a decode step): a block of threads takes a sequence whole, so that one launch also
// changes its length.  A wave takes the K or the V of one head, a unit of one token a
// lane, then units of the queries; what does not depend on the position is loaded before the
// position is known.  Bound by latency, that of the chain length, page, scale, codes: 32 sequences
// of 32 and 8 heads of 128 in bf16, 11 MB, take 6.7 us in a graph (8.1 each alone) where no block's
// scale grows.  Where one does, its held codes move a word a lane a trip, each waited for: with
// random tokens from a block's slot 8 to 55 some head's scale grows in nearly every step, which
// then takes 15.8 on average, and 26.6 where all heads' do (one sequence: 6.0, 7.0, 15.1).
constexpr int kFew = 4;  // tokens, by 16 units: a wave
template <typename Tag, int DK, int DV>
__global__ __launch_bounds__(1024) void append_few_kernel(Kv8 c, Kv8Append a) {
  using raw = typename Tag::raw;
  constexpr int NU = DK / 16;
  const int64_t b = blockIdx.x, S = c.slots();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id(), waves = blockDim.x >> 6;
  const int T = static_cast<int>(a.T), items = 2 * c.HKV, q_items = a.Q_out ? T * a.HQ * NU : 0;
  const bool pairs = a.pairs != 0;
  const int u = lane % 16, tok = lane / 16;
  float x[8], y[8], qx[8], qy[8];
  auto load_item = [&](int item) __attribute__((always_inline)) {
    const int h = item >> 1, is_v = item & 1;
    if (item >= items || tok >= T || 16 * u >= (is_v ? DV : DK)) return;
    const Unit un = is_v ? unit_of(u, DV, 0, false) : unit_of(u, DK, a.R, pairs);
    const raw* src = is_v ? static_cast<const raw*>(a.V) + (b * T + tok) * a.ldv + static_cast<int64_t>(h) * DV
                          : static_cast<const raw*>(a.K) + (b * T + tok) * a.ldk + static_cast<int64_t>(h) * DK;
    load_cvt<Tag, 8>(src + un.lo, x);
    load_cvt<Tag, 8>(src + un.hi, y);
  };
  auto load_query = [&](int i) __attribute__((always_inline)) {
    if (i >= q_items) return;
    const int row = i / NU;
    const Unit un = unit_of(i % NU, DK, a.R, pairs);
    const raw* src = static_cast<const raw*>(a.Q) + (b * T + row / a.HQ) * a.ldq + static_cast<int64_t>(row % a.HQ) * DK;
    load_cvt<Tag, 8>(src + un.lo, qx);
    load_cvt<Tag, 8>(src + un.hi, qy);
  };
  load_item(wave);
  load_query(threadIdx.x);
  const Span s = span_of(c, a, b);
  const int64_t blk0 = s.have / kBlk;
  // the first item's place and scales, ahead of the queries
  const int64_t at0 = s.have < s.end && wave < items ? kv8_block(c, b, blk0, wave >> 1) : -1;
  const uint32_t old0 = at0 >= 0 ? c.scales[at0 * 2 + (wave & 1)] : 0u;

  for (int i = threadIdx.x; i < q_items; i += blockDim.x) {
    if (i != static_cast<int>(threadIdx.x)) load_query(i);
    const int row = i / NU, t = row / a.HQ;
    const Unit un = unit_of(i % NU, DK, a.R, pairs);
    Angles g;
    load_angles(a, un, min(s.have + t, S - 1), g);
    turn(qx, qy, g, un, pairs);
    if (s.have + t >= S) {
      make_nan(qx);
      make_nan(qy);
    }
    raw* to = static_cast<raw*>(a.Q_out) + (b * T * a.HQ + row) * DK;
    store8<Tag>(to + un.lo, qx);
    store8<Tag>(to + un.hi, qy);
  }

  const int nblk = static_cast<int>((s.have + T - 1) / kBlk - blk0) + 1;
  for (int item = wave; item < items; item += waves) {
    if (item != wave) load_item(item);
    const int h = item >> 1, is_v = item & 1;
    const bool has = tok < T && 16 * u < (is_v ? DV : DK);
    const Unit un = is_v ? unit_of(u, DV, 0, false) : unit_of(u, DK, a.R, pairs);
    uint32_t top = 0;
    if (has) {
      if (!is_v) {
        Angles g;
        load_angles(a, un, min(s.have + tok, S - 1), g);
        turn(x, y, g, un, pairs);
        if (a.K_out) {
          if (s.have + tok >= S) {
            make_nan(x);
            make_nan(y);
          }
          raw* to = static_cast<raw*>(a.K_out) + ((b * T + tok) * c.HKV + h) * DK;
          store8<Tag>(to + un.lo, x);
          store8<Tag>(to + un.hi, y);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, max(finite_bits(x[i]), finite_bits(y[i])));
    }
    for (int n = 0; n < nblk; ++n) {  // the one or two blocks that the tokens lie on
      const int64_t first = (blk0 + n) * kBlk;
      if (first >= s.end) break;
      const bool known = item == wave && n == 0;
      const int64_t at = known ? at0 : kv8_block(c, b, blk0 + n, h);
      const int lo = static_cast<int>(max(s.have - first, int64_t{0}));
      const int hi = static_cast<int>(min(s.end - first, int64_t{kBlk}));
      if (at < 0 || lo >= hi) continue;  // the same for the whole wave
      uint8_t* const codes = c.codes + at * c.block_bytes() + (is_v ? kBlk * DK : 0);
      uint8_t* const scale_at = c.scales + at * 2 + is_v;
      const int t = static_cast<int>(s.have + tok - first);
      const bool mine = has && t >= lo && t < hi;
      const uint32_t old = lo == 0 ? 0u : known ? old0 : *scale_at;
      const uint32_t now = max(old, kv8_scale(wave_max_bits(mine ? top : 0u)));
      if (lane == 0) *scale_at = static_cast<uint8_t>(now);
      if (lo > 0 && now > old) {  // the block's held tokens, 4 codes a lane
        const float f = fall_of(old, now);
        for (int i = lane; i < (is_v ? DV * kBlk : lo * DK) / 4; i += kWave) {
          const int first_t = is_v ? word_token(i & 15) : 0;
          if (is_v && first_t >= lo) continue;
          uint32_t* w = reinterpret_cast<uint32_t*>(codes) + i;
          const uint32_t was = *w, keep = is_v && lo - first_t < 4 ? (1u << (8 * (lo - first_t))) - 1u : 0xffffffffu;
          *w = (rescale4(was, f) & keep) | (was & ~keep);
        }
        __threadfence();  // before bytes go in beside them
      }
      if (!mine) continue;
      const uint2 p = encode8(x, kv8_inverse(now)), q = encode8(y, kv8_inverse(now));
      if (!is_v) {
        *reinterpret_cast<uint2*>(codes + t * DK + un.lo) = p;
        *reinterpret_cast<uint2*>(codes + t * DK + un.hi) = q;
      } else {
        const uint32_t w[4] = {p.x, p.y, q.x, q.y};
        uint8_t* to = codes + v_place(t);
#pragma unroll
        for (int i = 0; i < 16; ++i) to[((i < 8 ? un.lo : un.hi) + (i & 7)) * kBlk] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
      }
    }
  }
  __syncthreads();  // every wave has read the length
  if (threadIdx.x == 0) {
    int32_t lost = static_cast<int32_t>(s.many - (s.end - s.have));
    for (int n = 0; n < nblk && (blk0 + n) * kBlk < s.end; ++n)
      if (kv8_block(c, b, blk0 + n, 0) < 0)
        lost += static_cast<int32_t>(min(s.end, (blk0 + n + 1) * kBlk) - max(s.have, (blk0 + n) * kBlk));
    c.length[b] = static_cast<int32_t>(s.end);
    if (lost) c.lost[b] += lost;
  }
}

// The counters of an append whose blocks read them.
__global__ __launch_bounds__(kNT) void append_counts_kernel(Kv8 c, Kv8Append a) {
  update_counts(c, span_of(c, a, blockIdx.x), blockIdx.x);
}

// Slots back as values; zeros for a slot that holds nothing.  A block of threads takes 64
// entries of a list, one head.  Where they are one block's slots in order (as
// the first N slots are, and runs that begin with a block), a thread takes 4 tokens by 8
// dimensions of V from words of 4 tokens; else it gathers bytes, which lie 64 apart in V, as the
// attention wants them.  Bound by memory: 2 x 16384 slots of 8 heads of 128 as bf16, 201 MB, take
// 46 us, 4.4 TB/s; gathered, 143.
__device__ __forceinline__ void decode8(uint32_t w0, uint32_t w1, float f, float (&x)[8]) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w0, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w0, true);
  const f32x2 c = __builtin_amdgcn_cvt_pk_f32_fp8(w1, false), d = __builtin_amdgcn_cvt_pk_f32_fp8(w1, true);
  x[0] = a[0] * f; x[1] = a[1] * f; x[2] = b[0] * f; x[3] = b[1] * f;
  x[4] = c[0] * f; x[5] = c[1] * f; x[6] = d[0] * f; x[7] = d[1] * f;
}

template <typename Tag>
__global__ __launch_bounds__(kNT) void rows_kernel(Kv8 c, const int32_t* __restrict__ slots, int64_t N, uint32_t lists,
                                                   typename Tag::raw* __restrict__ K, typename Tag::raw* __restrict__ V) {
  __shared__ int32_t slot_of[kBlk];
  __shared__ bool in_order;
  const int h = blockIdx.x % c.HKV;
  const uint32_t rest = blockIdx.x / c.HKV;
  const int64_t b = rest / lists, n0 = static_cast<int64_t>(rest % lists) * kBlk;
  const int many = static_cast<int>(min(N - n0, int64_t{kBlk}));
  const int32_t length = kv8_length(c, b);
  if (threadIdx.x < kBlk) {  // the first wave
    const int i = min(static_cast<int>(threadIdx.x), many - 1);
    const int32_t mine = slots ? slots[b * N + n0 + i] : static_cast<int32_t>(n0 + i);
    slot_of[threadIdx.x] = mine;
    const bool runs = ballot(mine != __builtin_amdgcn_readfirstlane(mine) + i) == 0;
    if (threadIdx.x == 0) in_order = runs;
  }
  __syncthreads();
  const int32_t first = slot_of[0];
  const bool run = in_order && first >= 0 && first < length && first % kBlk == 0;
  const int kc = c.DK / 8, vc = c.DV / 8;
  if (run) {
    const int64_t at = kv8_block(c, b, first >> 6, h);
    const uint8_t* codes = c.codes + at * c.block_bytes();
    const int held = at < 0 ? 0 : min(many, length - first);  // entries that hold something
    const float fk = at < 0 ? 0.0f : __uint_as_float(static_cast<uint32_t>(c.scales[at * 2]) << 23);
    const float fv = at < 0 ? 0.0f : __uint_as_float(static_cast<uint32_t>(c.scales[at * 2 + 1]) << 23);
    for (int i = threadIdx.x; i < many * kc; i += kNT) {
      const int t = i / kc, d = i % kc * 8;
      float x[8] = {};
      if (t < held) {
        const uint2 w = *reinterpret_cast<const uint2*>(codes + t * c.DK + d);
        decode8(w.x, w.y, fk, x);
      }
      store8<Tag>(K + ((b * N + n0 + t) * c.HKV + h) * c.DK + d, x);
    }
    for (int i = threadIdx.x; i < 16 * vc; i += kNT) {
      const int d = (i >> 6) * 32 + (i & 3) * 8, w = (i >> 2) & 15, t = word_token(w);
      if (t >= many) continue;
      uint32_t q[8] = {};
      if (t < held) {
        const uint32_t* from = reinterpret_cast<const uint32_t*>(codes + kBlk * c.DK + d * kBlk) + w;
#pragma unroll
        for (int x = 0; x < 8; ++x) q[x] = from[x * (kBlk / 4)];
      }
      uint32_t o[2][4];  // 4 dimensions by 4 tokens change places
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t a01 = __builtin_amdgcn_perm(q[4 * half + 1], q[4 * half], 0x05010400u), a23 = __builtin_amdgcn_perm(q[4 * half + 3], q[4 * half + 2], 0x05010400u);
        const uint32_t b01 = __builtin_amdgcn_perm(q[4 * half + 1], q[4 * half], 0x07030602u), b23 = __builtin_amdgcn_perm(q[4 * half + 3], q[4 * half + 2], 0x07030602u);
        o[half][0] = __builtin_amdgcn_perm(a23, a01, 0x05040100u);
        o[half][1] = __builtin_amdgcn_perm(a23, a01, 0x07060302u);
        o[half][2] = __builtin_amdgcn_perm(b23, b01, 0x05040100u);
        o[half][3] = __builtin_amdgcn_perm(b23, b01, 0x07060302u);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (t + e >= many) break;
        float x[8] = {};
        if (t + e < held) decode8(o[0][e], o[1][e], fv, x);
        store8<Tag>(V + ((b * N + n0 + t + e) * c.HKV + h) * c.DV + d, x);
      }
    }
    return;
  }
  for (int i = threadIdx.x; i < many * (kc + vc); i += kNT) {
    const int t = i / (kc + vc), ch = i % (kc + vc);
    const int32_t slot = slot_of[t];
    const int64_t row = (b * N + n0 + t) * c.HKV + h;
    float x[8] = {};
    const int64_t at = slot >= 0 && slot < length ? kv8_block(c, b, slot >> 6, h) : -1;
    if (at >= 0) {
      const uint8_t* codes = c.codes + at * c.block_bytes();
      const float f = __uint_as_float(static_cast<uint32_t>(c.scales[at * 2 + (ch < kc ? 0 : 1)]) << 23);
      if (ch < kc) {
        const uint2 w = *reinterpret_cast<const uint2*>(codes + (slot & 63) * c.DK + ch * 8);
        decode8(w.x, w.y, f, x);
      } else {
        const uint8_t* from = codes + kBlk * c.DK + (ch - kc) * 8 * kBlk + v_place(slot & 63);
        uint32_t w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          w[j] = from[(4 * j) * kBlk] | from[(4 * j + 1) * kBlk] << 8 | from[(4 * j + 2) * kBlk] << 16 |
                 static_cast<uint32_t>(from[(4 * j + 3) * kBlk]) << 24;
        decode8(w[0], w[1], f, x);
      }
    }
    if (ch < kc) store8<Tag>(K + row * c.DK + ch * 8, x);
    else store8<Tag>(V + row * c.DV + (ch - kc) * 8, x);
  }
}

template <typename Tag, int DK, int DV>
hipError_t append_dims(const Kv8& c, const Kv8Append& a, hipStream_t stream) {
  if (a.T <= kFew) {
    const int64_t items = 2 * c.HKV + (a.Q_out ? a.T * a.HQ * (DK / 16) / kWave : 0);
    const int waves = items >= 16 ? 16 : items >= 8 ? 8 : 4;
    append_few_kernel<Tag, DK, DV><<<static_cast<uint32_t>(c.B), waves * kWave, 0, stream>>>(c, a);
    return hipGetLastError();
  }
  const int nblk = static_cast<int>((a.T + kBlk - 2) / kBlk + 1);
  // The angles are loaded once for the heads of a group, so a group is as large as leaves two blocks a
  // compute unit for K and V and as many for the queries: 190 us for 2 x 16384 tokens of 32 and 8
  // heads of 128; smaller groups took 196 (4) to 219 (8).  Two run at once of up to 128 dimensions and of
  // 192 with V of 128, past that one.  us for one block / two / four a unit:
  //   32 and 8 heads of 128: 2000 tokens 12.9 / 13.8 / 14.4, 8192 36 / 42 / 48, 16384 91 / 105 / 104
  //   8 and 8: 4096 of 128 18.7 / 17.1 / 17.1, 8 x 1001 of 64 in fp32 22.0 / 20.1 / 20.1
  //   no queries, 8 heads, 3000 tokens: of 128 14.6 / 10.1 / 10.1, of 256 34.6 / 25.8 / 25.6
  //   16 and 4 heads: 2 x 8192 of 192 126 / 130 / 141, 16384 of 256 133 / 138 / 155
  // One is better by up to a seventh where queries outnumber keys, two by up to a third where not.
  const int64_t want = 2 * int64_t{device_cus() > 0 ? device_cus() : 256}, blocks = c.B * nblk;
  auto groups_of = [&](int64_t heads) { return static_cast<int>(std::min(heads, (want + blocks - 1) / blocks)); };
  constexpr int kSide = DK >= 96 ? 1 : 128 / DK;
  const int kv = groups_of((c.HKV + kSide - 1) / kSide), q = a.Q_out ? groups_of((a.HQ + kSide - 1) / kSide) : 0;
  // where the blocks read the length (to find their place, or as the count), a launch of its own changes it
  const bool update = a.start != nullptr && a.count != c.length;
  append_kernel<Tag, DK, DV><<<static_cast<uint32_t>(blocks * (kv + q)), kNT, 0, stream>>>(c, a, nblk, kv, q, update);
  if (!update) append_counts_kernel<<<static_cast<uint32_t>(c.B), kNT, 0, stream>>>(c, a);
  return hipGetLastError();
}

template <typename Tag>
hipError_t append_type(const Kv8& c, const Kv8Append& a, hipStream_t stream) {
  if (c.DK != c.DV) return append_dims<Tag, 192, 128>(c, a, stream);
  switch (c.DK) {
    case 32: return append_dims<Tag, 32, 32>(c, a, stream);
    case 64: return append_dims<Tag, 64, 64>(c, a, stream);
    case 96: return append_dims<Tag, 96, 96>(c, a, stream);
    case 128: return append_dims<Tag, 128, 128>(c, a, stream);
    case 192: return append_dims<Tag, 192, 192>(c, a, stream);
    default: return append_dims<Tag, 256, 256>(c, a, stream);
  }
}

}  // namespace

hipError_t launch_kv8_append(const Kv8& c, const Kv8Append& a, int dtype, hipStream_t stream) {
  if (c.B == 0) return hipSuccess;
  Kv8Append x = a;
  if (x.start == c.length) x.start = nullptr;  // the counters that the call changes
  if (x.T == 0) {
    if (x.start) append_counts_kernel<<<static_cast<uint32_t>(c.B), kNT, 0, stream>>>(c, x);
    return hipGetLastError();
  }
  return dtype == 0   ? append_type<F32>(c, x, stream)
         : dtype == 1 ? append_type<BF16>(c, x, stream)
                      : append_type<F16>(c, x, stream);
}

hipError_t launch_kv8_rows(const Kv8& c, const int32_t* slots, int64_t N, int dtype, void* K, void* V,
                           hipStream_t stream) {
  if (c.B == 0 || N == 0) return hipSuccess;
  const uint32_t lists = static_cast<uint32_t>((N + kBlk - 1) / kBlk);
  const uint32_t grid = static_cast<uint32_t>(c.B * lists * c.HKV);
  if (dtype == 0) rows_kernel<F32><<<grid, kNT, 0, stream>>>(c, slots, N, lists, static_cast<float*>(K), static_cast<float*>(V));
  else if (dtype == 1) rows_kernel<BF16><<<grid, kNT, 0, stream>>>(c, slots, N, lists, static_cast<uint16_t*>(K), static_cast<uint16_t*>(V));
  else rows_kernel<F16><<<grid, kNT, 0, stream>>>(c, slots, N, lists, static_cast<uint16_t*>(K), static_cast<uint16_t*>(V));
  return hipGetLastError();
}

}  // namespace dsa
