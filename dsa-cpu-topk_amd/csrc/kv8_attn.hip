// kv8_attn.hip -- attention of each sequence's last tokens over the paged 8-bit
// cache (gfx950).
//
//   O[b,t,h,:] = sum_s p_s V[b,s,h/G,:],  p = softmax_s(<Q[b,t,h], K[b,s,h/G]> scale)
// over the slots s that token t sees: s <= its own, and with a window s > its own -
// window or s < sinks.
//
// A wave takes 64 slots of one K/V head and RT tiles of 16 rows (the group's heads of the
// tokens, token by token) at a time, on 16x16x32 f16 products:
//   S^T = K . Q^T    A = K's codes, which f16 holds exactly; B = Q
//   O^T = V^T . P^T  A = V's codes as they lie in the cache; B = P straight from S^T's
//                    registers (lane group g holds tokens 16j + 4g + i of each row)
// The block's scales are powers of two: K's goes into the factor of the logits, V's is the
// unit in which a row's sums are held (a block of another unit is added apart, exactly).
// Sums are divided by those of p before the unit comes in, for each wave and each split, and
// joined as shares that add up to 1: a mean of numbers that fp32 holds stays one.
// So no value of the cache is rounded.  Rows of Q are scaled by a power of two into f16's
// range and enter as one f16 piece (16-bit types) or two (fp32, 23 bits); p likewise.
//
// Few rows or short rows of K (!SHARED): each of a block's four waves takes blocks of its own in turn, its
// operands straight into registers; K of the next block is on its way while p and V are
// multiplied, V while the logits are formed, the page id two turns ahead.  Bound by memory: 16
// caches of up to 32768 slots, 32 heads on 8 of 128, 834 MB, take 152 us, 5.5 TB/s (a large
// array is read at 6.35).  Operands by way of LDS, as below, or eight waves a block were slower.
//
// Many long rows, or few slots (SHARED): the waves take different rows of the same blocks.  Codes go to LDS by
// DMA, whole rows at a time and in two buffers (lanes next to each other fetch bytes next to
// each other: a lane's own operand is 16 bytes of a row of its own, which costs the L1 64
// accesses an instruction where this takes 16), rows' 16-byte chunks swizzled so that no two
// lanes meet on a bank when they are read as operands.  Bound by the vector instructions that widen
// the codes and weigh the logits, which 32 rows a wave share where there are enough (DK = 128 of
// 16-bit types: more have no registers): 4 x 48 tokens of 16 heads on one of 128 over 8191 slots,
// 10.5 GFLOP, take 30 us; 60 with waves on slots of their own.
#include <algorithm>

#include "dsa_launch.h"
#include "kv8.h"
#include "tile_common.h"

namespace dsa {
namespace {

struct AttnArgs {
  Kv8 c;
  const void* Q;
  const int32_t* count;
  int Tq, HQ, G;
  int row_tiles, splits;
  uint32_t few_chunks;  // sequences, K/V heads and splits where they are few, else 0
  int64_t n;       // slots that count
  int64_t window;  // 0: all
  int64_t sinks;
  float scale_log2;
  void* out;
  float* part;  // [B*Tq*HQ][splits][DV], each split's own result
  float2* ml;   // [B*Tq*HQ][splits]: maximum (log2) and sum
};

constexpr int kWaves = kNT / kWave;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// p is held as 2^(kUp + logit - maximum): what is small beside the largest then stays
// a normal f16 down to 2^-(14 + kUp).  The maximum moves when a logit passes it by
// kSlack, so p stays below 2^15.
constexpr float kUp = 10.0f, kSlack = 5.0f;

__device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float mul(float x, float y) {  // rounded by itself
#pragma clang fp contract(off)
  return x * y;
}
// Four codes as four f16.
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
  hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
}
__device__ __forceinline__ u32x4 widen8(uint32_t w0, uint32_t w1) {
  u32x4 x;
  uint32_t a, b, c, d;
  widen(w0, a, b);
  widen(w1, c, d);
  x[0] = a; x[1] = b; x[2] = c; x[3] = d;
  return x;
}
// Bit 7 of each byte that is e4m3's NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

template <typename Tag>
__device__ __forceinline__ void store4(typename Tag::raw* to, f32x4 y) {
  if constexpr (Tag::kBytes == 4) {
    *reinterpret_cast<f32x4*>(to) = y;
  } else if constexpr (__is_same(Tag, BF16)) {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<bf16x4*>(to) = __builtin_convertvector(y, bf16x4);
  } else {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<f16x4*>(to) = __builtin_convertvector(y, f16x4);
  }
}

// What token t of sequence b sees: slots [low, end) and those below sinks (and end).
struct Seen {
  int32_t low, end;
};
__device__ __forceinline__ Seen seen_by(const AttnArgs& a, int32_t len, int32_t many, int t) {
  Seen s;
  const int32_t own = len - many + t + 1;
  s.end = t < many ? max(0, min(own, static_cast<int32_t>(a.n))) : 0;
  s.low = a.window > 0 ? static_cast<int32_t>(max(int64_t{0}, own - a.window)) : 0;
  return s;
}

// Where the 16-byte chunk `c` of row r (of NC chunks) lies in LDS, and back: 16 rows' chunks
// of one number take all banks.
template <int NC>
__device__ __forceinline__ int chunk_at(int r, int c) {
  if constexpr ((NC & (NC - 1)) == 0) return c ^ ((r & 15) / (16 / NC));
  else return (c + (r & 15) / (NC == 12 ? 4 : 8)) % NC;
}
template <int NC>
__device__ __forceinline__ int chunk_of(int r, int at) {
  if constexpr ((NC & (NC - 1)) == 0) return at ^ ((r & 15) / (16 / NC));
  else return (at + NC - (r & 15) / (NC == 12 ? 4 : 8)) % NC;
}

template <typename Tag, int DK, int DV, int RT, bool SHARED>
__global__ __launch_bounds__(kNT, DK <= 128 || (SHARED && Tag::kBytes == 2) ? 2 : 1) void attn_kernel(AttnArgs a) {
  using raw = typename Tag::raw;
  constexpr int NP = Tag::kBytes == 4 ? 2 : 1;          // f16 pieces of Q and of p
  constexpr int NJ = DK / 64, HALF = DK % 64 != 0;      // 16-byte runs of a K row a lane, and 8-byte ones
  constexpr int NKS = 2 * NJ + HALF, NDT = DV / 16, NCK = DK / 16;
  constexpr int WR = SHARED ? kWaves : 1, WT = kWaves / WR;  // waves on different rows; on different slots
  constexpr int kTile = 16 * RT * WR;                        // rows of a block
  constexpr int kK = kBlk * DK, kV = kBlk * DV;              // bytes of a block's K and V
  // as objects of their own: a DMA into one is no write to another
  constexpr int kHold = SHARED ? 1 : 0;
  __shared__ __align__(16) uint8_t k_lds[kHold * kK + 16], v_lds[kHold * kV + 16], k2_lds[kHold * kK + 16], v2_lds[kHold * kV + 16];
  __shared__ __align__(16) float sum_o[SHARED ? 4 : WT * kTile * DV];
  __shared__ float sum_m[WT][kTile], sum_l[WT][kTile];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id();
  const int g = lane >> 4, col = lane & 15, wr = SHARED ? wave : 0, wt = SHARED ? 0 : wave;
  // Blocks of one chunk of slots and their row tiles go to one XCD (block i starts on XCD i % 8);
  // where a few chunks would not fill them alike, row tiles go round over all of them.
  const uint32_t few = a.few_chunks;
  const uint32_t chunk = few ? blockIdx.x % few : blockIdx.x % 8 + blockIdx.x / (8 * a.row_tiles) * 8;
  const uint32_t rt = few ? blockIdx.x / few : blockIdx.x / 8 % a.row_tiles;
  const int split = chunk % a.splits;
  const uint32_t bh = chunk / a.splits;
  const int h = bh % a.c.HKV;
  const int64_t b = bh / a.c.HKV;
  if (b >= a.c.B) return;

  // Q: lane holds row `col`, dims 64j + 16g .. +15 (the products' k-slots in the order of K's
  // runs).  Asked for first, made into pieces when K and V are on their way.
  constexpr int QW = Tag::kBytes / 2;  // 16 bytes of 8 elements
  u32x4 q_raw[RT][NKS][QW];
  const int rows = a.Tq * a.G;
  const int block_row = rt * kTile, block_rows = min(kTile, rows - block_row);
  const int first_row = block_row + wr * 16 * RT, last_row = min(first_row + 16 * RT, rows) - 1;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = min(first_row + 16 * r + col, rows - 1), t = row / a.G;
    const raw* src = static_cast<const raw*>(a.Q) + ((b * a.Tq + t) * a.HQ + h * a.G + row % a.G) * DK;
#pragma unroll
    for (int k = 0; k < NKS; ++k)
#pragma unroll
      for (int i = 0; i < QW; ++i)
        q_raw[r][k][i] = *reinterpret_cast<const u32x4*>(src + (k < 2 * NJ ? 64 * (k / 2) + 16 * g + 8 * (k % 2) : 64 * NJ + 8 * g) + 4 * i);
  }
  const int32_t len = kv8_length(a.c, b);
  const int32_t many = a.count ? max(0, min(a.count[b], a.Tq)) : a.Tq;
  const int32_t sinks = static_cast<int32_t>(a.sinks);  // at most the slots, 2^31 - 256
  // the blocks that any token of these rows sees: those of the first tokens, then near, near + 1, ...
  int32_t near = 0, nsink = 0, total = 0;
  {
    const int t0 = block_row / a.G, t1 = min((block_row + block_rows - 1) / a.G, many - 1);
    const Seen s0 = seen_by(a, len, many, t0), s1 = seen_by(a, len, many, t1);
    if (t1 >= t0 && s1.end > 0) {
      near = s0.low / kBlk;
      nsink = min((min(sinks, s1.end) + kBlk - 1) / kBlk, near);
      total = nsink + max(0, (s1.end + kBlk - 1) / kBlk - near);
    }
  }
  // of the wave's tokens that are any: the earliest and the latest
  const int t_lo = min(first_row, rows - 1) / a.G, t_hi = min(last_row / a.G, many - 1);
  const Seen lo = seen_by(a, len, many, t_lo), hi = seen_by(a, len, many, t_hi);
  const bool any_rows = first_row <= last_row && t_hi >= t_lo;

  u32x4 q[RT][NP][NKS];
  float factor[RT];
  Seen mine[RT];
  bool token[RT], odd_row[RT];
  auto split_q = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int t = min(first_row + 16 * r + col, rows - 1) / a.G;
      mine[r] = seen_by(a, len, many, t);
      token[r] = t < many;
      float x[NKS][8];
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < NKS; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (QW == 2) x[k][i] = __uint_as_float(q_raw[r][k][i >> 2][i & 3]);
          else x[k][i] = to_f32(Tag{}, static_cast<uint16_t>(i & 1 ? q_raw[r][k][0][i >> 1] >> 16 : q_raw[r][k][0][i >> 1] & 0xffffu));
          top = max(top, __float_as_uint(x[k][i]) & 0x7fffffffu);
        }
      top = max_xor32_u32(max_xor16_u32(top));
      odd_row[r] = top >= 0x7f800000u;  // every logit of such a row is Inf or NaN
      // the row's largest into [2^14, 2^15), with the scale's sign
      const int sh = odd_row[r] || top == 0 ? 0 : min(141 - static_cast<int>(top >> 23), 126);
      const float f = a.scale_log2 < 0.0f ? -pow2f(sh) : pow2f(sh);
      factor[r] = fabsf(a.scale_log2) * pow2f(-sh);
#pragma unroll
      for (int k = 0; k < NKS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = x[k][2 * i] * f, v = x[k][2 * i + 1] * f;
          if constexpr (NP == 2) {
            uint32_t hi16, lo16;
            split_pair(u, v, hi16, lo16);
            q[r][0][k][i] = hi16;
            q[r][1][k][i] = lo16;
          } else {
            q[r][0][k][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{u, v}), f16x2));
          }
        }
    }
  };

  float m[RT], l[RT];
  f32x4 o[RT][NDT];
  // V's scale byte in units of which a row's o is held, of a block in which the row weighs a
  // slot; 0: o is nothing yet.
  uint32_t unit[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.0f;
    unit[r] = 0;
#pragma unroll
    for (int d = 0; d < NDT; ++d) o[r][d] = f32x4{0, 0, 0, 0};
  }

  const int32_t step = a.splits * WT;
  const int32_t* const pages = a.c.pages + b * a.c.max_pages;
  auto block_of = [&](int32_t v) { return v < nsink ? v : near + v - nsink; };
  auto page_of = [&](int32_t v) { return pages[block_of(max(0, min(v, total - 1))) >> a.c.page_shift]; };  // of a block past the last: any
  // A block's place in the pool; where its page is none, it holds nothing: the pool's first
  // block stands in for the loads, and what it has there (its scale too) goes nowhere.
  auto place = [&](int32_t v, int32_t page, bool& held) __attribute__((always_inline)) {
    page = __builtin_amdgcn_readfirstlane(page);
    held = page >= 0 && page < a.c.NP;
    return held ? ((static_cast<int64_t>(page) * a.c.HKV + h) << a.c.page_shift) + (block_of(v) & ((1 << a.c.page_shift) - 1)) : int64_t{0};
  };
  auto scales_at = [&](int64_t at) { return static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(a.c.scales + at * 2)); };

  f32x4 st[RT][4];
  auto logits = [&](auto run, auto half) __attribute__((always_inline)) {  // 16 or 8 bytes of row 16j + col
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u32x4 x[NKS];
#pragma unroll
      for (int i = 0; i < NJ; ++i) {
        const u32x4 w = run(j, i);
        x[2 * i] = widen8(w[0], w[1]);
        x[2 * i + 1] = widen8(w[2], w[3]);
      }
      if (HALF) {
        const u32x2 w = half(j);
        x[NKS - 1] = widen8(w[0], w[1]);
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        st[r][j] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < NKS; ++k)
#pragma unroll
          for (int p2 = NP - 1; p2 >= 0; --p2) st[r][j] = mfma(x[k], q[r][p2][k], st[r][j]);
      }
    }
  };
  u32x4 p[RT][NP][2];
  uint32_t ok[RT];  // bit 4j + i: slot s0 + 16j + 4g + i is seen
  auto weights = [&](uint32_t sc, int32_t s0, bool inner) __attribute__((always_inline)) {
    const float ks = __uint_as_float((sc & 255u) << 23);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      // not below the least normal number: a masked -Inf times it stays one
      const float f = fmaxf(factor[r] * ks, 0x1p-126f);
      if (!inner) {
        ok[r] = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int32_t s = s0 + (e >> 2) * 16 + 4 * g + (e & 3);
          if (s < mine[r].end && (s >= mine[r].low || s < sinks)) ok[r] |= 1u << e;
          st[r][e >> 2][e & 3] = ok[r] >> e & 1u ? st[r][e >> 2][e & 3] : -INFINITY;
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, st[r][e >> 2][e & 3]);
      top = mul(max_xor32(max_xor16(top)), f);
      if (ballot(top > m[r] + kSlack)) {
        const float next = fmaxf(m[r], top);
        const float fall = m[r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[r] - next);
        m[r] = next;
        l[r] *= fall;
        // what has fallen to nothing has no unit either
        if (max_xor32_u32(max_xor16_u32(__float_as_uint(l[r]))) == 0) unit[r] = 0;
#pragma unroll
        for (int d = 0; d < NDT; ++d) o[r][d] *= fall;
      }
      const float ref = m[r] == -INFINITY ? 0.0f : m[r] - kUp;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          // (no fma: the maximum's product was rounded too, and far logits differ by more than exp2 takes)
          const float x = __builtin_amdgcn_exp2f(mul(st[r][j][i], f) - ref), y = __builtin_amdgcn_exp2f(mul(st[r][j][i + 1], f) - ref);
          const int e = 2 * (j & 1) + i / 2;
          if constexpr (NP == 2) {
            uint32_t hi16, lo16;
            split_pair(x, y, hi16, lo16);
            p[r][0][j >> 1][e] = hi16;
            p[r][1][j >> 1][e] = lo16;
            l[r] += x + y;
          } else {  // the sum takes p as the product does
            const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), f16x2));
            p[r][0][j >> 1][e] = w;
            l[r] = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), (f16x2{1, 1}), l[r], false);
          }
        }
    }
  };
  auto sums = [&](uint32_t sc, bool inner, auto read) __attribute__((always_inline)) {  // 16 bytes of dimension 16d + col
    // A NaN in V is for the rows that see its slot alone: where some do not, it goes
    // into their sums by hand and stays out of the product.
    bool fix = false;
    if (!inner) {
      uint32_t any = 0;
#pragma unroll
      for (int d = 0; d < NDT; ++d) {
        const u32x4 w = read(d);
        any |= nan_bytes(w[0]) | nan_bytes(w[1]) | nan_bytes(w[2]) | nan_bytes(w[3]);
      }
      fix = ballot(any != 0) != 0;
    }
    // A row in which none of the block's slots weighs anything (it sees none, or its p are all 0)
    // adds zeros whatever their unit, and keeps its own.
    const uint32_t vb = sc >> 8;
    uint32_t with[RT];
    bool apart = false;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      with[r] = vb;
      apart |= unit[r] != vb;
    }
    if (ballot(apart)) {
      apart = false;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        uint32_t any = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= p[r][0][0][e] | p[r][0][1][e];
        const bool weighs = max_xor32_u32(max_xor16_u32(any)) != 0;
        if (weighs && unit[r] == 0) unit[r] = vb;
        if (!weighs) with[r] = unit[r];
        apart |= unit[r] != with[r];
      }
    }
    if (!ballot(apart) && !fix) {
#pragma unroll
      for (int d = 0; d < NDT; ++d) {
        const u32x4 w = read(d), x = widen8(w[0], w[1]), y = widen8(w[2], w[3]);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int k = NP - 1; k >= 0; --k) {
            o[r][d] = mfma(x, p[r][k][0], o[r][d]);
            o[r][d] = mfma(y, p[r][k][1], o[r][d]);
          }
      }
      return;
    }
    // the larger scale becomes the unit: what is beyond fp32 below it weighs nothing
    float down[RT], add[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int up = static_cast<int>(with[r]) - static_cast<int>(unit[r]);
      down[r] = ldexpf(1.0f, -max(up, 0));
      add[r] = ldexpf(1.0f, min(up, 0));
      unit[r] = max(unit[r], with[r]);
    }
#pragma unroll
    for (int d = 0; d < NDT; ++d) {
      u32x4 w = read(d), is;  // is: e4m3's 1 where a NaN is, 0 elsewhere
      if (fix) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t bad = nan_bytes(w[e]) >> 7;
          is[e] = bad * 0x38u;
          w[e] &= ~(bad * 0xffu);
        }
      }
      const u32x4 x = widen8(w[0], w[1]), y = widen8(w[2], w[3]);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        f32x4 acc{0, 0, 0, 0};
#pragma unroll
        for (int k = NP - 1; k >= 0; --k) {
          acc = mfma(x, p[r][k][0], acc);
          acc = mfma(y, p[r][k][1], acc);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][d][e] = fmaf(acc[e], add[r], o[r][d][e] * down[r]);
        if (fix) {
          u32x4 see[2];  // 1 where seen, as p lies
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              see[j >> 1][2 * (j & 1) + i] =
                  (ok[r] >> (4 * j + 2 * i) & 1u ? 0x3c00u : 0u) | (ok[r] >> (4 * j + 2 * i + 1) & 1u ? 0x3c000000u : 0u);
          f32x4 hits = mfma(widen8(is[0], is[1]), see[0], f32x4{0, 0, 0, 0});
          hits = mfma(widen8(is[2], is[3]), see[1], hits);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (hits[e] > 0.0f) o[r][d][e] = __builtin_nanf("");
        }
      }
    }
  };
  auto is_inner = [&](int32_t s0) { return s0 + kBlk <= lo.end && (s0 >= hi.low || s0 + kBlk <= sinks); };

  if constexpr (!SHARED) {
    u32x4 kr[4][NJ > 0 ? NJ : 1], vr[NDT];
    u32x2 kh[4];
    constexpr bool AHEAD = NP * DK <= 384;  // fp32 rows of 256 leave no registers for the next K
    auto fetch_k = [&](const uint8_t* base) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint8_t* row = base + (16 * j + col) * DK;
#pragma unroll
        for (int i = 0; i < NJ; ++i) kr[j][i] = *reinterpret_cast<const u32x4*>(row + 64 * i + 16 * g);
        if (HALF) kh[j] = *reinterpret_cast<const u32x2*>(row + 64 * NJ + 8 * g);
      }
    };
    int32_t v = split * WT + wt;
    int32_t page1 = page_of(v + step);
    bool held = false;
    uint32_t sc = 0;
    const uint8_t* base = a.c.codes;
    auto go_to = [&](int32_t v2, int32_t page) __attribute__((always_inline)) {
      const int64_t at = place(v2, page, held);
      sc = scales_at(at);
      base = a.c.codes + at * (kK + kV);
    };
    if (v < total) {
      go_to(v, page_of(v));
      if (AHEAD) fetch_k(base);
    }
    __builtin_amdgcn_sched_barrier(0);
    split_q();
    for (; v < total; v += step) {
      if (!AHEAD) fetch_k(base);
#pragma unroll
      for (int d = 0; d < NDT; ++d) vr[d] = *reinterpret_cast<const u32x4*>(base + kK + (16 * d + col) * kBlk + 16 * g);
      const int32_t page2 = page_of(v + 2 * step);
      const bool held_now = held;
      __builtin_amdgcn_sched_barrier(0);
      logits([&](int j, int i) { return kr[j][i]; }, [&](int j) { return kh[j]; });
      const uint32_t sc_now = __builtin_amdgcn_readfirstlane(sc);  // asked for before K
      __builtin_amdgcn_sched_barrier(0);
      if (v + step < total) {
        go_to(v + step, page1);
        if (AHEAD) fetch_k(base);
      }
      page1 = page2;
      __builtin_amdgcn_sched_barrier(0);
      if (!held_now) continue;
      const int32_t s0 = block_of(v) * kBlk;
      const bool inner = is_inner(s0);
      weights(sc_now, s0, inner);
      sums(sc_now, inner, [&](int d) { return vr[d]; });
    }
  } else {
    // The DMA: an instruction brings 1 KiB, 64 lanes' 16 bytes, to LDS in their order.
    constexpr int kKI = kK / 1024, kVI = kV / 1024;
    constexpr int kMine = (kKI + kVI) / kWaves;  // of a wave: every fourth, K's first
    uint32_t off[kMine];
  #pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int n = wave + kWaves * i;
      if (n < kKI) {
        const int at = n * 64 + lane, r = at / NCK;
        off[i] = r * DK + 16 * chunk_of<NCK>(r, at % NCK);
      } else {
        const int at = (n - kKI) * 64 + lane, r = at / 4;
        off[i] = kK + r * kBlk + 16 * chunk_of<4>(r, at % 4);
      }
    }
    auto dma = [&](const uint8_t* base, int i, DSA_LDS uint8_t* dst) __attribute__((always_inline)) {
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, kK + kV, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, dst, 16, static_cast<int>(off[i]), 0, 0, 0);
    };
    DSA_LDS uint8_t* const kl[2] = {(DSA_LDS uint8_t*)k_lds, (DSA_LDS uint8_t*)k2_lds};
    DSA_LDS uint8_t* const vl[2] = {(DSA_LDS uint8_t*)v_lds, (DSA_LDS uint8_t*)v2_lds};
    auto fetch = [&](int64_t at, DSA_LDS uint8_t* kd, DSA_LDS uint8_t* vd) __attribute__((always_inline)) {
      const uint8_t* base = a.c.codes + at * (kK + kV);
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int n = wave + kWaves * i;
        if (kWaves * i + kWaves <= kKI || (kWaves * i < kKI && n < kKI)) dma(base, i, kd + n * 1024);
        else dma(base, i, vd + (n - kKI) * 1024);
      }
    };
    int32_t v = split;
    int32_t page1 = page_of(v + step);
    bool held = false;
    uint32_t sc = 0;
    if (v < total) {
      const int64_t at = place(v, page_of(v), held);
      sc = scales_at(at);
      fetch(at, kl[0], vl[0]);
    }
    __builtin_amdgcn_sched_barrier(0);
    split_q();
    wait_dma_keep<0>();
    block_sync_lds();
    auto turn = [&](DSA_LDS uint8_t* kc, DSA_LDS uint8_t* vc, DSA_LDS uint8_t* kn, DSA_LDS uint8_t* vn) __attribute__((always_inline)) {
      const uint32_t sc_now = __builtin_amdgcn_readfirstlane(sc);
      const bool held_now = held;
      const int32_t page2 = page_of(v + 2 * step);
      if (v + step < total) {
        const int64_t at = place(v + step, page1, held);
        sc = scales_at(at);
        fetch(at, kn, vn);
      }
      page1 = page2;
      __builtin_amdgcn_sched_barrier(0);
      const int32_t s0 = block_of(v) * kBlk;
      if (held_now && any_rows && s0 < hi.end && (s0 + kBlk > lo.low || s0 < sinks)) {
        const bool inner = is_inner(s0);
        const DSA_LDS uint8_t* const kp = kc + col * DK;
        const DSA_LDS uint8_t* const vp = vc + col * kBlk + 16 * chunk_at<4>(col, g);
        logits([&](int j, int i) { return *reinterpret_cast<const DSA_LDS u32x4*>(kp + 16 * j * DK + 16 * chunk_at<NCK>(col, 4 * i + g)); },
               [&](int j) { return *reinterpret_cast<const DSA_LDS u32x2*>(kp + 16 * j * DK + 16 * chunk_at<NCK>(col, 4 * NJ + (g >> 1)) + 8 * (g & 1)); });
        weights(sc_now, s0, inner);
        sums(sc_now, inner, [&](int d) { return *reinterpret_cast<const DSA_LDS u32x4*>(vp + 16 * d * kBlk); });
      }
      wait_dma_keep<0>();
      block_sync_lds();
      v += step;
    };
    while (v < total) {
      turn(kl[0], vl[0], kl[1], vl[1]);
      if (v < total) turn(kl[1], vl[1], kl[0], vl[0]);
    }
  }

#pragma unroll
  for (int r = 0; r < RT; ++r) {
    l[r] = sum_xor32(sum_xor16(l[r]));
    if (odd_row[r]) l[r] = __builtin_nanf("");
    if (!token[r]) {  // no token: sees nothing
      m[r] = -INFINITY;
      l[r] = 0.0f;
    }
    // Divided by the sum of weights before V's unit comes in: the mean of values that fp32 holds
    // is one too, where p times them, 2^10 and more, may not be.  (v_rcp_f32 is within 2^-23.)
    const float inv = l[r] == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(l[r]), us = __uint_as_float(unit[r] << 23);
#pragma unroll
    for (int d = 0; d < NDT; ++d) o[r][d] = token[r] ? o[r][d] * inv * us : f32x4{0, 0, 0, 0};
  }
  auto finish = [&](int row, int d, f32x4 x, float top, float all) __attribute__((always_inline)) {
    const int64_t hr = (b * a.Tq + row / a.G) * a.HQ + h * a.G + row % a.G;
    if (a.splits > 1) {
      *reinterpret_cast<f32x4*>(a.part + (hr * a.splits + split) * DV + d) = x;
      if (d == 0) a.ml[hr * a.splits + split] = make_float2(top, all);
    } else {
      store4<Tag>(static_cast<raw*>(a.out) + hr * DV + d, all == 0.0f ? x * __builtin_nanf("") : x);  // nothing is seen
    }
  };
  if constexpr (SHARED) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      if (first_row + 16 * r + col > last_row) continue;
#pragma unroll
      for (int d = 0; d < NDT; ++d) finish(first_row + 16 * r + col, 16 * d + 4 * g, o[r][d], m[r], l[r]);
    }
  } else {  // join the waves
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      if (g == 0) {
        sum_m[wt][16 * r + col] = m[r];
        sum_l[wt][16 * r + col] = l[r];
      }
#pragma unroll
      for (int d = 0; d < NDT; ++d) *reinterpret_cast<f32x4*>(sum_o + (wt * kTile + 16 * r + col) * DV + 16 * d + 4 * g) = o[r][d];
    }
    __syncthreads();
    constexpr int kQuads = DV / 4;
    for (int e = threadIdx.x; e < block_rows * kQuads; e += kNT) {
      const int r = e / kQuads, d = e % kQuads * 4;
      float top = sum_m[0][r];
#pragma unroll
      for (int w = 1; w < WT; ++w) top = fmaxf(top, sum_m[w][r]);
      const float ref = top == -INFINITY ? 0.0f : top;
      float share[WT], all = 0.0f;
      f32x4 x{0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < WT; ++w) all += share[w] = __builtin_amdgcn_exp2f(sum_m[w][r] - ref) * sum_l[w][r];
      const float inv = all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
      for (int w = 0; w < WT; ++w) x += *reinterpret_cast<const f32x4*>(sum_o + (w * kTile + r) * DV + d) * (share[w] * inv);
      finish(block_row + r, d, x, top, all);
    }
  }
}

constexpr int kMaxSplits = 512;

// Few splits of many rows: a thread joins 4 columns of a row, all splits on their way at once.
constexpr int kFewSplits = 8;
template <typename Tag>
__global__ __launch_bounds__(kNT) void join_few_kernel(const float* __restrict__ part, const float2* __restrict__ ml,
                                                       int splits, int DV, int64_t rows, typename Tag::raw* __restrict__ out) {
  const int quads = DV / 4, per = kNT / quads;
  const int64_t row = blockIdx.x * static_cast<int64_t>(per) + threadIdx.x / quads;
  if (threadIdx.x >= per * quads || row >= rows) return;
  const int d = threadIdx.x % quads * 4;
  float2 x[kFewSplits];
  float4 y[kFewSplits];
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    const int64_t at = row * splits + min(s, splits - 1);
    x[s] = ml[at];
    y[s] = *reinterpret_cast<const float4*>(part + at * DV + d);
  }
  float top = x[0].x;
#pragma unroll
  for (int s = 1; s < kFewSplits; ++s) top = fmaxf(top, x[s].x);
  const float ref = top == -INFINITY ? 0.0f : top;
  float all = 0.0f;
  f32x4 z{0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    if (s >= splits) break;
    all += x[s].y *= __builtin_amdgcn_exp2f(x[s].x - ref);
  }
  const float inv = 1.0f / all;  // nothing is seen: 0 * Inf
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    if (s >= splits) break;
    z += f32x4{y[s].x, y[s].y, y[s].z, y[s].w} * (x[s].y * inv);
  }
  store4<Tag>(out + row * DV + d, z);
}

// A block joins one row's splits: 20 of rows of 128, 31 MB in all, in 8 us.  (Threads that
// take 4 columns and every eighth split took 9, threads that hold all splits of 4 columns 28.)
template <typename Tag>
__global__ __launch_bounds__(kNT) void join_kernel(const float* __restrict__ part, const float2* __restrict__ ml,
                                                   int splits, int DV, typename Tag::raw* __restrict__ out) {
  __shared__ float factor[kMaxSplits];
  __shared__ float2 both[kWaves];
  const int64_t row = blockIdx.x;
  const float2* mine = ml + row * splits;
  float top = -INFINITY;
  for (int s = threadIdx.x; s < splits; s += kNT) top = fmaxf(top, mine[s].x);
  top = wave_max(top);
  if ((threadIdx.x & 63) == 0) both[threadIdx.x >> 6].x = top;
  __syncthreads();
  top = fmaxf(fmaxf(both[0].x, both[1].x), fmaxf(both[2].x, both[3].x));
  const float ref = top == -INFINITY ? 0.0f : top;
  float all = 0.0f;
  for (int s = threadIdx.x; s < splits; s += kNT) {
    const float2 x = mine[s];
    const float f = __builtin_amdgcn_exp2f(x.x - ref) * x.y;
    factor[s] = f;
    all += f;
  }
  all = wave_sum(all);
  if ((threadIdx.x & 63) == 0) both[threadIdx.x >> 6].y = all;
  __syncthreads();
  all = both[0].y + both[1].y + both[2].y + both[3].y;
  if (threadIdx.x >= DV) return;
  const float inv = 1.0f / all;  // nothing is seen: 0 * Inf
  float x = 0.0f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) x += factor[s] * inv * part[(row * splits + s) * DV + threadIdx.x];
  if constexpr (Tag::kBytes == 4) out[row * DV + threadIdx.x] = x;
  else if constexpr (__is_same(Tag, BF16)) out[row * DV + threadIdx.x] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
  else out[row * DV + threadIdx.x] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
}

// How rows and slots go over blocks and waves.
struct Plan {
  int splits, row_tiles;
  int rt;       // tiles of 16 rows a wave
  bool shared;  // a block's waves take different rows of the same slots
  int64_t ml, total;  // bytes
};

Plan plan_of(const Kv8& c, int64_t Tq, int HQ, int64_t n, int64_t window, int64_t sinks, bool fp32) {
  Plan p;
  const int64_t rows = Tq * (HQ / c.HKV), tiles = (rows + 15) / 16, pairs = c.B * c.HKV;
  int64_t most = (n + kBlk - 1) / kBlk;  // blocks that a row tile walks
  if (window > 0) {
    const int64_t near = (window + Tq - 1 + kBlk - 1) / kBlk + 1 + (sinks < n ? (sinks + kBlk - 1) / kBlk : most);
    most = near < most ? near : most;
  }
  const int64_t work = pairs * tiles * most;
  // Rows share blocks of slots by way of LDS where there are rows for it and, beyond the few
  // slots that leave a wave nothing of its own, enough to do to pay for the barriers and the
  // joins; the shorter K rows are, the fewer accesses that saves.  us, waves' own / shared (bf16):
  //   D 128, 48 rows: 32 pairs of 1024 slots 10.6 / 13.7, of 8192 29.3 / 26.0; 128 of 16384 187 / 127
  //   D 64: 128 pairs of 16384, 64 rows 79 / 84; D 192: 256 of 700, 48 rows 32.0 / 28.7
  //   D 64, 464 rows over 58 slots: 96 pairs 15.1 / 8.4; 800 rows over 100: 2 pairs 5.4 / 6.1
  p.shared = rows > 32 && (most <= 4 ? pairs * tiles >= 1024 : c.DK > 96 && work >= (c.DK > 128 ? 8192 : 12288));
  // 32 rows a wave share the widening of K and V where the registers hold them, against half
  // the blocks (16 / 32 rows):
  //   own, D 64, 64 rows: 32 pairs of 8192 slots 17.9 / 19.5; 256 of 4096 42.1 / 36.1
  //   shared, D 128, 4 pairs of 8192 slots: 512 rows 32.8 / 35.1, 640 38.3 / 38.1, 768 40.7 / 42.1,
  //     2048 70.3 / 62.0; 8 pairs: 256 29.6 / 31.9, 512 41.8 / 41.5, 768 58.4 / 56.3, 2048 123 / 103
  //   256 pairs of 4096: 64 78 / 96, 128 122 / 113, 192 163 / 171, 256 215 / 179, 512 384 / 334
  //   4 pairs of 32768: 192 37.0 / 39.4, 256 42.0 / 41.5, 384 59.1 / 53.7, 512 68.6 / 61.4, 768 101 / 87
  // (From 640 rows on 32 cost a few in 100 at most and win a tenth or more where there is much to do;
  // the latter would from 256 on.)
  p.rt = !fp32 && (p.shared ? c.DK == 128 && most > 4 && rows > 512 : c.DK <= 96 && rows > 16 && work >= 24576) ? 2 : 1;
  const int64_t tile = 16 * p.rt * (p.shared ? kWaves : 1), waves = p.shared ? 1 : kWaves;
  p.row_tiles = static_cast<int>((rows + tile - 1) / tile);
  // A few turns of a block's waves cost less than the launch that joins splits (one head's 5
  // turns: 10.6 whole, 10.4 split; 6: 11.9, 9.5; shared, 4: 13.7, 13.0), and a split takes two at least.
  const int64_t turns = (most + waves - 1) / waves;
  const int64_t steps = turns <= (p.shared ? 3 : 5) ? 1 : turns / 2;
  // as many splits as all run at once: the chunks go over 8 XCDs in equal numbers, and
  // one that waits for a place makes a second round (4 sequences, 48 rows of one head of 128
  // over 8191 slots: 35 us with 2 x 33 blocks an XCD of 2 x 32 places, 29 with 2 x 32)
  const int64_t room = (c.DK <= 128 || (p.shared && !fp32) ? 2 : 1) * int64_t{device_cus() > 0 ? device_cus() : 256};
  int64_t chunks = rows < 1 ? 0 : room / p.row_tiles;
  if (chunks >= 8) chunks = chunks / 8 * 8;
  int64_t splits = pairs < 1 || pairs >= chunks ? 1 : chunks / pairs;
  splits = splits > steps ? steps : splits;
  p.splits = static_cast<int>(splits > kMaxSplits ? kMaxSplits : splits);
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  const int64_t heads = c.B * Tq * HQ;
  p.ml = p.splits > 1 ? up(heads * p.splits * 8) : 0;
  p.total = p.ml + (p.splits > 1 ? up(heads * p.splits * c.DV * 4) : 0);
  return p;
}
// The workspace does not depend on the queries' type.
int64_t workspace_of(const Kv8& c, int64_t Tq, int HQ, int64_t n, int64_t window, int64_t sinks) {
  return std::max(plan_of(c, Tq, HQ, n, window, sinks, false).total, plan_of(c, Tq, HQ, n, window, sinks, true).total);
}

template <typename Tag, int DK, int DV>
void launch_dims(const AttnArgs& a, const Plan& p, uint32_t grid, hipStream_t stream) {
  if constexpr (Tag::kBytes == 2 && DK == 128)
    if (p.shared && p.rt == 2) return (void)(attn_kernel<Tag, DK, DV, 2, true><<<grid, kNT, 0, stream>>>(a));
  if constexpr (Tag::kBytes == 2 && DK <= 96)
    if (!p.shared && p.rt == 2) return (void)(attn_kernel<Tag, DK, DV, 2, false><<<grid, kNT, 0, stream>>>(a));
  if (p.shared) attn_kernel<Tag, DK, DV, 1, true><<<grid, kNT, 0, stream>>>(a);
  else attn_kernel<Tag, DK, DV, 1, false><<<grid, kNT, 0, stream>>>(a);
}

template <typename Tag>
hipError_t launch_type(const AttnArgs& a, const Plan& p, hipStream_t stream) {
  const int64_t chunks = a.few_chunks ? a.few_chunks : (a.c.B * a.c.HKV * p.splits + 7) / 8 * 8;
  const uint32_t grid = static_cast<uint32_t>(chunks * p.row_tiles);
  if (a.c.DK != a.c.DV) launch_dims<Tag, 192, 128>(a, p, grid, stream);
  else switch (a.c.DK) {
    case 32: launch_dims<Tag, 32, 32>(a, p, grid, stream); break;
    case 64: launch_dims<Tag, 64, 64>(a, p, grid, stream); break;
    case 96: launch_dims<Tag, 96, 96>(a, p, grid, stream); break;
    case 128: launch_dims<Tag, 128, 128>(a, p, grid, stream); break;
    case 192: launch_dims<Tag, 192, 192>(a, p, grid, stream); break;
    default: launch_dims<Tag, 256, 256>(a, p, grid, stream);
  }
  typename Tag::raw* const out = static_cast<typename Tag::raw*>(a.out);
  const int64_t rows = a.c.B * a.Tq * a.HQ;
  if (p.splits == 1) return hipGetLastError();
  // many rows: a few a block (with the attention, of 8496 rows 26 us, 34 with a block a row; of 128
  // 12.9 and 11.1)
  if (p.splits > kFewSplits || rows < 1024) {
    join_kernel<Tag><<<static_cast<uint32_t>(rows), kNT, 0, stream>>>(a.part, a.ml, p.splits, a.c.DV, out);
  } else {
    const int64_t per = kNT / (a.c.DV / 4);
    join_few_kernel<Tag><<<static_cast<uint32_t>((rows + per - 1) / per), kNT, 0, stream>>>(a.part, a.ml, p.splits, a.c.DV, rows, out);
  }
  return hipGetLastError();
}

}  // namespace

bool kv8_supported(int DK, int DV) {
  if (DK == 192 && DV == 128) return true;
  return DK == DV && (DK == 32 || DK == 64 || DK == 96 || DK == 128 || DK == 192 || DK == 256);
}

int64_t kv8_attn_workspace(const Kv8& c, int64_t Tq, int HQ, int64_t n, int64_t window, int64_t sinks) {
  return workspace_of(c, Tq, HQ, n, std::min(window, c.slots()), std::min(sinks, c.slots()));
}

hipError_t launch_kv8_attn(const Kv8& c, const void* Q, int dtype, const int32_t* count, int64_t Tq, int HQ,
                           int64_t n, int64_t window, int64_t sinks, float scale, void* out, void* ws,
                           hipStream_t stream) {
  window = std::min(window, c.slots());  // no token has more before it
  sinks = std::min(sinks, c.slots());
  const Plan p = plan_of(c, Tq, HQ, n, window, sinks, dtype == 0);
  AttnArgs a;
  a.c = c;
  a.Q = Q;
  a.count = count;
  a.Tq = static_cast<int>(Tq);
  a.HQ = HQ;
  a.G = HQ / c.HKV;
  a.row_tiles = p.row_tiles;
  a.splits = p.splits;
  // (12 heads of 64, 512 tokens of 8 each over 1000 slots: 41 us with two heads on four of the XCDs, 31
  // so; with many chunks the XCDs have much the same, and a chunk's row tiles one L2)
  a.few_chunks = c.B * c.HKV * p.splits < 64 ? static_cast<uint32_t>(c.B * c.HKV * p.splits) : 0u;
  a.n = n;
  a.window = window;
  a.sinks = sinks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = out;
  a.ml = static_cast<float2*>(ws);
  a.part = reinterpret_cast<float*>(static_cast<char*>(ws) + p.ml);
  return dtype == 0 ? launch_type<F32>(a, p, stream) : dtype == 1 ? launch_type<BF16>(a, p, stream) : launch_type<F16>(a, p, stream);
}

}  // namespace dsa
