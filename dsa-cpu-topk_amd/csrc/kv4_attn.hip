// kv4_attn.hip -- attention of new tokens over the 4-bit decode cache (gfx950):
//   p = softmax over the visible (or listed) slots of <Q, K> * scale
//   O = sum p V,   weight[b, slot] += sum over queries and heads of p
//
// One pass over the cache with a running maximum and sum.  A wave takes 32 slots
// at a time of one K/V head and up to 16 rows, query heads of its group (of all
// tokens together where they attend to the same slots), on v_mfma_f32_16x16x32_bf16:
//
//   S^T[slot, head] = K Q^T    A: a lane holds 8-element runs of one slot's K row,
//                              converted from e2m1 with their scale by one
//                              instruction a pair (exact in bf16);
//   O^T[d, head]  += V^T P^T   A: a lane holds W/16 columns of 8 slots (W = 128, 64
//                              or 32 columns at a time), pairs of slots put
//                              together by v_perm.
//
// The sum over a matrix instruction's 32 terms may take them in any order, as long
// as both operands agree.  So a lane's K run is what one wide load brings, and the
// slots of P are those whose logits the lane already has (rows 4g .. 4g+3 of S^T's
// two tiles, g = lane / 16): P needs no transposing.  The slots' rows come by wide
// loads one turn ahead and pass through the wave's own part of LDS, which gives
// their registers to the next ones and hands V's words and the scales to the
// lanes that take them.
//
// fp32 operands enter as bf16 pieces: Q as one (bf16), two (fp16) or three (fp32),
// p as three, which hold its 24 bits.  For up to 5 rows the three
// pieces of p stand side by side in the 16 columns (Q is repeated there, so each
// lane has the p whose piece it takes) and one instruction takes them all.
//
// Long caches are split: the tiles of 32 slots go to the blocks' waves in turn, and
// each block leaves its sums, relative to its own maximum, for the second launch
// to join.  That launch also adds the probabilities onto the slots' weights, from
// the logits that the first one stored.  A block's waves take four neighbouring
// heads, so that they read whole rows of the token-major cache (a read of the same
// 1 GiB by rows of 128 bytes a block 4.5-5.1 TB/s, of 512 6.0, linear 6.35).
//
// Measured, 16 sequences of up to 32768 slots, 32 heads on 8, D 128, bf16 (443 MB):
// 94 us, 4.7 TB/s (all of them full: 5.4).  The loads alone take 88 of the first
// launch's 90 us, the arithmetic alone 74-82 (about 190 vector and 16 matrix
// instructions a tile).  Short calls are bound by latency: 1.2 us to the sequence's
// length, 1-2 to its first rows, 0.5 a tile, 0.5-2 to join a block's waves, 3-6 for
// the second launch.
#include <type_traits>

#include "dsa_launch.h"
#include "kv4.h"
#include "tile_common.h"

namespace dsa {
namespace {

constexpr int kWaves = kNT / kWave;
constexpr int kTile = 32;                  // slots a wave takes at once
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;             // how far a logit may pass the running maximum, in powers of 2
constexpr float kNoSum = -1.0f;            // a split's sum of exponentials where it has no slots

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// A row of D elements in pieces of 128, 64 and 32 columns.
__host__ __device__ constexpr int seg_count(int D) { return D / 128 + (D % 128) / 64 + (D % 64) / 32; }
__host__ __device__ constexpr int seg_width(int D, int s) {
  return s < D / 128 ? 128 : s == D / 128 && D % 128 >= 64 ? 64 : 32;
}
__host__ __device__ constexpr int seg_at(int D, int s) {
  int at = 0;
  for (int i = 0; i < s; ++i) at += seg_width(D, i);
  return at;
}

struct AttnArgs {
  Kv4 c;
  const void* Q;
  const int32_t* slots;  // or null
  const int32_t* count;  // or null
  int Tq, HQ, G;
  int row_tiles;  // tiles of 16 rows
  int heads;  // K/V heads a block takes: 4, 2 or 1, its 4 / heads waves of each sharing the slots
  int64_t n, stride;  // slots a query; floats between rows of logits
  int splits;         // blocks that share a query's slots
  int join_cols;      // columns of a head that a joining block takes
  float scale;
  float* out;
  float* part;    // [B*Tq*HQ][splits][DV] sums, where splits > 1
  float2* ml;     // [B*Tq*HQ][splits] maximum (in powers of 2) and sum of exponentials, or null
  float* logits;  // [B*Tq*HQ][stride], in powers of 2, or null
};

template <int BYTES>
__device__ __forceinline__ uint32_t load_small(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  if constexpr (BYTES == 4) return __float_as_uint(buffer_load_f32(r, static_cast<int>(off), 0, 0));
  else if constexpr (BYTES == 2) return __builtin_amdgcn_raw_buffer_load_b16(r, static_cast<int>(off), 0, 0);
  else return __builtin_amdgcn_raw_buffer_load_b8(r, static_cast<int>(off), 0, 0);
}
// W / 8 bytes: a quarter of W codes.
template <int W>
__device__ __forceinline__ void load_codes(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t* to) {
  if constexpr (W == 128) {
    const dsa_f32x4 x = buffer_load_f32x4(r, static_cast<int>(off), 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = __float_as_uint(x[i]);
  } else if constexpr (W == 64) {
    const dsa_f32x2 x = buffer_load_f32x2(r, static_cast<int>(off), 0, 0);
    to[0] = __float_as_uint(x[0]);
    to[1] = __float_as_uint(x[1]);
  } else {
    to[0] = load_small<4>(r, off);
  }
}

// The sizes of a wave's 32 slots, in registers and in LDS.
template <int DK, int DV>
struct Shape {
  static constexpr int kScales = (DK > DV ? DK : DV) / 32;  // bytes a lane loads
  // their alignment: a half (K's or V's scales) starts at a multiple of it
  static constexpr int kUnit = DK % 128 == 0 && DV % 128 == 0 ? 4 : DK % 64 == 0 && DV % 64 == 0 ? 2 : 1;
  static constexpr int kLoads = (kScales + kUnit - 1) / kUnit;
  // LDS: K, V, scales
  static constexpr int kV = 2 * 16 * DK / 2, kS = kV + 2 * 16 * DV / 2;
  static constexpr int kBytes = kS + (DK + DV);  // a multiple of 16
};

// What a wave has loaded of its 32 slots, two tiles of 16.
template <int DK, int DV>
struct Frag {
  uint32_t k[2][DK / 32];  // a quarter of the row of slot lane % 16
  uint32_t v[2][DV / 32];  // a quarter of the row of slot 4 * (lane / 4 % 4) + lane / 16
  uint32_t s[Shape<DK, DV>::kLoads];  // K's (even lanes) or V's scales of slot lane / 2 of the 32
  uint32_t ok;  // bit i: slot i counts (for the block's one token)
};

constexpr uint32_t kNowhere = 0x80000000u;  // past any sequence's codes: such loads give zeros

// krow, vrow, srow: byte offsets of the slots' codes (of their scales: 1/16 of it).
template <int DK, int DV>
__device__ __forceinline__ void load_frag(Frag<DK, DV>& f, __amdgpu_buffer_rsrc_t rc,
                                          __amdgpu_buffer_rsrc_t rs, const uint32_t (&krow)[2],
                                          const uint32_t (&vrow)[2], uint32_t srow, int hk) {
  using S = Shape<DK, DV>;
  const int lane = threadIdx.x & 63;
  const uint32_t head = hk * (DK + DV) / 2;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int s = 0; s < seg_count(DK); ++s) {
      const int at = seg_at(DK, s);
      const uint32_t row = krow[t] + head + at / 2;
      if (seg_width(DK, s) == 128) load_codes<128>(rc, row + (lane >> 4) * 16, f.k[t] + at / 32);
      else if (seg_width(DK, s) == 64) load_codes<64>(rc, row + (lane >> 4) * 8, f.k[t] + at / 32);
      else load_codes<32>(rc, row + (lane >> 4) * 4, f.k[t] + at / 32);
    }
  }
  const uint32_t half = srow / 16 + hk * (DK + DV) / 32 + (lane & 1) * (DK / 32);
#pragma unroll
  for (int i = 0; i < S::kLoads; ++i) f.s[i] = load_small<S::kUnit>(rs, half + i * S::kUnit);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int s = 0; s < seg_count(DV); ++s) {
      const int at = seg_at(DV, s);
      const uint32_t row = vrow[t] + head + DK / 2 + at / 2;
      if (seg_width(DV, s) == 128) load_codes<128>(rc, row + (lane & 3) * 16, f.v[t] + at / 32);
      else if (seg_width(DV, s) == 64) load_codes<64>(rc, row + (lane & 3) * 8, f.v[t] + at / 32);
      else load_codes<32>(rc, row + (lane & 3) * 4, f.v[t] + at / 32);
    }
  }
}

// A wave's slots go through its own part of LDS, which leaves their registers to
// the next ones while these are worked on, and where V and the scales change lanes:
//   K      [tile][segment][lane], for the lane that wrote it;
//   V      [tile][segment][r][g] rows of W / 2 bytes, slot 4g + r of the tile, so that
//          the 64 lanes write, and for one r read, consecutive bytes;
//   scales [block][slot], four slots of a block in one word.
template <int DK, int DV>
__device__ __forceinline__ void stage(const Frag<DK, DV>& f, uint8_t* lds) {
  using S = Shape<DK, DV>;
  const int lane = threadIdx.x & 63;
  auto put = [&](uint8_t* at_lane0, const uint32_t* v, int W) {
    uint8_t* to = at_lane0 + lane * (W / 8);
    if (W == 128) *reinterpret_cast<uint4*>(to) = make_uint4(v[0], v[1], v[2], v[3]);
    else if (W == 64) *reinterpret_cast<uint2*>(to) = make_uint2(v[0], v[1]);
    else *reinterpret_cast<uint32_t*>(to) = v[0];
  };
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int s = 0; s < seg_count(DK); ++s)
      put(lds + t * 8 * DK + 8 * seg_at(DK, s), f.k[t] + seg_at(DK, s) / 32, seg_width(DK, s));
#pragma unroll
    for (int s = 0; s < seg_count(DV); ++s)
      put(lds + S::kV + t * 8 * DV + 8 * seg_at(DV, s), f.v[t] + seg_at(DV, s) / 32, seg_width(DV, s));
  }
  uint8_t* to = lds + S::kS + (lane & 1) * DK + (lane >> 1);  // 32 bytes a block
  const int mine = (lane & 1) ? DV / 32 : DK / 32;
#pragma unroll
  for (int i = 0; i < S::kScales; ++i)
    if (DK == DV || i < mine) to[i * 32] = static_cast<uint8_t>(f.s[i / S::kUnit] >> (i % S::kUnit * 8));
}

// The conversions read a scale's exponent bits alone (checked over all bytes with
// any sign and mantissa), so a byte of a word becomes a scale by one shift.
template <int BYTE>
__device__ __forceinline__ float scale_of(uint32_t w) {
  if constexpr (BYTE == 3) return __uint_as_float(w >> 1);
  else return __uint_as_float(w << (23 - 8 * BYTE));
}

// Orders a wave's LDS accesses, which the hardware takes in order, for the compiler.
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

template <int SEL>
__device__ __forceinline__ uint32_t cvt2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}
__device__ __forceinline__ float hi16(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_hi(float lo, float hi) {  // the upper halves
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, f32x4 c) {
  return Mfma16x16x32<BF16>::run(a, b, c);
}

// 8 elements of a query row, or their negatives, as NP pieces of bf16; zeros where not used.
template <typename Tag, int NP>
__device__ __forceinline__ void split_q8(const typename Tag::raw (&raw)[8], bool used, bool negative, u32x4 (&q)[NP]) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = used ? to_f32(Tag{}, raw[j]) : 0.0f;
    x[j] = negative ? -x[j] : x[j];
  }
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      q[i][j] = pack_hi(x[2 * j], x[2 * j + 1]);
      x[2 * j] -= hi16(x[2 * j]);
      x[2 * j + 1] -= hi16(x[2 * j + 1]);
    }
}

// Waves a SIMD holds: what the registers allow without spills.
__host__ __device__ constexpr int resident(int NP, int DK, int DV, bool side) {
  if (DK <= 64 || (DK <= 128 && NP == 1 && side)) return 4;
  if (DK <= 128 || (DV <= 128 && NP == 1)) return 3;
  return DK <= 192 || NP < 3 ? 2 : 1;
}

// A block's rows: one token's heads over the first slots or over listed ones, or
// all tokens' heads over the first slots.
enum Rows { kOne, kListed, kTokens };

template <typename Tag, int NP, int DK, int DV, bool SIDE, Rows ROWS>
__global__ __launch_bounds__(kNT, resident(NP, DK, DV, SIDE)) void attn_kernel(AttnArgs a) {
  using S = Shape<DK, DV>;
  constexpr bool LISTED = ROWS == kListed, MANY = ROWS == kTokens;
  constexpr int NW = DK / 32, NO = DV / 16, LD = DV + 4;
  constexpr int kSums = kWaves * 16 * LD * 4, kStages = kWaves * S::kBytes;
  __shared__ __align__(16) uint8_t lds[kSums > kStages ? kSums : kStages];  // the stages, then the sums
  float(*sum_o)[16][LD] = reinterpret_cast<float(*)[16][LD]>(lds);
  __shared__ float sum_m[kWaves][16], sum_l[kWaves][16];

  // Blocks go round-robin over the 8 XCDs; the blocks of one chunk (its heads)
  // read the same rows, so they go to one XCD, one after another.
  const uint32_t per = a.c.HKV / a.heads * a.row_tiles;
  const uint32_t i = blockIdx.x / 8, chunk = i / per * 8 + blockIdx.x % 8, member = i % per;
  const uint32_t groups = MANY ? 1 : a.Tq, bg = chunk / a.splits, b = bg / groups, t0 = bg % groups;
  if (b >= a.c.B) return;
  const int hk0 = member / a.row_tiles * a.heads, rt = member % a.row_tiles, split = chunk % a.splits;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
  const int hk = hk0 + wave % a.heads;  // the wave's K/V head
  const int share = wave / a.heads, shares = kWaves / a.heads;
  const int step = kTile * shares * a.splits;  // slots that the head's waves in all blocks take at once
  // the lane's row, a token's query head, and (SIDE) which piece of p it takes
  const int all_rows = MANY ? a.Tq * a.G : a.G;
  const int row = SIDE ? col % all_rows : rt * 16 + col;
  const int piece = SIDE ? col / all_rows : 0;
  const bool used = SIDE ? piece < 3 : row < all_rows;
  auto token_of = [&](int r) { return MANY ? r / a.G : 0; };
  // where row r of head hd stands in [B, Tq, HQ]
  const uint32_t bh = (b * a.Tq + t0) * a.HQ;  // all rows are fewer than 2^23
  auto head_of = [&](int hd, int r) -> uint32_t {
    const int t = token_of(r);
    return bh + t * a.HQ + hd * a.G + (r - t * a.G);
  };
  const uint32_t my_head = head_of(hk, used ? row : 0);

  // the query row, in the order of the K runs; asked for before anything waits
  typename Tag::raw q_raw[NW][8];
  {
    const typename Tag::raw* src = static_cast<const typename Tag::raw*>(a.Q) + static_cast<int64_t>(my_head) * DK;
#pragma unroll
    for (int s = 0; s < seg_count(DK); ++s) {
      const int W = seg_width(DK, s), at = seg_at(DK, s);
#pragma unroll
      for (int k = 0; k < W / 32; ++k)
        __builtin_memcpy(q_raw[at / 32 + k], __builtin_assume_aligned(src + at + g * (W / 4) + 8 * k, 16), sizeof(q_raw[0]));
    }
  }

  // `limit` slots for some of the block's rows (their last token sees the most),
  // `my_limit` for the lane's own.
  int32_t limit, my_limit;
  if constexpr (!MANY) {
    limit = kv4_visible(a.c.length, a.count, b, a.c.S, t0, a.Tq);
    if (!LISTED) limit = static_cast<int32_t>(min(static_cast<int64_t>(limit), a.n));
    my_limit = limit;
  } else {
    const int32_t n = a.count ? max(0, min(a.count[b], a.Tq)) : a.Tq, have = kv4_length(a.c.length, b, a.c.S) - n + 1;
    const int32_t most = static_cast<int32_t>(a.n);
    const int first = token_of(rt * 16), last = min(token_of(min(rt * 16 + 16, all_rows) - 1), n - 1);
    limit = last >= first ? max(0, min(have + last, most)) : 0;
    const int mine = token_of(used ? row : rt * 16);
    my_limit = mine < n ? max(0, min(have + mine, most)) : 0;
  }
  // Tiles go to the waves in turn, so that every block has its share of the slots in use.
  const int64_t j_end = LISTED ? (limit > 0 ? a.n : 0) : limit;
  const int64_t j_first = static_cast<int64_t>(split) * shares * kTile;
  const int rows = SIDE ? all_rows : min(16, all_rows - rt * 16);
  if (j_first >= j_end) {  // nothing here: no sum, and no sums to read
    for (int e = threadIdx.x; e < a.heads * rows; e += kNT) {
      const int64_t h = head_of(hk0 + e / rows, rt * 16 + e % rows);
      if (a.ml) a.ml[h * a.splits + split] = make_float2(-INFINITY, kNoSum);
      if (a.splits == 1)
        for (int d = 0; d < DV; ++d) a.out[h * DV + d] = __builtin_nanf("");
    }
    return;
  }

  const uint32_t mask1 = piece >= 1 ? 0xffff0000u : 0u, mask2 = piece >= 2 ? 0xffff0000u : 0u;

  const uint32_t cb = a.c.words() * 4;  // bytes of a slot's codes; of its scales: cb / 16
  const uint8_t* codes = a.c.codes + b * a.c.S * cb;
  const uint8_t* scales = a.c.scales + b * a.c.S * (cb / 16);
  // rows end at the last slot that counts: loads past it give zeros
  auto rsrc = [](const uint8_t* base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, static_cast<int>(bytes), 0x00020000);
  };
  const __amdgpu_buffer_rsrc_t all_codes = rsrc(codes, static_cast<int64_t>(limit) * cb);
  const __amdgpu_buffer_rsrc_t all_scales = rsrc(scales, static_cast<int64_t>(limit) * (cb / 16));
  const int32_t* list = LISTED ? a.slots + (static_cast<int64_t>(b) * a.Tq + t0) * a.n : nullptr;
  const int vslot = 4 * ((lane >> 2) & 3) + (lane >> 4);

  // A listed slot's offset, of entry j0 + lane % 32; read a step before the slots.
  auto entry = [&](int64_t j0) -> uint32_t {
    const int64_t j = j0 + (lane & 31);
    const uint32_t s = j < j_end ? static_cast<uint32_t>(list[j]) : ~0u;
    return s < static_cast<uint32_t>(limit) ? s * cb : kNowhere;
  };
  auto load = [&](Frag<DK, DV>& f, int64_t j0, uint32_t off) {
    if constexpr (LISTED) {
      auto from = [&](int l) { return static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(4 * l, static_cast<int>(off))); };
      const uint32_t krow[2] = {from(col), from(16 + col)}, vrow[2] = {from(vslot), from(16 + vslot)};
      load_frag<DK, DV>(f, all_codes, all_scales, krow, vrow, from(lane >> 1), hk);
      f.ok = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(off != kNowhere));
    } else {
      const uint32_t krow[2] = {col * cb, (16 + col) * cb}, vrow[2] = {vslot * cb, (16 + vslot) * cb};
      const int64_t rest = max(static_cast<int64_t>(0), limit - j0);
      if (!MANY) f.ok = rest >= kTile ? ~0u : (1u << rest) - 1;
      load_frag<DK, DV>(f, rsrc(codes + j0 * cb, rest * cb), rsrc(scales + j0 * (cb / 16), rest * (cb / 16)), krow,
                        vrow, (lane >> 1) * cb, hk);
    }
  };

  int64_t j = j_first + share * kTile;
  Frag<DK, DV> f;
  uint32_t off = LISTED ? entry(j) : 0;
  if (j < j_end) load(f, j, off);

  u32x4 q[NW][NP];
#pragma unroll
  for (int w = 0; w < NW; ++w) split_q8<Tag, NP>(q_raw[w], used, a.scale < 0.0f, q[w]);

  f32x4 o[NO];
#pragma unroll
  for (int i2 = 0; i2 < NO; ++i2) o[i2] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;
  // logits in powers of 2; a scale of 0 stays one above it, so that -inf stays -inf
  const float to2 = fmaxf(fabsf(a.scale) * kLog2e, 1.17549435e-38f);

  uint8_t* mine = lds + wave * S::kBytes;
  const uint8_t* my_s = mine + S::kS;
  auto compute = [&](uint32_t ok_all, int64_t j0) {
    f32x4 s[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
    for (int sg = 0; sg < seg_count(DK); ++sg) {
      const int W = seg_width(DK, sg), at = seg_at(DK, sg);
      const int block = (at + g * (W / 4)) / 32;
      const float e[2] = {scale_of<0>(my_s[block * 32 + col]), scale_of<0>(my_s[block * 32 + 16 + col])};
      uint32_t kw[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint8_t* from = mine + t * 8 * DK + 8 * at + lane * (W / 8);
        if (W == 128) {
          const uint4 x = *reinterpret_cast<const uint4*>(from);
          kw[t][0] = x.x; kw[t][1] = x.y; kw[t][2] = x.z; kw[t][3] = x.w;
        } else if (W == 64) {
          const uint2 x = *reinterpret_cast<const uint2*>(from);
          kw[t][0] = x.x; kw[t][1] = x.y;
        } else {
          kw[t][0] = *reinterpret_cast<const uint32_t*>(from);
        }
      }
#pragma unroll
      for (int j = 0; j < W / 32; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t x = kw[t][j];
          const u32x4 k = {cvt2<0>(x, e[t]), cvt2<1>(x, e[t]), cvt2<2>(x, e[t]), cvt2<3>(x, e[t])};
#pragma unroll
          for (int p = 0; p < NP; ++p) s[t] = mfma(k, q[at / 32 + j][p], s[t]);
        }
    }
    float p[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) p[r] = s[r >> 2][r & 3];
    const int32_t rest = my_limit - static_cast<int32_t>(j0);
    const uint32_t counts = !MANY ? ok_all : rest >= kTile ? ~0u : rest <= 0 ? 0u : (1u << rest) - 1;
    if (MANY ? __builtin_amdgcn_ballot_w64(counts != ~0u) != 0 : counts != ~0u) {
      const uint32_t ok = counts >> (4 * g);
#pragma unroll
      for (int r = 0; r < 8; ++r) p[r] = (ok >> ((r >> 2) * 16 + (r & 3))) & 1u ? p[r] : -INFINITY;
      // A value that is NaN meets p = 0 in the rows that do not see it: such blocks
      // become zeros here, and NaN the sums of the rows that do.
      if constexpr (MANY) {
#pragma unroll
        for (int bl = 0; bl < DV / 32; ++bl) {
          uint8_t* at = mine + S::kS + (DK / 32 + bl) * 32 + (lane & 31);
          const bool nan = *at == 255;
          const uint32_t bad = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(nan));
          if (bad == 0) continue;
          if (nan) *at = 0;
          if ((bad & counts) == 0) continue;
#pragma unroll
          for (int sg = 0; sg < seg_count(DV); ++sg)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if ((seg_at(DV, sg) + (4 * g + r) * (seg_width(DV, sg) / 16)) / 32 == bl)
#pragma unroll
                for (int i2 = 0; i2 < seg_width(DV, sg) / 16; ++i2) o[seg_at(DV, sg) / 16 + i2][r] = __builtin_nanf("");
        }
        wave_lds_order();
      }
    }
    if (a.logits && (SIDE ? piece == 0 : used)) {
      float* to = a.logits + my_head * a.stride + j0 + 4 * g;
      *reinterpret_cast<float4*>(to) = make_float4(p[0] * to2, p[1] * to2, p[2] * to2, p[3] * to2);
      *reinterpret_cast<float4*>(to + 16) = make_float4(p[4] * to2, p[5] * to2, p[6] * to2, p[7] * to2);
    }
    // The maximum moves only when a logit passes it by kSlack: exponentials up to
    // 2^8 do no harm in fp32, and most tiles then leave the sums as they are.
    // (IEEE maxima, one instruction for three; a NaN moves nothing and is in p anyway.)
    auto max2 = [](float x, float y) { return __builtin_elementwise_maximum(x, y); };
    const float top = to2 * max2(max2(max2(p[0], p[1]), max2(p[2], p[3])), max2(max2(p[4], p[5]), max2(p[6], p[7])));
    if (__builtin_amdgcn_ballot_w64(top > m + kSlack)) {
      const float next = fmaxf(m, max_xor32(max_xor16(top)));
      const float old = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - next);
      m = next;
      l *= old;
#pragma unroll
      for (int i2 = 0; i2 < NO; ++i2) o[i2] *= old;
    }
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      p[r] = __builtin_amdgcn_exp2f(fmaf(p[r], to2, -ref));
      l += p[r];
    }
    constexpr int NX = SIDE ? 1 : 3;
    u32x4 x[NX];
    if constexpr (SIDE) {
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        p[r] -= __uint_as_float(__float_as_uint(p[r]) & mask1);
        p[r] -= __uint_as_float(__float_as_uint(p[r]) & mask2);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) x[0][j] = pack_hi(p[2 * j], p[2 * j + 1]);
    } else {
#pragma unroll
      for (int k = 0; k < 3; ++k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[k][j] = pack_hi(p[2 * j], p[2 * j + 1]);
#pragma unroll
        for (int r = 0; r < 8; ++r) p[r] -= hi16(p[r]);
      }
    }
    int out = 0;
#pragma unroll
    for (int sg = 0; sg < seg_count(DV); ++sg) {
      const int W = seg_width(DV, sg), at = seg_at(DV, sg);
      uint32_t v[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const uint8_t* from = mine + S::kV + (r >> 2) * 8 * DV + 8 * at + ((r & 3) * 4 + g) * (W / 2) + col * (W / 32);
        v[r] = W == 128 ? *reinterpret_cast<const uint32_t*>(from)
               : W == 64 ? *reinterpret_cast<const uint16_t*>(from) : *from;
      }
      const uint8_t* sv = my_s + (DK / 32 + (at + col * (W / 16)) / 32) * 32 + 4 * g;
      const uint32_t e0 = *reinterpret_cast<const uint32_t*>(sv), e1 = *reinterpret_cast<const uint32_t*>(sv + 16);
      const float e[8] = {scale_of<0>(e0), scale_of<1>(e0), scale_of<2>(e0), scale_of<3>(e0),
                          scale_of<0>(e1), scale_of<1>(e1), scale_of<2>(e1), scale_of<3>(e1)};
#pragma unroll
      for (int pr = 0; pr < 4; ++pr) {
        if (pr >= W / 32) break;
        uint32_t y[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
          y[r] = pr == 0 ? cvt2<0>(v[r], e[r]) : pr == 1 ? cvt2<1>(v[r], e[r]) : pr == 2 ? cvt2<2>(v[r], e[r]) : cvt2<3>(v[r], e[r]);
        u32x4 lo, hi;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          lo[j] = __builtin_amdgcn_perm(y[2 * j + 1], y[2 * j], 0x05040100u);
          hi[j] = __builtin_amdgcn_perm(y[2 * j + 1], y[2 * j], 0x07060302u);
        }
#pragma unroll
        for (int k = 0; k < NX; ++k) {
          o[out] = mfma(lo, x[k], o[out]);
          o[out + 1] = mfma(hi, x[k], o[out + 1]);
        }
        out += 2;
      }
    }
  };

  if (j < j_end) {
    if (LISTED) off = entry(j + step);
    for (; j < j_end; j += step) {
      const uint32_t ok_all = MANY ? 0u : f.ok;
      wave_lds_order();
      stage<DK, DV>(f, mine);
      wave_lds_order();
      if (j + step < j_end) {
        load(f, j + step, off);
        if (LISTED) off = entry(j + 2 * step);
      }
      compute(ok_all, j);
    }
  }

  // Join the waves (and the pieces of p).
  __syncthreads();  // the sums lie where the stages were
  l = sum_xor32(sum_xor16(l));
  if (g == 0) {
    sum_m[wave][col] = m;
    sum_l[wave][col] = l;
  }
  if (col < (SIDE ? 3 * rows : rows)) {
    float* to = sum_o[wave][col];
#pragma unroll
    for (int sg = 0; sg < seg_count(DV); ++sg) {
      const int W = seg_width(DV, sg), at = seg_at(DV, sg);
#pragma unroll
      for (int r = 0; r < 4; ++r) {  // W / 16 columns from at + (4g + r) * W / 16 on
        float* row_at = to + at + (4 * g + r) * (W / 16);
        const f32x4* x = o + at / 16;
        if (W >= 64) {
          *reinterpret_cast<float4*>(row_at) = make_float4(x[0][r], x[1][r], x[2][r], x[3][r]);
          if (W == 128) *reinterpret_cast<float4*>(row_at + 4) = make_float4(x[4][r], x[5][r], x[6][r], x[7][r]);
        } else {
          *reinterpret_cast<float2*>(row_at) = make_float2(x[0][r], x[1][r]);
        }
      }
    }
  }
  __syncthreads();
  constexpr int kQuads = DV / 4;
  for (uint32_t e = threadIdx.x; e < static_cast<uint32_t>(a.heads * rows * kQuads); e += kNT) {
    const uint32_t hr = e / kQuads, d = e % kQuads * 4, hd = hr / rows, rw = hr % rows;
    float top = -INFINITY;
    for (int w = hd; w < kWaves; w += a.heads) top = fmaxf(top, sum_m[w][rw]);
    const float ref = top == -INFINITY ? 0.0f : top;
    float total = 0.0f;
    float4 x = {0, 0, 0, 0};
    for (int w = hd; w < kWaves; w += a.heads) {
      const float f = __builtin_amdgcn_exp2f(sum_m[w][rw] - ref);
      total += f * sum_l[w][rw];
      float4 y = *reinterpret_cast<const float4*>(&sum_o[w][rw][d]);
      if constexpr (SIDE) {  // the pieces, the small ones first
        const float4 y1 = *reinterpret_cast<const float4*>(&sum_o[w][rw + rows][d]);
        const float4 y2 = *reinterpret_cast<const float4*>(&sum_o[w][rw + 2 * rows][d]);
        y.x += y1.x + y2.x; y.y += y1.y + y2.y; y.z += y1.z + y2.z; y.w += y1.w + y2.w;
      }
      x.x += f * y.x; x.y += f * y.y; x.z += f * y.z; x.w += f * y.w;
    }
    const int64_t h = head_of(hk0 + hd, rt * 16 + rw);
    if (a.splits > 1) {
      *reinterpret_cast<float4*>(a.part + (h * a.splits + split) * DV + d) = x;
    } else {  // 0 / 0 where no logit is above -inf
      *reinterpret_cast<float4*>(a.out + h * DV + d) = make_float4(x.x / total, x.y / total, x.z / total, x.w / total);
    }
    if (d == 0 && a.ml) a.ml[h * a.splits + split] = make_float2(top, total);
  }
}

// One query head's maximum (0 where it is -inf) and sum over its splits, by 8 or 64 lanes.
// (A split without slots adds kNoSum * 2^-inf.)
template <int LANES>
__device__ __forceinline__ float2 join_ml(const float2* ml, int splits) {
  float top = -INFINITY, total = 0.0f;
#pragma unroll 4
  for (int s = threadIdx.x % LANES; s < splits; s += LANES) {
    const float2 x = ml[s];
    const float most = fmaxf(top, x.x), ref = most == -INFINITY ? 0.0f : most;
    total = total * __builtin_amdgcn_exp2f(top - ref) + x.y * __builtin_amdgcn_exp2f(x.x - ref);
    top = most;
  }
  float most = top;
  most = fmaxf(most, dpp_partner<1>(most));
  most = fmaxf(most, dpp_partner<2>(most));
  most = fmaxf(most, dpp_partner<4>(most));
  if (LANES == 64) most = max_xor32(max_xor16(fmaxf(most, dpp_partner<8>(most))));
  const float ref = most == -INFINITY ? 0.0f : most;
  total *= __builtin_amdgcn_exp2f(top - ref);
  total += dpp_partner<1>(total);
  total += dpp_partner<2>(total);
  total += dpp_partner<4>(total);
  if (LANES == 64) total = sum_xor32(sum_xor16(total + dpp_partner<8>(total)));
  return make_float2(ref, total);
}

constexpr int kMaxSplits = 512;  // what a joining block keeps factors of

// The first `joins` blocks join the splits of a.join_cols columns of a query head each
// (joins = 0: there is one split, or they are joined already); the others add query t's
// probabilities onto the weights of kNT slots of a sequence.  t < 0: of all
// queries, a slot having one thread.  Else one query's, listed ones: two queries
// never add to one slot at the same time, and a slot that one query lists twice
// takes the same addend twice, so that the sums have one order.
__global__ __launch_bounds__(kNT) void finish_kernel(AttnArgs a, int64_t joins, int t, int64_t per_b) {
  __shared__ float2 head[1024];
  __shared__ float4 sums[kNT];
  __shared__ float factor[kMaxSplits];
  if (blockIdx.x < joins) {
    const uint32_t cols = a.join_cols, parts = a.c.DV / cols, h = blockIdx.x / parts, d0 = blockIdx.x % parts * cols;
    const float2* ml = a.ml + static_cast<int64_t>(h) * a.splits;
    const float2 all = join_ml<64>(ml, a.splits);
    for (int s = threadIdx.x; s < a.splits; s += kNT) {
      const float2 x = ml[s];
      factor[s] = x.y == kNoSum ? kNoSum : __builtin_amdgcn_exp2f(x.x - all.x);
    }
    __syncthreads();
    // groups of threads take the splits in turn, a thread 4 columns
    const uint32_t quads = cols / 4, groups = kNT / quads, quad = threadIdx.x % quads, group = threadIdx.x / quads;
    const float* part = a.part + static_cast<int64_t>(h) * a.splits * a.c.DV + d0 + quad * 4;
    float4 x = {0, 0, 0, 0};
#pragma unroll 4
    for (int s = group; s < a.splits && group < groups; s += groups) {
      const float f = factor[s];
      if (f == kNoSum) continue;  // such a block has left none; a factor of 0 keeps a NaN one
      const float4 v = *reinterpret_cast<const float4*>(part + static_cast<int64_t>(s) * a.c.DV);
      x.x += f * v.x; x.y += f * v.y; x.z += f * v.z; x.w += f * v.w;
    }
    sums[threadIdx.x] = x;
    __syncthreads();
    if (threadIdx.x < cols) {
      float y = 0.0f;
      for (uint32_t s = 0; s < min(groups, static_cast<uint32_t>(a.splits)); ++s)
        y += reinterpret_cast<const float*>(sums + s * quads)[threadIdx.x];
      a.out[static_cast<int64_t>(h) * a.c.DV + d0 + threadIdx.x] = y / all.y;  // 0 / 0 where no logit is above -inf
    }
    return;
  }
  const uint32_t blk = blockIdx.x - static_cast<uint32_t>(joins), b = blk / static_cast<uint32_t>(per_b);
  const int64_t j = static_cast<int64_t>(blk % static_cast<uint32_t>(per_b)) * kNT + threadIdx.x;
  float* weight = a.c.weight + b * a.c.S;
  float sum = 0.0f;
  int32_t slot = -1;
  for (int tt = t < 0 ? 0 : t; tt < (t < 0 ? a.Tq : t + 1); ++tt) {
    const int64_t bt = static_cast<int64_t>(b) * a.Tq + tt;
    const int32_t seen = kv4_visible(a.c.length, a.count, b, a.c.S, tt, a.Tq);
    __syncthreads();
    for (int h0 = 0; h0 < a.HQ; h0 += kNT / 8) {
      const int h = h0 + threadIdx.x / 8;
      const float2 x = join_ml<8>(a.ml + (bt * a.HQ + min(h, a.HQ - 1)) * a.splits, a.splits);
      if (h < a.HQ && threadIdx.x % 8 == 0) head[h] = make_float2(x.x, 1.0f / x.y);
    }
    __syncthreads();
    const int32_t s = j >= a.n ? -1 : a.slots ? a.slots[bt * a.n + j] : static_cast<int32_t>(j);
    if (s < 0 || s >= seen) continue;
    slot = s;
    const float* logits = a.logits + bt * a.HQ * a.stride + j;
#pragma unroll 8
    for (int h = 0; h < a.HQ; ++h)
      sum += __builtin_amdgcn_exp2f(logits[h * a.stride] - head[h].x) * head[h].y;
  }
  if (slot < 0) return;
  if (a.slots) atomicAdd(weight + slot, sum);
  else weight[slot] += sum;
}

struct Plan {
  int splits, row_tiles, heads;
  bool side, many;
  int64_t ml, part, logits, total, stride;  // byte offsets; floats a row
};

// pieces: of Q (resident); the most splits come of the fewest.
Plan plan_of(const Kv4& c, int64_t Tq, int HQ, bool listed, int64_t n, bool accumulate, int pieces) {
  Plan p;
  const int64_t G = HQ / c.HKV, tiles = (G + 15) / 16;  // of 16 rows, one token's
  // Up to 8 turns of four waves on one head's slots cost less than the launch that
  // would join splits (255 listed slots, 8 heads of 64, fp32, 4 sequences: 11.3 us
  // with it, 8.8 without).  (Whether weights are accumulated does not enter: it
  // changes no bit of the output.)
  const bool alone = n <= 8 * kTile * kWaves;
  const int cus = device_cus() > 0 ? device_cus() : 256;
  const bool few = c.B * Tq * c.HKV * tiles <= 4 * cus;
  // Tokens that attend to the same slots, all but the last few, share a block's rows
  // where that leaves fewer tiles of rows (us with / without: 16 x 16384 slots of 8
  // heads of 128, groups of 4, 2 tokens 59 / 80, 4 tokens 62 / 137; 2 x 4096 slots, 64
  // tokens 42 / 83), unless there are few blocks of one turn anyway (4 x 500 slots of
  // 8 heads of 64 in fp32, 2 tokens 11.3 / 8.8).
  p.many = !listed && (Tq * G + 15) / 16 < Tq * tiles && !(alone && few);
  const int64_t rows = p.many ? Tq * G : G, groups = p.many ? c.B : c.B * Tq;
  p.side = rows <= 5;
  p.row_tiles = static_cast<int>((rows + 15) / 16);
  // Four neighbouring heads a block read whole rows of the cache together; few blocks
  // of one that have no splits finish sooner (us with four / one: 64 x 1024 slots of
  // 8 heads of 128 19.6 / 16.6, 256 x 512 of 8 of 64 17.3 / 19.6), and so does it where
  // the rows are gathered (2048 listed slots of 32 x 4 heads of 128 19.5 / 18.7, 256 x 4
  // of 64 55.5 / 41.3, 16 x 4 with groups of 16 22.4 / 16.6; of 64 x 8 49 / 53).
  p.heads = listed || (alone && few) ? 1 : c.HKV % 4 == 0 ? 4 : c.HKV % 2 == 0 ? 2 : 1;
  const int64_t blocks = groups * (c.HKV / p.heads) * p.row_tiles;
  const int unit = kTile * (kWaves / p.heads);  // slots that a block takes at once
  const int64_t steps = n > 0 ? (n + unit - 1) / unit : 1;
  // Two blocks a compute unit: 1, 2, 4 and 8 measured 108, 94, 93 and 109 us for
  // 16 x 32768 slots, 16.1, 12.9, 14.4 and 15.1 us for 16 x 4096.  One where a second
  // would wait (4 x 8192 slots, 16 heads on 4 of 256 in fp32: 24.4 us with two, 17.9).
  const int at_once = resident(pieces, c.DK, c.DV, p.side) < 2 ? 1 : 2;
  int64_t splits = alone || blocks < 1 ? 1 : (at_once * cus + blocks - 1) / blocks;
  splits = splits > steps ? steps : splits;
  splits = splits > kMaxSplits ? kMaxSplits : splits;
  p.splits = static_cast<int>(splits);
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  const int64_t heads = c.B * Tq * HQ;
  p.stride = (n + kTile - 1) / kTile * kTile;
  p.ml = 0;  // one split without weights needs nothing
  p.part = p.splits > 1 || accumulate ? up(heads * p.splits * 8) : 0;
  p.logits = p.part + (p.splits > 1 ? up(heads * p.splits * c.DV * 4) : 0);
  p.total = p.logits + (accumulate ? up(heads * p.stride * 4) : 0);
  return p;
}

template <typename Tag, int NP, int DK, int DV>
hipError_t launch_dims(const AttnArgs& a, const Plan& p, int64_t blocks, hipStream_t stream) {
  const uint32_t grid = static_cast<uint32_t>(blocks);
  auto run = [&](auto side) {
    constexpr bool SIDE = decltype(side)::value;
    if (a.slots) attn_kernel<Tag, NP, DK, DV, SIDE, kListed><<<grid, kNT, 0, stream>>>(a);
    else if (p.many) attn_kernel<Tag, NP, DK, DV, SIDE, kTokens><<<grid, kNT, 0, stream>>>(a);
    else attn_kernel<Tag, NP, DK, DV, SIDE, kOne><<<grid, kNT, 0, stream>>>(a);
  };
  if (p.side) run(std::true_type{});
  else run(std::false_type{});
  return hipGetLastError();
}

template <typename Tag, int NP>
hipError_t launch_type(const AttnArgs& a, const Plan& p, int64_t blocks, hipStream_t stream) {
  if (a.c.DK != a.c.DV) return launch_dims<Tag, NP, 192, 128>(a, p, blocks, stream);
  switch (a.c.DK) {
    case 32: return launch_dims<Tag, NP, 32, 32>(a, p, blocks, stream);
    case 64: return launch_dims<Tag, NP, 64, 64>(a, p, blocks, stream);
    case 96: return launch_dims<Tag, NP, 96, 96>(a, p, blocks, stream);
    case 128: return launch_dims<Tag, NP, 128, 128>(a, p, blocks, stream);
    case 192: return launch_dims<Tag, NP, 192, 192>(a, p, blocks, stream);
    default: return launch_dims<Tag, NP, 256, 256>(a, p, blocks, stream);
  }
}

}  // namespace

bool kv4_attn_supported(int DK, int DV) {
  if (DK == 192 && DV == 128) return true;
  return DK == DV && (DK == 32 || DK == 64 || DK == 96 || DK == 128 || DK == 192 || DK == 256);
}

int64_t kv4_attn_workspace(const Kv4& c, int64_t Tq, int HQ, bool listed, int64_t n, bool accumulate) {
  return plan_of(c, Tq, HQ, listed, n, accumulate, 1).total;
}

hipError_t launch_kv4_attn(const Kv4& c, const void* Q, int dtype, const int32_t* slots,
                           const int32_t* count, int64_t Tq, int HQ, int64_t n, bool accumulate,
                           float scale, float* out, void* ws, hipStream_t stream) {
  const Plan p = plan_of(c, Tq, HQ, slots != nullptr, n, accumulate, dtype == 0 ? 3 : dtype == 1 ? 1 : 2);
  char* base = static_cast<char*>(ws);
  AttnArgs a;
  a.c = c;
  a.Q = Q;
  a.slots = slots;
  a.count = count;
  a.Tq = static_cast<int>(Tq);
  a.HQ = HQ;
  a.G = HQ / c.HKV;
  a.row_tiles = p.row_tiles;
  a.heads = p.heads;
  a.n = n;
  a.stride = p.stride;
  a.splits = p.splits;
  // many splits are joined by more blocks (1 x 32768 slots, 256 splits of 8 heads:
  // 27.9 us by the head, 16.8 by 32 columns; 128 heads of 16 sequences, 4 splits:
  // 38.6 and 44.4)
  a.join_cols = p.splits > 32 ? 32 : c.DV;
  a.scale = scale;
  a.out = out;
  a.ml = p.total > 0 ? reinterpret_cast<float2*>(base + p.ml) : nullptr;
  a.part = reinterpret_cast<float*>(base + p.part);
  a.logits = accumulate ? reinterpret_cast<float*>(base + p.logits) : nullptr;
  const int64_t chunks = ((p.many ? c.B : c.B * Tq) * p.splits + 7) / 8 * 8;
  const int64_t blocks = chunks * (c.HKV / p.heads) * p.row_tiles;
  hipError_t e = dtype == 0   ? launch_type<F32, 3>(a, p, blocks, stream)
                 : dtype == 1 ? launch_type<BF16, 1>(a, p, blocks, stream)
                              : launch_type<F16, 2>(a, p, blocks, stream);
  if (e != hipSuccess) return e;
  int64_t joins = p.splits > 1 ? c.B * Tq * HQ * (c.DV / a.join_cols) : 0;
  const int64_t per_b = accumulate ? (n + kNT - 1) / kNT : 0;
  for (int t = slots ? 0 : -1; t < (slots && accumulate ? a.Tq : slots ? 1 : 0); ++t) {
    const uint32_t grid = static_cast<uint32_t>(joins + per_b * c.B);
    if (grid > 0) finish_kernel<<<grid, kNT, 0, stream>>>(a, joins, t, per_b);
    joins = 0;
  }
  return hipGetLastError();
}

}  // namespace dsa
