// kv8_attn.hip -- attention of each sequence's last tokens over the paged 8-bit
// cache (gfx950).
//
//   O[b,t,h,:] = sum_s p_s V[b,s,h/G,:],  p = softmax_s(<Q[b,t,h], K[b,s,h/G]> scale)
// over the slots s that token t sees: s <= its own, and with a window s > its own -
// window or s < sinks.
//
// A wave takes 64 slots of one K/V head and 16 rows (the group's heads of the tokens,
// token by token) at a time, on 16x16x32 f16 products:
//   S^T = K . Q^T    A = K's codes, which f16 holds exactly; B = Q
//   O^T = V^T . P^T  A = V's codes as they lie in the cache; B = P straight from S^T's
//                    registers (lane group g holds tokens 16j + 4g + i of each row)
// The block's scales are powers of two: K's goes into the factor of the logits, V's
// onto the sums of each 64 slots, in fp32.  So no value of the cache is rounded.  Rows
// of Q are scaled by a power of two into f16's range and enter as one f16 piece
// (16-bit types) or two (fp32, 23 bits); p likewise.
#include <algorithm>

#include "dsa_launch.h"
#include "kv8.h"

namespace dsa {
namespace {

constexpr int kNT = 256, kWaves = 4, kRows = 16;

struct AttnArgs {
  Kv8 c;
  const void* Q;
  const int32_t* count;
  int Tq, HQ, G;
  int row_tiles, splits;
  int64_t n;       // slots that count
  int64_t window;  // 0: all
  int64_t sinks;
  float scale_log2;
  void* out;
  float* part;  // [B*Tq*HQ][splits][DV]
  float2* ml;   // [B*Tq*HQ][splits]: maximum (log2) and sum
};

// p is held as 2^(kUp + logit - maximum): what is small beside the largest then stays
// a normal f16 down to 2^-(14 + kUp).  The maximum moves when a logit passes it by
// kSlack, so p stays below 2^15.
constexpr float kUp = 10.0f, kSlack = 5.0f;

__device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
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

template <typename Tag, int DK, int DV>
__global__ __launch_bounds__(kNT) void attn_kernel(AttnArgs a) {
  using raw = typename Tag::raw;
  constexpr int NP = Tag::kBytes == 4 ? 2 : 1;          // f16 pieces of Q and of p
  constexpr int NJ = DK / 64, HALF = DK % 64 != 0;      // 16-byte runs of a K row a lane, and 8-byte ones
  constexpr int NKS = 2 * NJ + HALF, NDT = DV / 16;
  __shared__ float sum_m[kWaves][kRows], sum_l[kWaves][kRows];
  __shared__ __align__(16) float sum_o[kWaves][kRows][DV];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id();
  const int g = lane >> 4, col = lane & 15;
  // Blocks of one chunk of slots and their row tiles go to one XCD (block i starts on XCD i % 8).
  const uint32_t chunk = blockIdx.x % 8 + blockIdx.x / (8 * a.row_tiles) * 8, rt = blockIdx.x / 8 % a.row_tiles;
  const int split = chunk % a.splits;
  const uint32_t bh = chunk / a.splits;
  const int h = bh % a.c.HKV;
  const int64_t b = bh / a.c.HKV;
  if (b >= a.c.B) return;

  const int rows = a.Tq * a.G;
  const int32_t len = kv8_length(a.c, b);
  const int32_t many = a.count ? max(0, min(a.count[b], a.Tq)) : a.Tq;
  const int first_row = rt * kRows, last_row = min(first_row + kRows, rows) - 1;
  const int row = min(first_row + col, rows - 1), t = row / a.G;
  const Seen mine = seen_by(a, len, many, t);
  // of the tile's tokens that are any: the earliest and the latest
  const int t_lo = first_row / a.G, t_hi = min(last_row / a.G, many - 1);
  const Seen lo = seen_by(a, len, many, t_lo), hi = seen_by(a, len, many, t_hi);
  const int32_t sinks = static_cast<int32_t>(a.sinks);  // at most the slots, 2^31 - 256
  int32_t near = 0, nsink = 0, total = 0;
  if (t_hi >= t_lo && hi.end > 0) {
    near = lo.low / kBlk;
    nsink = min((min(sinks, hi.end) + kBlk - 1) / kBlk, near);
    total = nsink + max(0, (hi.end + kBlk - 1) / kBlk - near);
  }

  // Q: lane holds row `col`, dims 64j + 16g .. +15 (the products' k-slots in the order of K's runs).
  u32x4 q[NP][NKS];
  float unscale = 1.0f;
  {
    const raw* src = static_cast<const raw*>(a.Q) + ((b * a.Tq + t) * a.HQ + h * a.G + row % a.G) * DK;
    float x[NKS][8];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < NKS; ++k) {
      const int d = k < 2 * NJ ? 64 * (k / 2) + 16 * g + 8 * (k % 2) : 64 * NJ + 8 * g;
      load_cvt<Tag, 8>(src + d, x[k]);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[k][i]) & 0x7fffffffu);
    }
    top = max_xor32_u32(max_xor16_u32(top));
    // the row's largest into [2^14, 2^15); a row that is not finite stays so
    const int sh = top >= 0x7f800000u || top == 0 ? 0 : min(141 - static_cast<int>(top >> 23), 126);
    const float f = pow2f(sh);
    unscale = pow2f(-sh);
#pragma unroll
    for (int k = 0; k < NKS; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float u = x[k][2 * i] * f, v = x[k][2 * i + 1] * f;
        if constexpr (NP == 2) {
          uint32_t hi16, lo16;
          split_pair(u, v, hi16, lo16);
          q[0][k][i] = hi16;
          q[1][k][i] = lo16;
        } else {
          q[0][k][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{u, v}), f16x2));
        }
      }
    if (top >= 0x7f800000u) unscale = __builtin_nanf("");  // every logit of such a row is Inf or NaN
  }

  float m = -INFINITY, l = 0.0f;
  f32x4 o[NDT];
#pragma unroll
  for (int d = 0; d < NDT; ++d) o[d] = f32x4{0, 0, 0, 0};

  const int32_t step = a.splits * kWaves;
  for (int32_t v = split * kWaves + wave; v < total; v += step) {
    const int32_t blk = v < nsink ? v : near + v - nsink;
    const int64_t at = kv8_block(a.c, b, blk, h);
    if (at < 0) continue;  // uniform; a page that is none holds nothing
    const uint8_t* base = a.c.codes + at * a.c.block_bytes();
    const uint32_t sc = *reinterpret_cast<const uint16_t*>(a.c.scales + at * 2);
    u32x4 kr[4][NJ > 0 ? NJ : 1];
    uint2 kh[4];
    u32x4 vr[NDT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint8_t* p = base + (16 * j + col) * DK;
#pragma unroll
      for (int i = 0; i < NJ; ++i) kr[j][i] = *reinterpret_cast<const u32x4*>(p + 64 * i + 16 * g);
      if (HALF) kh[j] = *reinterpret_cast<const uint2*>(p + 64 * NJ + 8 * g);
    }
#pragma unroll
    for (int d = 0; d < NDT; ++d)
      vr[d] = *reinterpret_cast<const u32x4*>(base + kBlk * DK + (16 * d + col) * kBlk + 16 * g);

    f32x4 st[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      st[j] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < NKS; ++k) {
        const u32x4 x = k < 2 * NJ ? widen8(kr[j][k / 2][2 * (k % 2)], kr[j][k / 2][2 * (k % 2) + 1]) : widen8(kh[j].x, kh[j].y);
#pragma unroll
        for (int p = NP - 1; p >= 0; --p) st[j] = mfma(x, q[p][k], st[j]);
      }
    }

    const float f = a.scale_log2 * __uint_as_float((sc & 255u) << 23) * unscale;
    const int32_t s0 = blk * kBlk;
    const bool inner = s0 + kBlk <= lo.end && (s0 >= hi.low || s0 + kBlk <= sinks);
    float top = -INFINITY;
    uint32_t ok = 0xffffu;  // bit 4j + i: slot s0 + 16j + 4g + i is seen
    if (!inner) {
      ok = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int32_t s = s0 + (e >> 2) * 16 + 4 * g + (e & 3);
        if (s < mine.end && (s >= mine.low || s < sinks)) ok |= 1u << e;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = st[j][i] * f;
        st[j][i] = ok >> (4 * j + i) & 1u ? x : -INFINITY;
        top = fmaxf(top, st[j][i]);
      }
    top = max_xor32(max_xor16(top));
    if (ballot(top > m + kSlack)) {
      const float next = fmaxf(m, top);
      const float fall = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - next);
      m = next;
      l *= fall;
#pragma unroll
      for (int d = 0; d < NDT; ++d) o[d] *= fall;
    }
    const float ref = m == -INFINITY ? 0.0f : m - kUp;
    u32x4 p[NP][2];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const float x = __builtin_amdgcn_exp2f(st[j][i] - ref), y = __builtin_amdgcn_exp2f(st[j][i + 1] - ref);
        l += x + y;
        const int e = 2 * (j & 1) + i / 2;
        if constexpr (NP == 2) {
          uint32_t hi16, lo16;
          split_pair(x, y, hi16, lo16);
          p[0][j >> 1][e] = hi16;
          p[1][j >> 1][e] = lo16;
        } else {
          p[0][j >> 1][e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), f16x2));
        }
      }
    // A NaN in V is for the rows that see its slot alone: where some do not, it goes
    // into their sums by hand and stays out of the product.
    if (!inner) {
      uint32_t any = 0;
#pragma unroll
      for (int d = 0; d < NDT; ++d)
#pragma unroll
        for (int w = 0; w < 4; ++w) any |= nan_bytes(vr[d][w]);
      if (ballot(any != 0)) {
        u32x4 see[2];  // 1 where seen, as p lies
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            see[j >> 1][2 * (j & 1) + i] =
                (ok >> (4 * j + 2 * i) & 1u ? 0x3c00u : 0u) | (ok >> (4 * j + 2 * i + 1) & 1u ? 0x3c000000u : 0u);
#pragma unroll
        for (int d = 0; d < NDT; ++d) {
          u32x4 is;  // e4m3's 1 where a NaN is, 0 elsewhere
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t bad = nan_bytes(vr[d][w]) >> 7;
            is[w] = bad * 0x38u;
            vr[d][w] &= ~(bad * 0xffu);
          }
          f32x4 hits = mfma(widen8(is[0], is[1]), see[0], f32x4{0, 0, 0, 0});
          hits = mfma(widen8(is[2], is[3]), see[1], hits);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (hits[r] > 0.0f) o[d][r] = __builtin_nanf("");
        }
      }
    }
    const float vs = __uint_as_float((sc >> 8) << 23);
#pragma unroll
    for (int d = 0; d < NDT; ++d) {
      const u32x4 x = widen8(vr[d][0], vr[d][1]), y = widen8(vr[d][2], vr[d][3]);
      f32x4 acc{0, 0, 0, 0};
#pragma unroll
      for (int k = NP - 1; k >= 0; --k) {
        acc = mfma(x, p[k][0], acc);
        acc = mfma(y, p[k][1], acc);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) o[d][r] = fmaf(acc[r], vs, o[d][r]);
    }
  }

  // Join the waves.
  l = sum_xor32(sum_xor16(l));
  if (t >= many) {  // no token: sees nothing
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int d = 0; d < NDT; ++d) o[d] = f32x4{0, 0, 0, 0};
  }
  if (g == 0) {
    sum_m[wave][col] = m;
    sum_l[wave][col] = l;
  }
#pragma unroll
  for (int d = 0; d < NDT; ++d)
    *reinterpret_cast<float4*>(&sum_o[wave][col][16 * d + 4 * g]) = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
  __syncthreads();
  constexpr int kQuads = DV / 4;
  for (int e = threadIdx.x; e < (last_row - first_row + 1) * kQuads; e += kNT) {
    const int r = e / kQuads, d = e % kQuads * 4;
    float top = sum_m[0][r];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, sum_m[w][r]);
    const float ref = top == -INFINITY ? 0.0f : top;
    float all = 0.0f;
    float4 x = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(sum_m[w][r] - ref);
      const float4 y = *reinterpret_cast<const float4*>(&sum_o[w][r][d]);
      all += f * sum_l[w][r];
      x.x += f * y.x; x.y += f * y.y; x.z += f * y.z; x.w += f * y.w;
    }
    const int rr = first_row + r;
    const int64_t hr = (b * a.Tq + rr / a.G) * a.HQ + h * a.G + rr % a.G;
    if (a.splits > 1) {
      *reinterpret_cast<float4*>(a.part + (hr * a.splits + split) * DV + d) = x;
      if (d == 0) a.ml[hr * a.splits + split] = make_float2(top, all);
    } else {  // 0 / 0 where nothing is seen
      raw* to = static_cast<raw*>(a.out) + hr * DV + d;
      const float inv = 1.0f / all;
      const f32x4 y{x.x * inv, x.y * inv, x.z * inv, x.w * inv};
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
  }
}

constexpr int kMaxSplits = 512;

// A block joins one row's splits.
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
    const float f = __builtin_amdgcn_exp2f(x.x - ref);
    factor[s] = f;
    all += f * x.y;
  }
  all = wave_sum(all);
  if ((threadIdx.x & 63) == 0) both[threadIdx.x >> 6].y = all;
  __syncthreads();
  all = both[0].y + both[1].y + both[2].y + both[3].y;
  if (threadIdx.x >= DV) return;
  float x = 0.0f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) x += factor[s] * part[(row * splits + s) * DV + threadIdx.x];
  x /= all;
  if constexpr (Tag::kBytes == 4) out[row * DV + threadIdx.x] = x;
  else if constexpr (__is_same(Tag, BF16)) out[row * DV + threadIdx.x] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
  else out[row * DV + threadIdx.x] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
}

struct Plan {
  int splits, row_tiles;
  int64_t ml, total;  // bytes
};

Plan plan_of(const Kv8& c, int64_t Tq, int HQ, int64_t n, int64_t window, int64_t sinks) {
  Plan p;
  p.row_tiles = static_cast<int>((Tq * (HQ / c.HKV) + kRows - 1) / kRows);
  int64_t most = (n + kBlk - 1) / kBlk;  // blocks that a row tile walks
  if (window > 0) {
    const int64_t near = (window + Tq - 1 + kBlk - 1) / kBlk + 1 + (sinks < n ? (sinks + kBlk - 1) / kBlk : most);
    most = near < most ? near : most;
  }
  const int64_t steps = most > kWaves ? (most + kWaves - 1) / kWaves : 1;
  const int64_t blocks = c.B * c.HKV * p.row_tiles;
  const int cus = device_cus() > 0 ? device_cus() : 256;
  int64_t splits = blocks < 1 ? 1 : (2 * cus + blocks - 1) / blocks;
  splits = splits > steps ? steps : splits;
  p.splits = static_cast<int>(splits > kMaxSplits ? kMaxSplits : splits);
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  const int64_t heads = c.B * Tq * HQ;
  p.ml = p.splits > 1 ? up(heads * p.splits * 8) : 0;
  p.total = p.ml + (p.splits > 1 ? up(heads * p.splits * c.DV * 4) : 0);
  return p;
}

template <typename Tag>
hipError_t launch_type(const AttnArgs& a, const Plan& p, hipStream_t stream) {
  const int64_t chunks = (a.c.B * a.c.HKV * p.splits + 7) / 8 * 8;
  const uint32_t grid = static_cast<uint32_t>(chunks * p.row_tiles);
  if (a.c.DK != a.c.DV) attn_kernel<Tag, 192, 128><<<grid, kNT, 0, stream>>>(a);
  else switch (a.c.DK) {
    case 32: attn_kernel<Tag, 32, 32><<<grid, kNT, 0, stream>>>(a); break;
    case 64: attn_kernel<Tag, 64, 64><<<grid, kNT, 0, stream>>>(a); break;
    case 96: attn_kernel<Tag, 96, 96><<<grid, kNT, 0, stream>>>(a); break;
    case 128: attn_kernel<Tag, 128, 128><<<grid, kNT, 0, stream>>>(a); break;
    case 192: attn_kernel<Tag, 192, 192><<<grid, kNT, 0, stream>>>(a); break;
    default: attn_kernel<Tag, 256, 256><<<grid, kNT, 0, stream>>>(a);
  }
  if (p.splits > 1)
    join_kernel<Tag><<<static_cast<uint32_t>(a.c.B * a.Tq * a.HQ), kNT, 0, stream>>>(
        a.part, a.ml, p.splits, a.c.DV, static_cast<typename Tag::raw*>(a.out));
  return hipGetLastError();
}

}  // namespace

bool kv8_supported(int DK, int DV) {
  if (DK == 192 && DV == 128) return true;
  return DK == DV && (DK == 32 || DK == 64 || DK == 96 || DK == 128 || DK == 192 || DK == 256);
}

int64_t kv8_attn_workspace(const Kv8& c, int64_t Tq, int HQ, int64_t n, int64_t window, int64_t sinks) {
  return plan_of(c, Tq, HQ, n, std::min(window, c.slots()), std::min(sinks, c.slots())).total;
}

hipError_t launch_kv8_attn(const Kv8& c, const void* Q, int dtype, const int32_t* count, int64_t Tq, int HQ,
                           int64_t n, int64_t window, int64_t sinks, float scale, void* out, void* ws,
                           hipStream_t stream) {
  window = std::min(window, c.slots());  // no token has more before it
  sinks = std::min(sinks, c.slots());
  const Plan p = plan_of(c, Tq, HQ, n, window, sinks);
  AttnArgs a;
  a.c = c;
  a.Q = Q;
  a.count = count;
  a.Tq = static_cast<int>(Tq);
  a.HQ = HQ;
  a.G = HQ / c.HKV;
  a.row_tiles = p.row_tiles;
  a.splits = p.splits;
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
