// kv8_cache.hip -- what goes into the paged 8-bit cache and comes back out of it
// (gfx950).
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

// Elements d0 .. d0+7 of the row at `p` (one head of one token), rotated by table row `at`.
template <typename Tag>
__device__ __forceinline__ void load_rotated(const typename Tag::raw* p, int d0, int R, bool pairs,
                                             const float* cos, const float* sin, int64_t at, float (&x)[8]) {
  load_cvt<Tag, 8>(p + d0, x);
  if (d0 >= R) return;
  const int half = R / 2;
  if (pairs) {
    float c[4], s[4];
    load_f32<4>(cos + at * half + d0 / 2, c);
    load_f32<4>(sin + at * half + d0 / 2, s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = turn_a(a, b, c[i], s[i]);
      x[2 * i + 1] = turn_b(a, b, c[i], s[i]);
    }
  } else {
    const bool low = d0 < half;
    const int j = low ? d0 : d0 - half;
    float y[8], c[8], s[8];
    load_cvt<Tag, 8>(p + (low ? d0 + half : d0 - half), y);
    load_f32<8>(cos + at * half + j, c);
    load_f32<8>(sin + at * half + j, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = low ? turn_a(x[i], y[i], c[i], s[i]) : turn_b(y[i], x[i], c[i], s[i]);
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
__device__ void update_counts(const Kv8& c, const Span& s, int64_t b) {
  __shared__ int32_t bad;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  const int shift = c.page_shift + 6;
  int32_t mine = 0;
  for (int64_t p = (s.have >> shift) + threadIdx.x; p << shift < s.end; p += kNT) {
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

// One block of threads takes one block of 64 slots of one head: rotates, finds the
// scales, encodes, writes.  Thread (r, ch) holds elements 8 ch .. 8 ch + 7 of tokens
// r, r + RP, ...
template <int D>
struct Tile {
  static constexpr int kChunks = D / 8, kRows = kNT / kChunks, kPasses = (kBlk + kRows - 1) / kRows;
};

template <typename Tag, int DK, int DV>
__global__ __launch_bounds__(kNT) void append_kernel(Kv8 c, Kv8Append a, int nblk, uint32_t kv_blocks, int update) {
  using raw = typename Tag::raw;
  using TK = Tile<DK>;
  using TV = Tile<DV>;
  constexpr int kRowBytes = 80;  // of a dimension's 64 codes in LDS
  __shared__ uint32_t tops[2][4];
  __shared__ __align__(16) uint8_t vt[DV * kRowBytes];
  const float* cos = a.cos;
  const float* sin = a.sin;
  const int64_t S = c.slots();

  if (blockIdx.x >= kv_blocks) {  // the queries, 8 elements a thread
    const int64_t items = c.B * a.T * a.HQ * TK::kChunks;
    const int64_t i = (blockIdx.x - kv_blocks) * static_cast<int64_t>(kNT) + threadIdx.x;
    if (i >= items) return;
    const int d0 = static_cast<int>(i % TK::kChunks) * 8;
    const int64_t row = i / TK::kChunks, h = row % a.HQ, bt = row / a.HQ, b = bt / a.T;
    const int64_t at = span_of(c, a, b).have + bt % a.T;
    float x[8];
    load_rotated<Tag>(static_cast<const raw*>(a.Q) + bt * a.ldq + h * DK, d0, a.R, a.pairs, cos, sin, min(at, S - 1), x);
    if (at >= S) {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = __builtin_nanf("");
    }
    store8<Tag>(static_cast<raw*>(a.Q_out) + row * DK + d0, x);
    return;
  }

  const int h = blockIdx.x % c.HKV;
  const uint32_t rest = blockIdx.x / c.HKV;
  const int64_t b = rest / nblk;
  const Span s = span_of(c, a, b);
  const int64_t blk = (s.have >> 6) + rest % nblk, first = blk * kBlk;
  // the call's tokens on this block: all, and those that are stored
  const int lo = static_cast<int>(max(s.have - first, int64_t{0}));
  const int all = static_cast<int>(min(s.have + a.T - first, int64_t{kBlk}));
  const int64_t at_block = first < s.end ? kv8_block(c, b, blk, h) : -1;
  const int hi = at_block >= 0 ? static_cast<int>(min(s.end - first, int64_t{kBlk})) : lo;
  uint8_t* const codes = c.codes + at_block * c.block_bytes();

  float k[TK::kPasses][8], v[TV::kPasses][8];
  uint32_t top_k = 0, top_v = 0;
  {
    const int ch = threadIdx.x % TK::kChunks, r0 = threadIdx.x / TK::kChunks;
    const raw* src = static_cast<const raw*>(a.K) + (b * a.T - s.have + first) * a.ldk + static_cast<int64_t>(h) * DK;
#pragma unroll
    for (int p = 0; p < TK::kPasses; ++p) {
      const int t = r0 + p * TK::kRows;
      if (r0 >= TK::kRows || t < lo || t >= all || (t >= hi && !a.K_out)) continue;
      load_rotated<Tag>(src + t * a.ldk, ch * 8, a.R, a.pairs, cos, sin, min(first + t, S - 1), k[p]);
      if (a.K_out) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = first + t < S ? k[p][i] : __builtin_nanf("");
        store8<Tag>(static_cast<raw*>(a.K_out) + ((b * a.T - s.have + first + t) * c.HKV + h) * DK + ch * 8, y);
      }
      if (t < hi) {
#pragma unroll
        for (int i = 0; i < 8; ++i) top_k = max(top_k, finite_bits(k[p][i]));
      }
    }
  }
  if (lo < hi) {  // the same for the whole block
    {
      const int ch = threadIdx.x % TV::kChunks, r0 = threadIdx.x / TV::kChunks;
      const raw* src = static_cast<const raw*>(a.V) + (b * a.T - s.have + first) * a.ldv + static_cast<int64_t>(h) * DV;
#pragma unroll
      for (int p = 0; p < TV::kPasses; ++p) {
        const int t = r0 + p * TV::kRows;
        if (r0 >= TV::kRows || t < lo || t >= hi) continue;
        load_cvt<Tag, 8>(src + t * a.ldv + ch * 8, v[p]);
#pragma unroll
        for (int i = 0; i < 8; ++i) top_v = max(top_v, finite_bits(v[p][i]));
      }
    }
    uint8_t* const scale_at = c.scales + at_block * 2;
    const uint32_t old_k = lo > 0 ? scale_at[0] : 0u, old_v = lo > 0 ? scale_at[1] : 0u;
    top_k = wave_max_bits(top_k);
    top_v = wave_max_bits(top_v);
    if ((threadIdx.x & 63) == 0) {
      tops[0][threadIdx.x >> 6] = top_k;
      tops[1][threadIdx.x >> 6] = top_v;
    }
    __syncthreads();  // the old scales have been read
    const uint32_t new_k = max(old_k, kv8_scale(max(max(tops[0][0], tops[0][1]), max(tops[0][2], tops[0][3]))));
    const uint32_t new_v = max(old_v, kv8_scale(max(max(tops[1][0], tops[1][1]), max(tops[1][2], tops[1][3]))));
    if (threadIdx.x == 0) {
      scale_at[0] = static_cast<uint8_t>(new_k);
      scale_at[1] = static_cast<uint8_t>(new_v);
    }
    // Held tokens whose block's scale grows are rounded again, to the new one.
    if (lo > 0 && new_k > old_k) {
      const float f = new_k - old_k > 40 ? 0.0f : __uint_as_float((127u + old_k - new_k) << 23);
      for (int i = threadIdx.x; i < lo * DK / 4; i += kNT) {
        uint32_t* w = reinterpret_cast<uint32_t*>(codes) + i;
        *w = rescale4(*w, f);
      }
    }
    if (lo > 0 && new_v > old_v) {
      const float f = new_v - old_v > 40 ? 0.0f : __uint_as_float((127u + old_v - new_v) << 23);
      for (int i = threadIdx.x; i < DV * kBlk / 4; i += kNT) {
        const int t = (i & 3) * 16 + ((i >> 2) & 3) * 4;  // word i of the rows: tokens t .. t + 3
        if (t >= lo) continue;
        uint32_t* w = reinterpret_cast<uint32_t*>(codes + kBlk * DK) + i;
        const uint32_t was = *w, now = rescale4(was, f);
        const uint32_t keep = lo - t >= 4 ? 0xffffffffu : (1u << (8 * (lo - t))) - 1u;
        *w = (now & keep) | (was & ~keep);
      }
    }
    {
      const int ch = threadIdx.x % TK::kChunks, r0 = threadIdx.x / TK::kChunks;
      const float f = kv8_inverse(new_k);
#pragma unroll
      for (int p = 0; p < TK::kPasses; ++p) {
        const int t = r0 + p * TK::kRows;
        if (r0 >= TK::kRows || t < lo || t >= hi) continue;
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = scaled(k[p][i], f);
        *reinterpret_cast<uint2*>(codes + t * DK + ch * 8) =
            make_uint2(encode4(y[0], y[1], y[2], y[3]), encode4(y[4], y[5], y[6], y[7]));
      }
    }
    {  // V changes from rows of tokens to rows of dimensions through LDS
      const int ch = threadIdx.x % TV::kChunks, r0 = threadIdx.x / TV::kChunks;
      const float f = kv8_inverse(new_v);
#pragma unroll
      for (int p = 0; p < TV::kPasses; ++p) {
        const int t = r0 + p * TV::kRows;
        if (r0 >= TV::kRows || t < lo || t >= hi) continue;
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = scaled(v[p][i], f);
        const uint32_t w[2] = {encode4(y[0], y[1], y[2], y[3]), encode4(y[4], y[5], y[6], y[7])};
#pragma unroll
        for (int i = 0; i < 8; ++i)  // dimension 8 ch + i in row i * chunks + ch: no two lanes on a bank
          vt[(i * TV::kChunks + ch) * kRowBytes + v_place(t)] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
      }
    }
    __syncthreads();  // also: held codes have been rewritten before bytes go in beside them
    uint8_t* const to = codes + kBlk * DK;
    if (hi - lo == kBlk) {
      for (int i = threadIdx.x; i < DV * 4; i += kNT) {
        const int d = i >> 2, row = (d & 7) * TV::kChunks + (d >> 3);
        reinterpret_cast<uint4*>(to)[i] = *reinterpret_cast<const uint4*>(vt + row * kRowBytes + (i & 3) * 16);
      }
    } else {  // bytes: the others' stay as they are
      for (int i = threadIdx.x; i < DV * (hi - lo); i += kNT) {
        const int d = i % DV, t = lo + i / DV, row = (d & 7) * TV::kChunks + (d >> 3);
        to[d * kBlk + v_place(t)] = vt[row * kRowBytes + v_place(t)];
      }
    }
  }
  if (update && h == 0 && rest % nblk == 0) update_counts(c, s, b);
}

// The counters of an append whose blocks read them.
__global__ __launch_bounds__(kNT) void append_counts_kernel(Kv8 c, Kv8Append a) {
  update_counts(c, span_of(c, a, blockIdx.x), blockIdx.x);
}

// Slots back as values, 8 elements of one head's K or V a thread; zeros for a slot
// that holds nothing.
template <typename Tag>
__global__ __launch_bounds__(kNT) void rows_kernel(Kv8 c, const int32_t* __restrict__ slots, int64_t N,
                                                   typename Tag::raw* __restrict__ K, typename Tag::raw* __restrict__ V) {
  const int kc = c.DK / 8, per = kc + c.DV / 8;
  const int64_t i = blockIdx.x * static_cast<int64_t>(kNT) + threadIdx.x;
  if (i >= c.B * N * c.HKV * per) return;
  const int ch = static_cast<int>(i % per);
  const int64_t row = i / per, bn = row / c.HKV, b = bn / N;
  const int h = static_cast<int>(row % c.HKV);
  const int64_t slot = slots ? static_cast<int64_t>(slots[bn]) : bn % N;
  float x[8] = {};
  if (slot >= 0 && slot < kv8_length(c, b)) {
    const int64_t at = kv8_block(c, b, slot >> 6, h);
    if (at >= 0) {
      const uint8_t* codes = c.codes + at * c.block_bytes();
      const int t = static_cast<int>(slot & 63);
      uint32_t w[2];
      if (ch < kc) {
        const uint2 u = *reinterpret_cast<const uint2*>(codes + t * c.DK + ch * 8);
        w[0] = u.x;
        w[1] = u.y;
      } else {
        const uint8_t* from = codes + kBlk * c.DK + (ch - kc) * 8 * kBlk + v_place(t);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          w[j] = from[(4 * j) * kBlk] | from[(4 * j + 1) * kBlk] << 8 | from[(4 * j + 2) * kBlk] << 16 |
                 static_cast<uint32_t>(from[(4 * j + 3) * kBlk]) << 24;
      }
      const float f = __uint_as_float(static_cast<uint32_t>(c.scales[at * 2 + (ch < kc ? 0 : 1)]) << 23);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], false), d = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], true);
        x[4 * j] = a[0] * f; x[4 * j + 1] = a[1] * f; x[4 * j + 2] = d[0] * f; x[4 * j + 3] = d[1] * f;
      }
    }
  }
  if (ch < kc) store8<Tag>(K + row * c.DK + ch * 8, x);
  else store8<Tag>(V + row * c.DV + (ch - kc) * 8, x);
}

template <typename Tag, int DK, int DV>
hipError_t append_dims(const Kv8& c, const Kv8Append& a, hipStream_t stream) {
  const int nblk = static_cast<int>((a.T + kBlk - 2) / kBlk + 1);
  const uint32_t kv = static_cast<uint32_t>(c.B * c.HKV * nblk);
  const int64_t q_items = a.Q_out ? c.B * a.T * a.HQ * (DK / 8) : 0;
  const uint32_t grid = kv + static_cast<uint32_t>((q_items + kNT - 1) / kNT);
  // where the blocks read the length to find their place, a launch of its own changes it
  append_kernel<Tag, DK, DV><<<grid, kNT, 0, stream>>>(c, a, nblk, kv, a.start != nullptr);
  if (!a.start) append_counts_kernel<<<static_cast<uint32_t>(c.B), kNT, 0, stream>>>(c, a);
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
  const int64_t items = c.B * N * c.HKV * ((c.DK + c.DV) / 8);
  const uint32_t grid = static_cast<uint32_t>((items + kNT - 1) / kNT);
  if (dtype == 0) rows_kernel<F32><<<grid, kNT, 0, stream>>>(c, slots, N, static_cast<float*>(K), static_cast<float*>(V));
  else if (dtype == 1) rows_kernel<BF16><<<grid, kNT, 0, stream>>>(c, slots, N, static_cast<uint16_t*>(K), static_cast<uint16_t*>(V));
  else rows_kernel<F16><<<grid, kNT, 0, stream>>>(c, slots, N, static_cast<uint16_t*>(K), static_cast<uint16_t*>(V));
  return hipGetLastError();
}

}  // namespace dsa
