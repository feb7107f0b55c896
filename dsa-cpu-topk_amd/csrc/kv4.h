// kv4.h -- the 4-bit decode cache: its buffers, the format's conversions and
// the launchers behind dsa_kv4_* (include/dsa_amd.h).
//
// A token's keys and values sit in one slot, token-major:
//   codes  [B, S, HKV, (DK+DV)/2]   e2m1, K then V of a head, even element low
//   scales [B, S, HKV, (DK+DV)/32]  E8M0, one per 32 elements, same order
// so 8 elements are the 32-bit word u of a slot's codes and its scale is byte
// u / 4 of its scales, for every HKV, DK and DV.
#pragma once

#include "dsa_device.h"

namespace dsa {

struct Kv4 {
  uint8_t* codes;
  uint8_t* scales;
  void* k_idx;        // [B, S, DI] or null
  int32_t* length;    // [B] slots in use
  int32_t* seen;      // [B] tokens appended so far: the next one's position
  int32_t* lost;      // [B] tokens that found no free slot
  int32_t* position;  // [B, S]
  float* weight;      // [B, S]
  int64_t B, S;
  int HKV, DK, DV, DI, idx_bytes;
  __host__ __device__ int words() const { return HKV * (DK + DV) / 8; }        // of a slot's codes
  __host__ __device__ int scale_bytes() const { return HKV * (DK + DV) / 32; }  // of a slot's scales
};

// Slots in use of sequence b, whatever the buffer holds.
__device__ __forceinline__ int32_t kv4_length(const int32_t* length, int64_t b, int64_t S) {
  return max(0, min(length[b], static_cast<int32_t>(S)));
}

// How many slots query t of sequence b sees: its own token is the last of
// them.  count (or null: Tq) of the Tq queries are tokens, the others see none.
__device__ __forceinline__ int32_t kv4_visible(const int32_t* length, const int32_t* count, int64_t b,
                                               int64_t S, int t, int Tq) {
  const int32_t n = count ? max(0, min(count[b], Tq)) : Tq;
  return t < n ? max(0, kv4_length(length, b, S) - n + t + 1) : 0;
}

// An E8M0 byte as the fp32 scale the conversions take: 255 becomes +inf, for
// which they give NaN.
__device__ __forceinline__ float e8m0(uint32_t byte) { return __uint_as_float(byte << 23); }

// The scale byte of a block whose largest magnitude has these bits: the least
// e with max < 7 * 2^e, so that no element is further from its code than half
// of the grid's widest step (6 is the largest code, steps of 2 below it).
// Adding 1/4 of the mantissa's range carries exactly where the mantissa is
// 1.75 or more.  2 .. 252 keep every value a normal, finite fp32.
__device__ __forceinline__ uint32_t e8m0_of_max(uint32_t maxbits) {
  if (maxbits >= 0x7f800000u) return 255u;  // Inf or NaN: the block reads back as NaN
  const int e = static_cast<int>((maxbits + 0x200000u) >> 23) - 2;
  return static_cast<uint32_t>(min(max(e, 2), 252));
}

// 8 elements as they lie in memory; the bits of their largest magnitude as an
// fp32's (Inf's or above where one is not finite); their codes, x / scale to the
// nearest e2m1 (ties to even, 6 beyond it), exact because the scale is a power
// of two.  16-bit types stay packed in pairs: their magnitudes order as integers.
template <typename Tag>
struct Octet {
  uint32_t w[2 * Tag::kBytes];
  __device__ __forceinline__ void load(const typename Tag::raw* p) {
    __builtin_memcpy(w, __builtin_assume_aligned(p, 16), sizeof(w));
  }
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (Tag::kBytes == 4) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
      return m;
    } else {
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 m = __builtin_bit_cast(u16x2, w[0] & 0x7fff7fffu);
#pragma unroll
      for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
      return __float_as_uint(to_f32(Tag{}, max(m[0], m[1])));
    }
  }
  __device__ __forceinline__ uint32_t codes(float scale) const {
    uint32_t c = 0;
    c = pair<0>(c, scale);
    c = pair<1>(c, scale);
    c = pair<2>(c, scale);
    return pair<3>(c, scale);
  }
  template <int I>
  __device__ __forceinline__ uint32_t pair(uint32_t c, float scale) const {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    if constexpr (Tag::kBytes == 4)
      return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(w[2 * I]), __uint_as_float(w[2 * I + 1]), scale, I);
    else if constexpr (__is_same(Tag, BF16))
      return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[I]), scale, I);
    else
      return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, w[I]), scale, I);
  }
};
__device__ __forceinline__ void e2m1_unpack8(uint32_t w, float scale, float (&x)[8]) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
  const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2);
  const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
  x[0] = a[0]; x[1] = a[1]; x[2] = b[0]; x[3] = b[1];
  x[4] = c[0]; x[5] = c[1]; x[6] = d[0]; x[7] = d[1];
}

// Tokens into the cache (kv4_cache.hip).  K [B,T,HKV,DK], V [B,T,HKV,DV] of
// `dtype`; new_idx [B,T,DI] of the cache's index type or null; weight [B,T] or
// null (0); count [B] or null (T).
hipError_t launch_kv4_append(const Kv4& c, const void* K, const void* V, int dtype,
                             const void* new_idx, const float* weight, const int32_t* count,
                             int64_t T, bool restart, hipStream_t stream);
// N slots a sequence back as values; slots null: 0 .. N-1.
hipError_t launch_kv4_rows(const Kv4& c, const int32_t* slots, int64_t N, int dtype, void* K, void* V,
                           hipStream_t stream);
// Down to `keep` slots a sequence; src, dst [B, M], M = min(keep, S - keep).
hipError_t launch_kv4_evict(const Kv4& c, int64_t keep, int64_t recent, int32_t* src, int32_t* dst,
                            hipStream_t stream);
// Down to S - count[b] (null: T) slots; src, dst [B, T].
hipError_t launch_kv4_make_room(const Kv4& c, const int32_t* count, int64_t T, int64_t recent, int32_t* src,
                                int32_t* dst, hipStream_t stream);

// Indexer scores [B, Tq, span] (kv4_indexer.hip); dtype (of q and w): key_dtype (the
// cache's) or fp32.
hipError_t launch_kv4_indexer(const Kv4& c, const void* q, const void* w, int dtype, int key_dtype,
                              const int32_t* count, int64_t Tq, int HI, int64_t span, float* scores,
                              hipStream_t stream);

// Attention over the cache (kv4_attn.hip): n slots a query, those of `slots`
// [B, Tq, n] or (null) the first n.
bool kv4_attn_supported(int DK, int DV);
int64_t kv4_attn_workspace(const Kv4& c, int64_t Tq, int HQ, bool listed, int64_t n, bool accumulate);
hipError_t launch_kv4_attn(const Kv4& c, const void* Q, int dtype, const int32_t* slots,
                           const int32_t* count, int64_t Tq, int HQ, int64_t n, bool accumulate,
                           float scale, float* out, void* ws, hipStream_t stream);

}  // namespace dsa
