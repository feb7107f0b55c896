// kv8.h -- the paged 8-bit cache: its buffers, the format's conversions and the
// launchers behind dsa_kv8_* and dsa_window_attention (include/dsa_amd.h).
//
// A page of the pool holds 64 * 2^page_shift slots, in blocks of 64 of one head:
//   codes  [NP, HKV, page/64, 64*(DK+DV)]  e4m3: K [64][DK], then V [DV][64]
//   scales [NP, HKV, page/64, 2]           E8M0, of the block's K and of its V
// A block is what a wave of the attention multiplies at once.  V lies dimension by
// dimension, a dimension's 64 tokens in the order in which the matrix instructions
// take them (v_place), so that a lane's 16 bytes are its operand and nothing is
// transposed on the way.
#pragma once

#include "dsa_device.h"

namespace dsa {

constexpr int kBlk = 64;  // slots a block

struct Kv8 {
  uint8_t* codes;
  uint8_t* scales;
  const int32_t* pages;  // [B, max_pages] page ids
  int32_t* length;       // [B] slots in use
  int32_t* lost;         // [B] tokens that found no slot
  int64_t B, NP, max_pages;
  int HKV, DK, DV;
  int page_shift;  // a page is 64 << page_shift slots
  __host__ __device__ int64_t slots() const { return (max_pages * kBlk) << page_shift; }
  __host__ __device__ int block_bytes() const { return kBlk * (DK + DV); }
};

// Where token t of a block lies in a dimension's 64 bytes of V: lane group g of a
// 16x16x32 product gets, of each 16 tokens 16j .. 16j+15, the four 16j + 4g + i.
__host__ __device__ __forceinline__ int v_place(int t) { return ((t >> 2) & 3) * 16 + (t >> 4) * 4 + (t & 3); }

__device__ __forceinline__ int32_t kv8_length(const Kv8& c, int64_t b) {
  return max(0, min(c.length[b], static_cast<int32_t>(c.slots())));
}
// Block `blk` of sequence b and head h in units of blocks of the pool; negative where
// its page id names no page.
__device__ __forceinline__ int64_t kv8_block(const Kv8& c, int64_t b, int64_t blk, int h) {
  const int64_t page = c.pages[b * c.max_pages + (blk >> c.page_shift)];
  if (page < 0 || page >= c.NP) return -1;
  return ((page * c.HKV + h) << c.page_shift) + (blk & ((1 << c.page_shift) - 1));
}

// The scale byte of a block whose largest finite magnitude has these bits: the least
// e with max <= 448 * 2^e (the largest e4m3 value), so that nothing saturates; at
// least 2^-117, so that the least code, 2^-9, stands for a normal fp32.
__device__ __forceinline__ uint32_t kv8_scale(uint32_t maxbits) {
  const int e = static_cast<int>((maxbits + 0x1fffffu) >> 23) - 8;
  return static_cast<uint32_t>(min(max(e, 10), 247));
}
__device__ __forceinline__ float kv8_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Tokens into the cache (kv8_cache.hip).  Token strides ldk, ldv, ldq in elements.
struct Kv8Append {
  const void *K, *V, *Q;     // [B,T,HKV,DK], [B,T,HKV,DV], [B,T,HQ,DK] (Q may be null)
  void *K_out, *Q_out;       // rotated, dense; may be null
  int64_t ldk, ldv, ldq;
  const float *cos, *sin;    // [>= slots, R/2]
  const int32_t *start, *count;
  int64_t T;
  int HQ, R, pairs;
};
hipError_t launch_kv8_append(const Kv8& c, const Kv8Append& a, int dtype, hipStream_t stream);
hipError_t launch_kv8_rows(const Kv8& c, const int32_t* slots, int64_t N, int dtype, void* K, void* V,
                           hipStream_t stream);

// Attention over the cache (kv8_attn.hip): the first n slots; window 0: all of them.
bool kv8_supported(int DK, int DV);
int64_t kv8_attn_workspace(const Kv8& c, int64_t Tq, int HQ, int64_t n, int64_t window, int64_t sinks);
hipError_t launch_kv8_attn(const Kv8& c, const void* Q, int dtype, const int32_t* count, int64_t Tq, int HQ,
                           int64_t n, int64_t window, int64_t sinks, float scale, void* out, void* ws,
                           hipStream_t stream);

// Attention of prompts (window_attn.hip).
struct WindowArgs {
  const void *Q, *K, *V;
  void* out;             // [B,T,HQ,D] dense, Q's type
  const int32_t* count;  // [B] or null
  int64_t B, ldq, ldk, ldv;
  int T, HQ, HKV, D;
  int window, sinks;  // 1 <= window <= T, 0 <= sinks <= T
  float scale;
};
bool window_attn_supported(int D);
hipError_t launch_window_attn(const WindowArgs& a, int dtype, hipStream_t stream);

}  // namespace dsa
