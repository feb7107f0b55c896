// kv4_cache.hip -- what goes into the 4-bit decode cache, comes back out of it,
// and is evicted from it (gfx950).
#include "kv4.h"

namespace dsa {
namespace {

constexpr int kNT = 256;

// ---------------------------------------------------------------------------
// Append.  A thread owns word u of a slot (8 elements of one head's K or V)
// and quantises it for the block's tokens; the four lanes of a 32-element
// block share its largest magnitude.
// ---------------------------------------------------------------------------
template <typename Tag>
__global__ __launch_bounds__(kNT) void append_kernel(Kv4 c, const typename Tag::raw* __restrict__ K,
                                                     const typename Tag::raw* __restrict__ V,
                                                     const uint4* __restrict__ new_idx,
                                                     const float* __restrict__ weight,
                                                     const int32_t* __restrict__ count, int64_t T,
                                                     int per_block, int restart, int update) {
  const int64_t b = blockIdx.y;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * per_block;
  const int32_t have = restart ? 0 : kv4_length(c.length, b, c.S);
  const int32_t before = restart ? 0 : c.seen[b];
  const int64_t many = count ? max(0, static_cast<int>(min(static_cast<int64_t>(count[b]), T))) : T;
  const int64_t stored = min(many, c.S - have);
  const int64_t i1 = min(i0 + per_block, stored);

  const int words = c.words(), per_head = (c.DK + c.DV) / 8, kw = c.DK / 8;
  for (int u = threadIdx.x; u < words; u += kNT) {  // words is a multiple of 8
    const int h = u / per_head, r = u - h * per_head;
    const bool isk = r < kw;
    const typename Tag::raw* src =
        isk ? K + (b * T * c.HKV + h) * c.DK + r * 8 : V + (b * T * c.HKV + h) * c.DV + (r - kw) * 8;
    const int64_t step = static_cast<int64_t>(c.HKV) * (isk ? c.DK : c.DV);
    for (int64_t i = i0; i < i1; ++i) {
      float x[8];
      load_cvt<Tag, 8>(src + i * step, x);
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
      m = max(m, dpp_u32<0xB1>(m));  // quad_perm [1,0,3,2]
      m = max(m, dpp_u32<0x4E>(m));  // quad_perm [2,3,0,1]
      const uint32_t s = e8m0_of_max(m);
      const uint32_t w = s == 255u ? 0u : e2m1_pack8(x, e8m0(s));
      const int64_t slot = b * c.S + have + i;
      reinterpret_cast<uint32_t*>(c.codes)[slot * words + u] = w;
      if ((u & 3) == 0) c.scales[slot * c.scale_bytes() + u / 4] = static_cast<uint8_t>(s);
    }
  }
  if (new_idx) {
    const int chunks = c.DI * c.idx_bytes / 16;
    for (int64_t i = i0 * chunks + threadIdx.x; i < i1 * chunks; i += kNT)
      static_cast<uint4*>(c.k_idx)[(b * c.S + have) * chunks + i] = new_idx[b * T * chunks + i];
  }
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kNT) {
    c.position[b * c.S + have + i] = before + static_cast<int32_t>(i);
    c.weight[b * c.S + have + i] = weight ? weight[b * T + i] : 0.0f;
  }
  if (update) {  // the sequence's only block
    __syncthreads();
    if (threadIdx.x == 0) {
      c.length[b] = have + static_cast<int32_t>(stored);
      c.seen[b] = before + static_cast<int32_t>(many);
      c.lost[b] = (restart ? 0 : c.lost[b]) + static_cast<int32_t>(many - stored);
    }
  }
}

// The counters of an append that took more than one block a sequence.
__global__ void append_counts_kernel(Kv4 c, const int32_t* __restrict__ count, int64_t T, int restart) {
  const int64_t b = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  if (b >= c.B) return;
  const int32_t have = restart ? 0 : kv4_length(c.length, b, c.S);
  const int64_t many = count ? max(0, static_cast<int>(min(static_cast<int64_t>(count[b]), T))) : T;
  const int64_t stored = min(many, c.S - have);
  c.length[b] = have + static_cast<int32_t>(stored);
  c.seen[b] = (restart ? 0 : c.seen[b]) + static_cast<int32_t>(many);
  c.lost[b] = (restart ? 0 : c.lost[b]) + static_cast<int32_t>(many - stored);
}

// ---------------------------------------------------------------------------
// Rows back: word u of a slot as 8 values; zeros for a slot that holds nothing.
// ---------------------------------------------------------------------------
template <typename Tag>
__device__ __forceinline__ void store8(typename Tag::raw* p, const float (&x)[8]) {
  if constexpr (Tag::kBytes == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (__is_same(Tag, BF16)) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        w[j] = __builtin_bit_cast(uint32_t,
                                  __builtin_convertvector((f32x2{x[2 * j], x[2 * j + 1]}), bf16x2));
      } else {
        w[j] = __builtin_bit_cast(uint32_t,
                                  __builtin_convertvector((f32x2{x[2 * j], x[2 * j + 1]}), f16x2));
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename Tag>
__global__ __launch_bounds__(kNT) void rows_kernel(Kv4 c, const int32_t* __restrict__ slots, int64_t N,
                                                   int per_block, typename Tag::raw* __restrict__ K,
                                                   typename Tag::raw* __restrict__ V) {
  const int64_t b = blockIdx.y;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * per_block, i1 = min(i0 + per_block, N);
  const int32_t have = kv4_length(c.length, b, c.S);
  const int words = c.words(), per_head = (c.DK + c.DV) / 8, kw = c.DK / 8;
  for (int u = threadIdx.x; u < words; u += kNT) {
    const int h = u / per_head, r = u - h * per_head;
    const bool isk = r < kw;
    typename Tag::raw* dst =
        isk ? K + (b * N * c.HKV + h) * c.DK + r * 8 : V + (b * N * c.HKV + h) * c.DV + (r - kw) * 8;
    const int64_t step = static_cast<int64_t>(c.HKV) * (isk ? c.DK : c.DV);
    for (int64_t i = i0; i < i1; ++i) {
      const int64_t s = slots ? slots[b * N + i] : i;
      float x[8] = {};
      if (s >= 0 && s < have) {
        const int64_t slot = b * c.S + s;
        e2m1_unpack8(reinterpret_cast<const uint32_t*>(c.codes)[slot * words + u],
                     e8m0(c.scales[slot * c.scale_bytes() + u / 4]), x);
      }
      store8<Tag>(dst + i * step, x);
    }
  }
}

// ---------------------------------------------------------------------------
// Evict.  One block a sequence finds the E = length - keep slots that go: the
// E smallest keys, the order-preserving bits of the weight, above all of them
// for a protected (recent) slot; among equals the highest slots go.  Then the
// i-th kept slot at or past `keep` moves into the i-th freed slot below it: no
// slot is both read and written, and no more slots move than have to.
// ---------------------------------------------------------------------------
constexpr int kET = 1024;

__global__ __launch_bounds__(kET) void evict_select_kernel(Kv4 c, int64_t keep, int64_t recent,
                                                           int64_t M, int32_t* __restrict__ src,
                                                           int32_t* __restrict__ dst) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t wsum[kET / kWave];
  __shared__ uint32_t pick[2];
  const int64_t b = blockIdx.x;
  const int32_t n = kv4_length(c.length, b, c.S);
  const float* weight = c.weight + b * c.S;
  const int32_t* position = c.position + b * c.S;
  src += b * M;
  dst += b * M;
  if (n <= keep) {
    for (int64_t i = threadIdx.x; i < M; i += kET) src[i] = dst[i] = -1;
    return;
  }
  const int64_t first_kept = static_cast<int64_t>(c.seen[b]) - recent;
  auto key_of = [&](int s) {
    return position[s] >= first_kept ? 0xffffffffu : float_to_key(weight[s]);
  };
  uint32_t prefix = 0, want = n - static_cast<int32_t>(keep);  // the want-th smallest is the last to go
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kET) hist[i] = 0;
    __syncthreads();
    for (int s = threadIdx.x; s < n; s += kET) {
      const uint32_t k = key_of(s);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&hist[(k >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      uint32_t below = 0, bin = 0;
      while (bin < 255 && below + hist[bin] < want) below += hist[bin++];
      pick[0] = bin;
      pick[1] = want - below;
    }
    __syncthreads();
    prefix |= pick[0] << shift;
    want = pick[1];
    __syncthreads();
  }
  // `want` of the slots with key == prefix go: the last ones
  uint32_t ties = 0, unused;
  for (int s = threadIdx.x; s < n; s += kET) ties += key_of(s) == prefix;
  block_exclusive_sum<kET>(ties, wsum, unused);
  ties = unused;
  uint32_t tie0 = 0, free0 = 0, away0 = 0;
  for (int s0 = 0; s0 < n; s0 += kET) {
    const int s = s0 + threadIdx.x;
    const uint32_t k = s < n ? key_of(s) : 0u;
    const bool tie = s < n && k == prefix;
    uint32_t total;
    const uint32_t at = tie0 + block_exclusive_sum<kET>(tie, wsum, total);
    tie0 += total;
    const bool goes = s < n && (k < prefix || (tie && at >= ties - want));
    const bool freed = goes && s < keep, away = s < n && !goes && s >= keep;
    const uint32_t where = block_exclusive_sum<kET>((freed ? 1u : 0u) | (away ? 0x10000u : 0u), wsum, total);
    if (freed) dst[free0 + (where & 0xffffu)] = s;
    if (away) src[away0 + (where >> 16)] = s;
    free0 += total & 0xffffu;
    away0 += total >> 16;
  }
  for (int64_t i = free0 + threadIdx.x; i < M; i += kET) src[i] = dst[i] = -1;
  if (threadIdx.x == 0) c.length[b] = static_cast<int32_t>(keep);
}

// Copies `bytes` bytes with the wave.  Rows of a multiple of 16 bytes start at one
// too; the others are scales, few bytes and an odd number for some DK + DV.
__device__ __forceinline__ void wave_copy(uint8_t* dst, const uint8_t* src, int bytes) {
  const int lane = threadIdx.x & (kWave - 1);
  if (bytes % 16 == 0) {
    for (int i = lane; i < bytes / 16; i += kWave)
      reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(src)[i];
  } else {
    for (int i = lane; i < bytes; i += kWave) dst[i] = src[i];
  }
}

__global__ __launch_bounds__(kNT) void evict_move_kernel(Kv4 c, int64_t M, const int32_t* __restrict__ src,
                                                         const int32_t* __restrict__ dst) {
  const int64_t b = blockIdx.y;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * (kNT / kWave) + threadIdx.x / kWave;
  if (i >= M || src[b * M + i] < 0) return;
  const int64_t u = b * c.S + src[b * M + i], v = b * c.S + dst[b * M + i];
  const int cb = c.words() * 4, sb = c.scale_bytes(), ib = c.DI * c.idx_bytes;
  wave_copy(c.codes + v * cb, c.codes + u * cb, cb);
  wave_copy(c.scales + v * sb, c.scales + u * sb, sb);
  if (c.k_idx) wave_copy(static_cast<uint8_t*>(c.k_idx) + v * ib, static_cast<uint8_t*>(c.k_idx) + u * ib, ib);
  if ((threadIdx.x & (kWave - 1)) == 0) {
    c.position[v] = c.position[u];
    c.weight[v] = c.weight[u];
  }
}

}  // namespace

hipError_t launch_kv4_append(const Kv4& c, const void* K, const void* V, int dtype,
                             const void* new_idx, const float* weight, const int32_t* count, int64_t T,
                             bool restart, hipStream_t stream) {
  const int per_block = 4;
  const int64_t blocks = (T + per_block - 1) / per_block;
  const dim3 grid(static_cast<uint32_t>(blocks), static_cast<uint32_t>(c.B));
  const int update = blocks == 1;
  const uint4* idx = static_cast<const uint4*>(new_idx);
  if (blocks == 0) {
    // a restart without tokens: the counters alone
  } else if (dtype == 0)
    append_kernel<F32><<<grid, kNT, 0, stream>>>(c, static_cast<const float*>(K), static_cast<const float*>(V),
                                                 idx, weight, count, T, per_block, restart, update);
  else if (dtype == 1)
    append_kernel<BF16><<<grid, kNT, 0, stream>>>(c, static_cast<const uint16_t*>(K), static_cast<const uint16_t*>(V),
                                                  idx, weight, count, T, per_block, restart, update);
  else
    append_kernel<F16><<<grid, kNT, 0, stream>>>(c, static_cast<const uint16_t*>(K), static_cast<const uint16_t*>(V),
                                                 idx, weight, count, T, per_block, restart, update);
  if (!update)
    append_counts_kernel<<<static_cast<uint32_t>((c.B + 255) / 256), 256, 0, stream>>>(c, count, T, restart);
  return hipGetLastError();
}

hipError_t launch_kv4_rows(const Kv4& c, const int32_t* slots, int64_t N, int dtype, void* K, void* V,
                           hipStream_t stream) {
  const int per_block = 4;
  const dim3 grid(static_cast<uint32_t>((N + per_block - 1) / per_block), static_cast<uint32_t>(c.B));
  if (dtype == 0)
    rows_kernel<F32><<<grid, kNT, 0, stream>>>(c, slots, N, per_block, static_cast<float*>(K), static_cast<float*>(V));
  else if (dtype == 1)
    rows_kernel<BF16><<<grid, kNT, 0, stream>>>(c, slots, N, per_block, static_cast<uint16_t*>(K), static_cast<uint16_t*>(V));
  else
    rows_kernel<F16><<<grid, kNT, 0, stream>>>(c, slots, N, per_block, static_cast<uint16_t*>(K), static_cast<uint16_t*>(V));
  return hipGetLastError();
}

hipError_t launch_kv4_evict(const Kv4& c, int64_t keep, int64_t recent, int32_t* src, int32_t* dst,
                            hipStream_t stream) {
  if (keep >= c.S) return hipSuccess;
  const int64_t M = keep < c.S - keep ? keep : c.S - keep;
  evict_select_kernel<<<static_cast<uint32_t>(c.B), kET, 0, stream>>>(c, keep, recent, M, src, dst);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || M == 0) return e;
  const int rows = kNT / kWave;
  evict_move_kernel<<<dim3(static_cast<uint32_t>((M + rows - 1) / rows), static_cast<uint32_t>(c.B)), kNT, 0, stream>>>(c, M, src, dst);
  return hipGetLastError();
}

}  // namespace dsa
