// kv4_cache.hip -- what goes into the 4-bit decode cache, comes back out of it,
// and is evicted from it (gfx950).
//
// Measured: 2 x 16384 tokens of 8 heads of 128 in bf16 in (187 MB) 46 us and back
// out (170 MB) 27 us, 4.9 TB/s together where a copy reaches 5.2; eviction's select
// 7.2 us for 32 sequences of 2049 slots with the one slot that moves, 10.8 for 8 of
// 4099, a chain of passes over registers, histogram and scans; its moves 5.2 us for
// 8 x 760 slots.
#include "kv4.h"

namespace dsa {
namespace {

constexpr int kNT = 256;

// How a block's threads cover its tokens: a thread owns word u of a slot (8
// elements of one head's K or V) for every `step`-th of the block's tokens, so
// that the head and the source's stride are worked out once, and small slots
// still take all threads.  words is a multiple of 4, so the 4 lanes of a
// 32-element block stay 4 neighbours.
struct Cover {
  int u, first, step;  // past the slot's words: nothing to do
  bool is_k;
  int64_t at, stride;  // elements: of word u in the first token's K or V, from token to token
};
__device__ __forceinline__ Cover cover(const Kv4& c, int base) {
  const int words = c.words(), per_head = (c.DK + c.DV) / 8, kw = c.DK / 8;
  Cover t;
  t.step = max(1, kNT / words);
  t.first = words < kNT ? threadIdx.x / words : 0;
  t.u = words < kNT ? threadIdx.x - t.first * words : base + threadIdx.x;
  if (t.first >= t.step) t.u = words;
  const int h = t.u / per_head, r = t.u - h * per_head;
  t.is_k = r < kw;
  t.at = t.is_k ? static_cast<int64_t>(h) * c.DK + r * 8 : static_cast<int64_t>(h) * c.DV + (r - kw) * 8;
  t.stride = static_cast<int64_t>(c.HKV) * (t.is_k ? c.DK : c.DV);
  return t;
}

// ---------------------------------------------------------------------------
// Append, bound by memory: a thread's kAhead tokens are on their way at once
// (2, 4 and 8 measured 46, 49 and 53 us for 2 x 16384 tokens of 8 heads of 128 in
// bf16, 187 MB).
// ---------------------------------------------------------------------------
constexpr int kAhead = 2, kRowsAhead = 4;

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

  const int words = c.words();
  const int64_t slot0 = b * c.S + have;
  for (int base = 0; base < words; base += kNT) {
    const Cover t = cover(c, base);
    if (t.u >= words) continue;
    const int nb = static_cast<int>(max(static_cast<int64_t>(0), i1 - i0));  // at most kAhead a thread
    const typename Tag::raw* src = (t.is_k ? K : V) + (b * T + i0) * t.stride + t.at;
    uint32_t* codes = reinterpret_cast<uint32_t*>(c.codes) + (slot0 + i0) * words + t.u;
    uint8_t* scales = c.scales + (slot0 + i0) * (words / 4) + t.u / 4;
    const int stride = static_cast<int>(t.stride);
    Octet<Tag> x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (t.first + k * t.step < nb) x[k].load(src + (t.first + k * t.step) * stride);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = t.first + k * t.step;
      if (i >= nb) break;  // the same for the 4 lanes of a block
      uint32_t m = x[k].top();
      m = max(m, dpp_u32<0xB1>(m));  // quad_perm [1,0,3,2]
      m = max(m, dpp_u32<0x4E>(m));  // quad_perm [2,3,0,1]
      const uint32_t s = e8m0_of_max(m);
      codes[i * words] = s == 255u ? 0u : x[k].codes(e8m0(s));
      if ((t.u & 3) == 0) scales[i * (words / 4)] = static_cast<uint8_t>(s);
    }
  }
  if (new_idx) {
    const int chunks = c.DI * c.idx_bytes / 16;
    for (int64_t i = i0 * chunks + threadIdx.x; i < i1 * chunks; i += kNT)
      static_cast<uint4*>(c.k_idx)[slot0 * chunks + i] = new_idx[b * T * chunks + i];
  }
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kNT) {
    c.position[slot0 + i] = before + static_cast<int32_t>(i);
    c.weight[slot0 + i] = weight ? weight[b * T + i] : 0.0f;
  }
  if (update && blockIdx.x == 0) {  // the sequence's only block, or no block reads the counters
    __syncthreads();
    if (threadIdx.x == 0) {
      c.length[b] = have + static_cast<int32_t>(stored);
      c.seen[b] = before + static_cast<int32_t>(many);
      c.lost[b] = (restart ? 0 : c.lost[b]) + static_cast<int32_t>(many - stored);
    }
  }
}

// The counters of an append whose blocks read them.
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
  const int words = c.words();
  for (int base = 0; base < words; base += kNT) {
    const Cover t = cover(c, base);
    if (t.u >= words) continue;
    typename Tag::raw* dst = (t.is_k ? K : V) + b * N * t.stride + t.at;
#pragma unroll kRowsAhead
    for (int64_t i = i0 + t.first; i < i1; i += t.step) {
      const int64_t s = slots ? slots[b * N + i] : i;
      float x[8] = {};
      if (s >= 0 && s < have) {
        const int64_t slot = b * c.S + s;
        e2m1_unpack8(reinterpret_cast<const uint32_t*>(c.codes)[slot * words + t.u],
                     e8m0(c.scales[slot * (words / 4) + t.u / 4]), x);
      }
      store8<Tag>(dst + i * t.stride, x);
    }
  }
}

// Copies `bytes` bytes, a multiple of Unit's, with the wave.
template <typename Unit>
__device__ __forceinline__ void wave_copy(uint8_t* dst, const uint8_t* src, int bytes) {
  const int n = bytes / static_cast<int>(sizeof(Unit));
  for (int i = threadIdx.x & (kWave - 1); i < n; i += kWave)
    reinterpret_cast<Unit*>(dst)[i] = reinterpret_cast<const Unit*>(src)[i];
}

// Slot u's token into slot v, by a wave.
__device__ __forceinline__ void wave_move(const Kv4& c, int64_t u, int64_t v) {
  const int cb = c.words() * 4, sb = c.scale_bytes(), ib = c.DI * c.idx_bytes;
  // codes and index keys are 16-byte aligned, in rows of multiples of it; scales are
  // 4-byte aligned, few bytes and an odd number for some DK + DV
  wave_copy<uint4>(c.codes + v * cb, c.codes + u * cb, cb);
  if (sb % 4 == 0) wave_copy<uint32_t>(c.scales + v * sb, c.scales + u * sb, sb);
  else wave_copy<uint8_t>(c.scales + v * sb, c.scales + u * sb, sb);
  if (c.k_idx) wave_copy<uint4>(static_cast<uint8_t*>(c.k_idx) + v * ib, static_cast<uint8_t*>(c.k_idx) + u * ib, ib);
  if ((threadIdx.x & (kWave - 1)) == 0) {
    c.position[v] = c.position[u];
    c.weight[v] = c.weight[u];
  }
}

// ---------------------------------------------------------------------------
// Evict.  One block a sequence finds the E = length - keep slots that go: the
// E smallest keys, the order-preserving bits of the weight, above all of them
// for a protected (recent) slot; among equals the highest slots go.  Then the
// i-th kept slot at or past `keep` moves into the i-th freed slot below it: no
// slot is both read and written, and no more slots move than have to.
//
// A thread holds VPT neighbouring slots' keys in registers (longer caches are
// read again in every pass, VPT * 1024 slots at a time).  The E-th smallest key
// is found by halving the range by 1024: a histogram of the keys between lo and
// hi, whose bins cut that range evenly, and the bin that holds the E-th; done when
// the bin's keys all go, or are all equal.  Few keys share a bin of weights spread
// like real ones, so two passes are the rule, and few lanes add to one bin at once
// (four passes over fixed bytes of the key, read again from memory: 44-51 us).
// ---------------------------------------------------------------------------
constexpr int kET = 1024, kBins = 1024;
constexpr int kInPlace = 64;  // most moves that the selecting block makes itself

// The block's sum of v before this thread's, and over all (kET threads).
__device__ __forceinline__ uint32_t evict_scan(uint32_t v, uint32_t* wsum, uint32_t& total) {
  return block_exclusive_sum<kET>(v, wsum, total);
}

// What stays of a sequence: `keep` slots, or (room) as many as leave count[b] (or
// null: `keep`) of the S free.
template <int VPT>
__global__ __launch_bounds__(kET) void evict_select_kernel(Kv4 c, int64_t keep, int64_t recent, bool room,
                                                           const int32_t* __restrict__ count, int64_t M,
                                                           int32_t* __restrict__ src, int32_t* __restrict__ dst) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t wsum[kET / kWave], wlo[kET / kWave], whi[kET / kWave];
  __shared__ uint32_t pick[3];
  __shared__ int32_t from[kInPlace], to[kInPlace];
  const int64_t b = blockIdx.x;
  const int32_t n = kv4_length(c.length, b, c.S);
  const float* weight = c.weight + b * c.S;
  const int32_t* position = c.position + b * c.S;
  src += b * M;
  dst += b * M;
  constexpr uint32_t kProtected = 0xffffffffu;  // above every weight's key
  const int64_t first_kept = static_cast<int64_t>(c.seen[b]) - recent;
  const int32_t S = static_cast<int32_t>(c.S);
  constexpr int kSpan = VPT * kET;
  uint32_t key[VPT];
  auto read = [&](int s0) {  // keys of slots s0 + VPT * thread .., which may be past n
    const int s = s0 + threadIdx.x * VPT;
    float w[VPT];
    int32_t p[VPT];
    if (s + VPT <= S) {  // 16 bytes at once, at any multiple of 4
#pragma unroll
      for (int i = 0; i < VPT; i += 4) {
        __builtin_memcpy(w + i, weight + s + i, 16);
        __builtin_memcpy(p + i, position + s + i, 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        w[i] = s + i < S ? weight[s + i] : 0.0f;
        p[i] = s + i < S ? position[s + i] : 0;
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) key[i] = p[i] >= first_kept ? kProtected : float_to_key(w[i]);
  };
  read(0);  // on its way together with the length
  if (room) keep = c.S - (count ? max(static_cast<int64_t>(0), min(static_cast<int64_t>(count[b]), keep)) : keep);
  if (n <= keep) {
    for (int64_t i = threadIdx.x; i < M; i += kET) src[i] = dst[i] = -1;
    return;
  }
  const bool once = n <= kSpan;
  auto each = [&](auto f) {  // f(slot, key) for the thread's slots of a span that count
    for (int s0 = 0; s0 < n; s0 += kSpan) {
      if (!once) read(s0);
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (s0 + static_cast<int>(threadIdx.x) * VPT + i < n) f(key[i]);
    }
  };

  const uint32_t E = n - static_cast<int32_t>(keep);
  uint32_t lo = kProtected, hi = 0, open = 0;  // of the slots that are not protected
  each([&](uint32_t k) {
    if (k != kProtected) {
      lo = min(lo, k);
      hi = max(hi, k);
      ++open;
    }
  });
  lo = wave_extreme_u32<false>(lo);
  hi = wave_extreme_u32<true>(hi);
  if ((threadIdx.x & 63) == 0) {
    wlo[threadIdx.x / kWave] = lo;
    whi[threadIdx.x / kWave] = hi;
  }
  uint32_t unprotected;
  evict_scan(open, wsum, unprotected);  // its barriers publish wlo and whi too
#pragma unroll
  for (int w = 0; w < kET / kWave; ++w) {
    lo = min(lo, wlo[w]);
    hi = max(hi, whi[w]);
  }
  // keys below `lo` go, those above `hi` stay, and of the ties between them `want`
  uint32_t want = E, ties = 0;
  if (E > unprotected) {  // more protected than stay: the last of them go too
    lo = hi = kProtected;
    want = E - unprotected;
    ties = n - unprotected;
  } else {
    ties = unprotected;
    while (want != ties && lo != hi) {  // some key between lo and hi goes, and some stays
      const int shift = max(0, 32 - static_cast<int>(__builtin_clz(hi - lo)) - 10);
      __syncthreads();
      hist[threadIdx.x] = 0;
      __syncthreads();
      each([&](uint32_t k) {
        if (k >= lo && k <= hi) atomicAdd(&hist[(k - lo) >> shift], 1u);
      });
      __syncthreads();
      const uint32_t mine = hist[threadIdx.x];
      uint32_t total;
      const uint32_t below = evict_scan(mine, wsum, total);
      if (below < want && want <= below + mine) {
        pick[0] = threadIdx.x;
        pick[1] = want - below;
        pick[2] = mine;
      }
      __syncthreads();
      lo += pick[0] << shift;
      hi = min(hi, lo + ((1u << shift) - 1));
      want = pick[1];
      ties = pick[2];
    }
  }

  // The lists, in order of slots.
  uint32_t tie0 = 0, free0 = 0, away0 = 0, total;
  for (int s0 = 0; s0 < n; s0 += kSpan) {
    if (!once) read(s0);
    const int s = s0 + threadIdx.x * VPT;
    uint32_t tie = 0;
    if (want != ties) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) tie += s + i < n && key[i] == lo;
      const uint32_t before = tie0 + evict_scan(tie, wsum, total);
      tie0 += total;
      tie = before;
    }
    uint64_t freed = 0, away = 0;  // the thread's slots, a bit each
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (s + i >= n) continue;
      bool goes = key[i] < lo || (key[i] <= hi && want == ties);
      if (want != ties && key[i] == lo) goes = tie++ >= ties - want;
      if (goes && s + i < keep) freed |= 1ull << i;
      if (!goes && s + i >= keep) away |= 1ull << i;
    }
    // both counts of a span in one sum, 16 bits each (kSpan <= 2^14)
    const uint32_t before = evict_scan(popc64(freed) | popc64(away) << 16, wsum, total);
    uint32_t f = free0 + (before & 0xffffu), w = away0 + (before >> 16);
    free0 += total & 0xffffu;
    away0 += total >> 16;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (freed >> i & 1) {
        if (M <= kInPlace) to[f] = s + i;
        dst[f++] = s + i;
      }
      if (away >> i & 1) {
        if (M <= kInPlace) from[w] = s + i;
        src[w++] = s + i;
      }
    }
  }
  for (int64_t i = free0 + threadIdx.x; i < M; i += kET) src[i] = dst[i] = -1;
  if (threadIdx.x == 0) c.length[b] = static_cast<int32_t>(keep);
  if (M <= kInPlace) {
    __syncthreads();
    for (uint32_t i = threadIdx.x / kWave; i < free0; i += kET / kWave) wave_move(c, b * c.S + from[i], b * c.S + to[i]);
  }
}

__global__ __launch_bounds__(kNT) void evict_move_kernel(Kv4 c, int64_t M, const int32_t* __restrict__ src,
                                                         const int32_t* __restrict__ dst) {
  const int64_t b = blockIdx.y;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * (kNT / kWave) + threadIdx.x / kWave;
  if (i >= M || src[b * M + i] < 0) return;
  wave_move(c, b * c.S + src[b * M + i], b * c.S + dst[b * M + i]);
}

// Tokens of a block whose threads take `each` of them.
int tokens_per_block(const Kv4& c, int each) {
  const int words = c.words();
  return each * (words < kNT ? kNT / words : 1);
}

}  // namespace

hipError_t launch_kv4_append(const Kv4& c, const void* K, const void* V, int dtype,
                             const void* new_idx, const float* weight, const int32_t* count, int64_t T,
                             bool restart, hipStream_t stream) {
  const int per_block = tokens_per_block(c, kAhead);
  const int64_t blocks = (T + per_block - 1) / per_block;
  const dim3 grid(static_cast<uint32_t>(blocks), static_cast<uint32_t>(c.B));
  const int update = blocks == 1 || (restart && blocks > 0);
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
  const int per_block = tokens_per_block(c, kRowsAhead);
  const dim3 grid(static_cast<uint32_t>((N + per_block - 1) / per_block), static_cast<uint32_t>(c.B));
  if (dtype == 0)
    rows_kernel<F32><<<grid, kNT, 0, stream>>>(c, slots, N, per_block, static_cast<float*>(K), static_cast<float*>(V));
  else if (dtype == 1)
    rows_kernel<BF16><<<grid, kNT, 0, stream>>>(c, slots, N, per_block, static_cast<uint16_t*>(K), static_cast<uint16_t*>(V));
  else
    rows_kernel<F16><<<grid, kNT, 0, stream>>>(c, slots, N, per_block, static_cast<uint16_t*>(K), static_cast<uint16_t*>(V));
  return hipGetLastError();
}

namespace {

hipError_t launch_evict(const Kv4& c, int64_t keep, int64_t recent, bool room, const int32_t* count,
                        int64_t M, int32_t* src, int32_t* dst, hipStream_t stream) {
  const uint32_t grid = static_cast<uint32_t>(c.B);
  if (c.S <= 4 * kET) evict_select_kernel<4><<<grid, kET, 0, stream>>>(c, keep, recent, room, count, M, src, dst);
  else evict_select_kernel<16><<<grid, kET, 0, stream>>>(c, keep, recent, room, count, M, src, dst);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || M <= kInPlace) return e;
  const int rows = kNT / kWave;
  evict_move_kernel<<<dim3(static_cast<uint32_t>((M + rows - 1) / rows), static_cast<uint32_t>(c.B)), kNT, 0, stream>>>(c, M, src, dst);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv4_evict(const Kv4& c, int64_t keep, int64_t recent, int32_t* src, int32_t* dst,
                            hipStream_t stream) {
  if (keep >= c.S) return hipSuccess;
  return launch_evict(c, keep, recent, false, nullptr, keep < c.S - keep ? keep : c.S - keep, src, dst, stream);
}

// No more slots move than are freed, T at most.
hipError_t launch_kv4_make_room(const Kv4& c, const int32_t* count, int64_t T, int64_t recent, int32_t* src,
                                int32_t* dst, hipStream_t stream) {
  if (T == 0) return hipSuccess;
  return launch_evict(c, T, recent, true, count, T, src, dst, stream);
}

}  // namespace dsa
