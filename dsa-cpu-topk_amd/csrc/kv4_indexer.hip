// kv4_indexer.hip -- lightning indexer of new tokens against the cached index
// keys (gfx950):
//   I[b,t,s] = sum_j w[b,t,j] * ReLU(<q[b,t,j,:], k[b,s,:]>)  for visible s, else -inf
//
// The index keys are the bulk of the bytes (DI of them a slot, for 4 bytes of
// score a token) and are read once: a wave takes 16 * KB slots into registers
// as B operands, a lane a quarter of one slot's row, and walks the heads, 16 at a
// time, as A operands.  A block serves up to kTokens of a sequence's tokens, whose
// q rows (in the order in which lanes read them) and weights lie in LDS.  A lane's
// four results are four heads of one slot: ReLU, weight and sum stay in the lane,
// and one sum over the four lane groups ends a slot.
//
// fp32 takes the fp32 matrix instruction (its 157 TFLOP/s are about what 64 heads
// of 128 need at the memory's rate, fewer heads need less).  fp32 queries over 16-bit
// keys take it too: the keys are read as they are and widened in registers, so that
// no operand is rounded.
//
// Measured: 8 sequences of up to 32768 slots, 64 heads of 128, bf16 (62 MB): 14.9 us,
// 4.1 TB/s; the loads alone 13.7.  Full ones in fp32: 8 heads of 64 14.7 us, 4.6 TB/s;
// 64 heads of 128 46 us, bound by the matrix instruction; over bf16 keys 11.5 and 47.
#include "dsa_launch.h"
#include "kv4.h"
#include "tile_common.h"

namespace dsa {
namespace {

constexpr int kWaves = kNT / kWave;
constexpr int kTokens = 4;              // of one block
constexpr int kMaxLds = 64 * 1024;      // of q and weights; wider q rows are read through L2

struct IndexArgs {
  Kv4 c;
  const void* q;
  const void* w;
  const int32_t* count;
  int Tq, per, groups;  // tokens a block, groups of them a sequence
  int HI, blocks;  // that share a group's slots, a tile to each of their waves in turn
  int64_t span;    // slots scored
  float* scores;
};

template <typename Tag>
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, f32x4 acc) {
  if constexpr (Tag::kBytes == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), acc, 0, 0, 0);
    return acc;
  } else {
    return Mfma16x16x32<Tag>::run(a, b, acc);
  }
}

// Piece c of a lane's quarter of a key row, as the matrix instruction's type Tag.
template <typename Tag, typename Key, int NK>
__device__ __forceinline__ u32x4 key_piece(const u32x4 (&k)[NK], int c) {
  if constexpr (__is_same(Tag, Key)) {
    return k[c];
  } else {
    u32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = k[c / 2][c % 2 * 2 + i / 2];
      x[i] = __float_as_uint(to_f32(Key{}, static_cast<uint16_t>(i % 2 ? w >> 16 : w)));
    }
    return x;
  }
}

// Tag: the type of q and w; Key: of the cached keys, the same or (Tag fp32) a 16-bit one.
template <typename Tag, typename Key, int DI, int KB, bool IN_LDS>
__global__ __launch_bounds__(kNT) void indexer_kernel(IndexArgs a) {
  using raw = typename Tag::raw;
  constexpr int ROW = DI * Tag::kBytes, NC = ROW / 64;  // bytes of a row, 16-byte pieces of a lane's quarter
  constexpr int KROW = DI * Key::kBytes, NK = KROW / 64;  // of the keys
  extern __shared__ u32x4 lds[];
  const int nht = (a.HI + 15) / 16;
  const uint32_t bg = blockIdx.x / a.blocks, b = bg / a.groups;
  const int t0 = static_cast<int>(bg % a.groups) * a.per, nt = min(a.per, a.Tq - t0);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x & 63, g = lane >> 4, r16 = lane & 15;
  int32_t limit = 0;  // slots that some token of the group sees
  for (int t = 0; t < nt; ++t) limit = max(limit, kv4_visible(a.c.length, a.count, b, a.c.S, t0 + t, a.Tq));
  const int64_t bt0 = static_cast<int64_t>(b) * a.Tq + t0;
  const int64_t end = min(a.span, static_cast<int64_t>(limit));
  constexpr int kTile = 16 * KB;
  const int64_t step = static_cast<int64_t>(a.blocks) * kWaves * kTile;
  int64_t s = static_cast<int64_t>(blockIdx.x % a.blocks * kWaves + wave) * kTile;
  const bool busy = static_cast<int64_t>(blockIdx.x % a.blocks) * kWaves * kTile < end;  // one of the block's waves is

  const char* keys = static_cast<const char*>(a.c.k_idx) + b * a.c.S * KROW;
  auto load = [&](u32x4 (&k)[KB][NK], int64_t s0) {  // rows past the last visible one give zeros
    const __amdgpu_buffer_rsrc_t r = rows_rsrc(keys, s0, limit, KROW);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int c = 0; c < NK; ++c)
        k[kb][c] = __builtin_bit_cast(u32x4, buffer_load_f32x4(r, (16 * kb + r16) * KROW + g * (KROW / 4) + c * 16, 0, 0));
  };
  u32x4 k0[KB][NK], k1[KB][NK];
  if (s < end) load(k0, s);

  const char* q = static_cast<const char*>(a.q) + bt0 * a.HI * ROW;
  const raw* w = static_cast<const raw*>(a.w) + bt0 * a.HI;
  float* weights = reinterpret_cast<float*>(lds + (IN_LDS ? nt * nht * NC * 64 : 0));
  auto piece = [&](int t, int ht, int c) {  // the lane's A operand
    const int h = 16 * ht + r16;
    u32x4 x = {0, 0, 0, 0};
    if (h < a.HI) x = *reinterpret_cast<const u32x4*>(q + (static_cast<int64_t>(t) * a.HI + h) * ROW + g * (ROW / 4) + c * 16);
    return x;
  };
  if (busy && IN_LDS) {
    for (int i = wave; i < nt * nht * NC; i += kWaves)
      lds[i * 64 + lane] = piece(i / (nht * NC), i / NC % nht, i % NC);
  }
  for (int i = threadIdx.x; busy && i < nt * nht * 16; i += kNT) {
    const int t = i / (nht * 16), h = i % (nht * 16);
    weights[i] = h < a.HI ? to_f32(Tag{}, w[t * a.HI + h]) : 0.0f;
  }
  __syncthreads();

  auto compute = [&](const u32x4 (&k)[KB][NK], int64_t s0) {
    for (int t = 0; t < nt; ++t) {
      float sum[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) sum[kb] = 0.0f;
      for (int ht = 0; ht < nht; ++ht) {
        f32x4 acc[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) acc[kb] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const u32x4 x = IN_LDS ? lds[((t * nht + ht) * NC + c) * 64 + lane] : piece(t, ht, c);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) acc[kb] = mfma16<Tag>(x, key_piece<Tag, Key>(k[kb], c), acc[kb]);
        }
        const float4 wv = *reinterpret_cast<const float4*>(weights + (t * nht + ht) * 16 + 4 * g);
        // Rows past HI are zeros, and 0 * Inf is NaN there: they stay out of the sum.
        const int heads = a.HI - 16 * ht;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          // the IEEE maximum: a NaN stays one
          f32x4 r;
#pragma unroll
          for (int i = 0; i < 4; ++i) r[i] = __builtin_elementwise_maximum(acc[kb][i], 0.0f);
          if (heads < 16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = 4 * g + i < heads ? r[i] : 0.0f;
          }
          sum[kb] = fmaf(wv.x, r[0], sum[kb]);
          sum[kb] = fmaf(wv.y, r[1], sum[kb]);
          sum[kb] = fmaf(wv.z, r[2], sum[kb]);
          sum[kb] = fmaf(wv.w, r[3], sum[kb]);
        }
      }
      float mine = 0.0f;  // lane group g stores the slots of tile g
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const float x = sum_xor32(sum_xor16(sum[kb]));
        mine = g == kb ? x : mine;
      }
      const int64_t at = s0 + 16 * g + r16;
      const int32_t seen = kv4_visible(a.c.length, a.count, b, a.c.S, t0 + t, a.Tq);
      if (g < KB && at < a.span) a.scores[(bt0 + t) * a.span + at] = at < seen ? mine : -INFINITY;
    }
  };
  while (s < end) {
    if (s + step < end) load(k1, s + step);
    compute(k0, s);
    s += step;
    if (s >= end) break;
    if (s + step < end) load(k0, s + step);
    compute(k1, s);
    s += step;
  }
  for (; s < a.span; s += step)  // the tiles that nothing sees
    for (int t = 0; t < nt; ++t)
      if (lane < kTile && s + lane < a.span) a.scores[(bt0 + t) * a.span + s + lane] = -INFINITY;
}

template <typename Tag, typename Key, int DI>
hipError_t launch_di(IndexArgs a, hipStream_t stream) {
  constexpr int ROW = DI * Tag::kBytes, KROW = DI * Key::kBytes;
  // 32 registers of keys a stage, at most the 4 tiles that 4 lane groups store
  constexpr int KB = KROW <= 128 ? 4 : KROW <= 256 ? 2 : 1;
  const int nht = (a.HI + 15) / 16;
  const int row_lds = nht * 16 * (ROW + 4);  // of one token
  a.per = a.Tq < kTokens ? a.Tq : kTokens;
  while (a.per > 1 && a.per * row_lds > kMaxLds) --a.per;
  a.groups = (a.Tq + a.per - 1) / a.per;
  const bool in_lds = a.per * row_lds <= kMaxLds;
  const int step = 16 * KB * kWaves;
  const int64_t rows = a.c.B * a.groups, steps = (a.span + step - 1) / step;
  // two blocks a compute unit (1, 2, 3, 4 and 8 measured 18.6, 15.1, 16.7, 16.6 and
  // 19.3 us for 8 x 32768 slots, 64 heads of 128 in bf16)
  const int cus = device_cus() > 0 ? device_cus() : 256;
  const int64_t blocks = (2 * cus + rows - 1) / rows;
  a.blocks = static_cast<int>(blocks < 1 ? 1 : blocks > steps ? steps : blocks);
  const uint32_t grid = static_cast<uint32_t>(rows * a.blocks);
  if (in_lds)
    indexer_kernel<Tag, Key, DI, KB, true><<<grid, kNT, a.per * row_lds, stream>>>(a);
  else
    indexer_kernel<Tag, Key, DI, KB, false><<<grid, kNT, nht * 64, stream>>>(a);
  return hipGetLastError();
}

template <typename Tag, typename Key>
hipError_t launch_tag(const IndexArgs& a, hipStream_t stream) {
  switch (a.c.DI) {
    case 16:
      if constexpr (Key::kBytes == 4) return launch_di<Tag, Key, 16>(a, stream);
      return hipErrorNotSupported;
    case 32: return launch_di<Tag, Key, 32>(a, stream);
    case 64: return launch_di<Tag, Key, 64>(a, stream);
    case 128: return launch_di<Tag, Key, 128>(a, stream);
    default: return launch_di<Tag, Key, 256>(a, stream);
  }
}

}  // namespace

hipError_t launch_kv4_indexer(const Kv4& c, const void* q, const void* w, int dtype, int key_dtype,
                              const int32_t* count, int64_t Tq, int HI, int64_t span, float* scores, hipStream_t stream) {
  IndexArgs a;
  a.c = c;
  a.q = q;
  a.w = w;
  a.count = count;
  a.Tq = static_cast<int>(Tq);
  a.HI = HI;
  a.span = span;
  a.scores = scores;
  if (dtype != key_dtype) return key_dtype == 1 ? launch_tag<F32, BF16>(a, stream) : launch_tag<F32, F16>(a, stream);
  return dtype == 0   ? launch_tag<F32, F32>(a, stream)
         : dtype == 1 ? launch_tag<BF16, BF16>(a, stream)
                      : launch_tag<F16, F16>(a, stream);
}

}  // namespace dsa
