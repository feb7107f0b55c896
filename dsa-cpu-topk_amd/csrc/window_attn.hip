// window_attn.hip -- attention of prompts over a sliding window and the first tokens
// (gfx950).
//
//   O[b,t,h,:] = sum_s p_s V[b,s,h/G,:],  p = softmax_s(<Q[b,t,h], K[b,s,h/G]> scale)
// over s <= t with s > t - window or s < sinks.
//
// A block takes 128 queries of one head, a wave 32 (or 64 and 16), and walks the tiles of 64 keys that
// any of them sees: those of the first tokens, then those of the window.  K and V go to
// LDS by DMA, two buffers each, the products run transposed,
//   S^T = K . Q^T,  O^T = V^T . P^T,
// so that P goes from the first product's registers into the second one's, and the
// softmax is one pass with a running maximum and sum in fp32.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "dsa_launch.h"
#include "kv8.h"
#include "tile_common.h"
#include "window_walk.h"

namespace dsa {
namespace {

struct Win {
  const void *Q, *K, *V;
  void* out;
  const int32_t* count;
  int64_t B, ldq, ldk, ldv;
  int T, HQ, HKV, G, window, sinks;
  float scale_log2;  // positive: times a masked -Inf it is one
  uint32_t flip;     // Q's sign bits, where the scale is negative
};

template <int TQ, int KT>
__device__ __forceinline__ Walk walk_in(const Win& a, int64_t b, int t0) {
  return walk_of<TQ, KT>(a.count ? max(0, min(a.count[b], a.T)) : a.T, a.window, a.sinks, t0);
}

// Block -> (tile of queries, batch, head), the latest tiles, which see most, first.  The
// sequences' K/V heads lie innermost, so that the tiles of one go to one XCD where they are a
// multiple of 8 (block i starts on XCD i % 8), and all XCDs have the same work where they are
// not: one head of 128, 8 query heads, 8192 tokens, window 1000, 312 us on one XCD, 60 on all;
// 9 K/V heads, 16384 tokens, window 2048, 977 with two on one of them, 695 so.  (At D = 256 the
// same loses: 36 heads on 9, 2121 us with a head's tiles on one XCD, 2497 so.)
// (32-bit throughout: a 64-bit division costs as much as a short prompt's tile.)
template <int TQ>
__device__ __forceinline__ void place(const Win& a, int& t0, int64_t& b, int& h, int& hk) {
  const uint32_t ntile = static_cast<uint32_t>(a.T + TQ - 1) / TQ, G = a.G, HKV = a.HKV;
  const uint32_t pairs = static_cast<uint32_t>(a.B) * HKV;  // (b, K/V head)
  const uint32_t i = blockIdx.x / pairs, pair = blockIdx.x - i * pairs, tile = i / G, bb = pair / HKV;
  t0 = static_cast<int>((ntile - 1 - tile) * TQ);
  b = bb;
  hk = static_cast<int>(pair - bb * HKV);
  h = static_cast<int>(hk * G + (i - tile * G));
}
template <int TQ>
int64_t blocks_of(const Win& a) {
  return a.B * a.HQ * ((a.T + TQ - 1) / TQ);
}

__device__ __forceinline__ float mul(float x, float y) {  // rounded by itself
#pragma clang fp contract(off)
  return x * y;
}
// 2^(x scale - ref).  An fma keeps x scale whole, where ref, the maximum's product, was
// rounded: at logits of 2^28 (f16: 2^25) and more all p of a row may be beyond or below a 16-bit
// type, which leaves no finite result, and the careful pass rounds each as ref was.
template <bool CAREFUL>
__device__ __forceinline__ float weight(float x, float scale, float ref) {
  return __builtin_amdgcn_exp2f(CAREFUL ? mul(x, scale) - ref : fmaf(x, scale, -ref));
}
__device__ __forceinline__ bool finite_f32(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
// p is held as 2^(kUp + logit - maximum), the maximum moves when a tile's passes it by kSlack.
// bf16 has fp32's range; in f16 what is small beside the largest then stays normal down to 2^-24
// of it, and p below 2^15.
template <typename Tag>
constexpr float kUp = __is_same(Tag, F16) ? 10.0f : 0.0f;
template <typename Tag>
constexpr float kSlack = __is_same(Tag, F16) ? 5.0f : 8.0f;
// Bit 15 of each half that is Inf or NaN.
template <typename Tag>
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) {
  constexpr uint32_t kExp = __is_same(Tag, BF16) ? 0x7f807f80u : 0x7c007c00u, kOne = __is_same(Tag, BF16) ? 0x00800080u : 0x04000400u;
  return ((w & kExp) + kOne) & 0x80008000u;
}

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

// ---------------------------------------------------------------------------
// 16-bit inputs: 16x16x32 products.  P is rounded to the inputs' type for the second
// one and for the sum it is divided by (an output of that type holds no more).
//
// What a query does not see must not reach it, NaN and Inf included.  Keys are
// masked by a select of the logit.  In V a product with a p of 0 would carry them, which
// shows in the result: a block whose result is not finite is run again with V's
// non-finite elements taken out of the product and added to the rows that see them.
//
// Bound by the products and, in turn with them, the softmax: 32768 tokens, 32 heads on 8 of 128,
// window 2048, 1073 GFLOP of pairs that are seen, take 1.11-1.14 ms, 0.94-0.97 PFLOP/s where a
// large product reaches 1.2; the matrix units are busy in 45 of 100 cycles.  (A tenth more with
// whole tiles in one loop with the others than with a loop of their own.)
// ---------------------------------------------------------------------------
template <typename Tag, int D, int QT>
__global__ __launch_bounds__(kNT, D >= 128 ? 2 : QT == 2 ? 3 : 4) void window_kernel(Win a) {
  using raw = typename Tag::raw;
  using M = Mfma16x16x32<Tag>;
  // Keys of a tile: at D = 256 half as many let two blocks share a compute unit (11 sequences of
  // 543 tokens, 4 heads: 30 us with 64 keys, 23 with 32).  A lane has E logits of one query.
  constexpr int KT = D == 256 ? 32 : 64, NJ = KT / 16, E = 4 * NJ;
  using L = TileLds<D, KT>;
  constexpr int TQ = 64 * QT, NKS = D / 32, NDT = D / 16;
  constexpr int KJ = D == 256 ? 1 : NJ;          // 16-key tiles whose K fragments are read at once
  constexpr int PW = L::BYTES / 1024 / (kNT / kWave);
  __shared__ __align__(16) uint8_t k0[L::BYTES], k1[L::BYTES], v0[L::BYTES], v1[L::BYTES];

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = lane_id(), g = lane >> 4, c16 = lane & 15;
  int t0, h, hk;
  int64_t b;
  place<TQ>(a, t0, b, h, hk);
  const Walk walk = walk_in<TQ, KT>(a, b, t0);
  const int T = a.T, n = walk.n, window = a.window, sinks = a.sinks;
  const int tw = t0 + 16 * QT * wave, wave_last = min(tw + 16 * QT - 1, n - 1);
  raw* const out = static_cast<raw*>(a.out) + (b * T * a.HQ + h) * D;

  const raw* Qb = static_cast<const raw*>(a.Q) + b * T * a.ldq + static_cast<int64_t>(h) * D;
  const char* const kbase = reinterpret_cast<const char*>(static_cast<const raw*>(a.K) + b * T * a.ldk + static_cast<int64_t>(hk) * D);
  const char* const vbase = reinterpret_cast<const char*>(static_cast<const raw*>(a.V) + b * T * a.ldv + static_cast<int64_t>(hk) * D);
  const uint32_t krow = static_cast<uint32_t>(a.ldk) * 2u, vrow = static_cast<uint32_t>(a.ldv) * 2u;
  uint32_t koff[PW], voff[PW];  // of this wave's 16-byte chunks within a tile
#pragma unroll
  for (int i = 0; i < PW; ++i) {
    const int P = (wave * PW + i) * 64 + lane, r = P / L::NCH, pc = P % L::NCH;
    koff[i] = static_cast<uint32_t>(r) * krow + 16u * static_cast<uint32_t>(pc ^ L::swz_k(r));
    voff[i] = static_cast<uint32_t>(r) * vrow + 16u * static_cast<uint32_t>(pc ^ L::swz_v(r));
  }
  // rows past the sequence read as zeros
  auto fetch = [&](int kt, DSA_LDS uint8_t* kd, DSA_LDS uint8_t* vd) __attribute__((always_inline)) {
    dma_tile<PW>(rows_rsrc(kbase, kt * KT, n, krow), koff, kd, wave);
    dma_tile<PW>(rows_rsrc(vbase, kt * KT, n, vrow), voff, vd, wave);
  };
  DSA_LDS uint8_t* const kl0 = (DSA_LDS uint8_t*)k0;
  DSA_LDS uint8_t* const kl1 = (DSA_LDS uint8_t*)k1;
  DSA_LDS uint8_t* const vl0 = (DSA_LDS uint8_t*)v0;
  DSA_LDS uint8_t* const vl1 = (DSA_LDS uint8_t*)v1;

  u32x4 qf[QT][NKS];
  int tq[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    tq[qt] = tw + 16 * qt + c16;
    const raw* q = Qb + min(tq[qt], T - 1) * a.ldq;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qf[qt][ks] = *reinterpret_cast<const u32x4*>(q + 32 * ks + 8 * g) ^ a.flip;
  }
  int kofs[NKS], vofs[NDT];  // LDS reads within a tile
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) kofs[ks] = c16 * (2 * D) + 16 * ((4 * ks + g) ^ L::swz_k(c16));
  {
    const int vr = 4 * g + (c16 >> 2);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
      vofs[dt] = vr * (2 * D) + 16 * ((2 * dt + ((c16 & 3) >> 1)) ^ L::swz_v(vr)) + 8 * (c16 & 1);
  }

  f32x4 o[NDT][QT];
  float m[QT], lpart[QT];
  auto run = [&](auto careful) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(careful)::value;
    constexpr int VG = NDT < 4 || CAREFUL ? 2 : 4;  // 16-dim tiles whose V fragments are read at once
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      m[qt] = -INFINITY;
      lpart[qt] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[dt][qt] = f32x4{0, 0, 0, 0};
    }
    auto compute = [&](auto masked, int s0, const DSA_LDS uint8_t* kl, const DSA_LDS uint8_t* vl) __attribute__((always_inline)) {
      constexpr bool MASKED = decltype(masked)::value;
      f32x4 st[NJ][QT];
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int jp = 0; jp < NJ; jp += KJ) {
        u32x4 ka[KJ][NKS];
#pragma unroll
        for (int jj = 0; jj < KJ; ++jj)
#pragma unroll
          for (int ks = 0; ks < NKS; ++ks)
            ka[jj][ks] = *reinterpret_cast<const DSA_LDS u32x4*>(kl + kofs[ks] + 16 * (jp + jj) * (2 * D));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int jj = 0; jj < KJ; ++jj) {
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) st[jp + jj][qt] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) st[jp + jj][qt] = M::run(ka[jj][ks], qf[qt][ks], st[jp + jj][qt]);
        }
      }
      __builtin_amdgcn_s_setprio(0);
      u32x4 pf[QT][NJ / 2];
      bool grow = false;
      float alpha[QT];
      uint32_t ok[QT];  // bit 4j + r: key s0 + 16j + 4g + r is seen
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        float mx = -INFINITY;
        ok[qt] = 0xffffu;
        if constexpr (MASKED) {
          const int far = tq[qt] - s0 - 4 * g, near = far - window, sink = sinks - s0 - 4 * g;
          if constexpr (CAREFUL) {
            ok[qt] = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const int s = 16 * (e >> 2) + (e & 3);
              ok[qt] |= s <= far && (s > near || s < sink) ? 1u << e : 0u;
              st[e >> 2][qt][e & 3] = ok[qt] >> e & 1u ? st[e >> 2][qt][e & 3] : -INFINITY;
            }
          } else if (s0 >= sinks) {  // near < s <= far in one comparison
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const int s = 16 * (e >> 2) + (e & 3);
              st[e >> 2][qt][e & 3] = static_cast<uint32_t>(far - s) < static_cast<uint32_t>(window) ? st[e >> 2][qt][e & 3] : -INFINITY;
            }
          } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const int s = 16 * (e >> 2) + (e & 3);
              st[e >> 2][qt][e & 3] = s <= far && (s > near || s < sink) ? st[e >> 2][qt][e & 3] : -INFINITY;
            }
          }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) mx = fmaxf(mx, st[e >> 2][qt][e & 3]);
        mx = mul(max_xor32(max_xor16(mx)), a.scale_log2);
        const bool up = mx > m[qt] + kSlack<Tag>;
        const float m_new = up ? mx : m[qt];
        alpha[qt] = up ? __builtin_amdgcn_exp2f(m[qt] - m_new) : 1.f;
        grow |= up && m[qt] != -INFINITY;
        m[qt] = m_new;
        const float ref = m_new == -INFINITY ? 0.f : m_new - kUp<Tag>;
#pragma unroll
        for (int e = 0; e < E; ++e) st[e >> 2][qt][e & 3] = weight<CAREFUL>(st[e >> 2][qt][e & 3], a.scale_log2, ref);
#pragma unroll
        for (int jj = 0; jj < NJ / 2; ++jj)
          pf[qt][jj] = u32x4{M::pack(st[2 * jj][qt][0], st[2 * jj][qt][1]), M::pack(st[2 * jj][qt][2], st[2 * jj][qt][3]),
                             M::pack(st[2 * jj + 1][qt][0], st[2 * jj + 1][qt][1]), M::pack(st[2 * jj + 1][qt][2], st[2 * jj + 1][qt][3])};
      }
      if (ballot(grow)) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          lpart[qt] *= alpha[qt];
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) o[dt][qt] *= alpha[qt];
        }
      }
#pragma unroll
      for (int jj = 0; jj < NJ / 2; ++jj)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) lpart[qt] = M::dot2_ones(pf[qt][jj][e], lpart[qt]);
      uint32_t odd = 0;
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int dg = 0; dg < NDT; dg += VG) {
        u32x4 vfrag[VG][NJ / 2];
#pragma unroll
        for (int d = 0; d < VG; ++d)
#pragma unroll
          for (int jj = 0; jj < NJ / 2; ++jj) {
            const DSA_LDS uint8_t* va = vl + vofs[dg + d] + 32 * jj * (2 * D);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DSA_LDS s16x4*)va);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DSA_LDS s16x4*)(va + 16 * (2 * D)));
            const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
            vfrag[d][jj] = u32x4{l2.x, l2.y, h2.x, h2.y};
            if constexpr (CAREFUL) {
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                const uint32_t bad = odd_halves<Tag>(vfrag[d][jj][w]);
                odd |= bad;
                vfrag[d][jj][w] &= ~((bad >> 15) * 0xffffu);
              }
            }
          }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < VG; ++d)
#pragma unroll
          for (int jj = 0; jj < NJ / 2; ++jj)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) o[dg + d][qt] = M::run(vfrag[d][jj], pf[qt][jj], o[dg + d][qt]);
      }
      __builtin_amdgcn_s_setprio(0);
      if constexpr (CAREFUL) {
        if (ballot(odd != 0)) {
          const raw* v = reinterpret_cast<const raw*>(vbase) + static_cast<int64_t>(s0) * a.ldv;
          for (int s = 0; s < min(KT, n - s0); ++s) {  // key s0 + s: lane group s / 4 % 4, entry 4 (s / 16) + s % 4
            const int from = ((s >> 2) & 3) * 16 + c16;
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
              float mine = 0.0f;  // this lane's p of entry 4 (s / 16) + s % 4, as the product took it
#pragma unroll
              for (int e = 0; e < E; ++e) {
                const uint32_t w = pf[qt][e >> 3][(e >> 1) & 3];
                const float pe = to_f32(Tag{}, static_cast<uint16_t>(e & 1 ? w >> 16 : w & 0xffffu));
                mine = e == 4 * (s >> 4) + (s & 3) ? pe : mine;
              }
              const float p = __shfl(mine, from, kWave);
              const bool yes = static_cast<uint32_t>(__shfl(static_cast<int>(ok[qt]), from, kWave)) >> (4 * (s >> 4) + (s & 3)) & 1u;
#pragma unroll
              for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const float x = to_f32(Tag{}, v[s * a.ldv + 16 * dt + 4 * g + r]);
                  if (yes && !finite_f32(x)) o[dt][qt][r] += p * x;
                }
            }
          }
        }
      }
    };
    if (walk.total > 0) fetch(walk.tile(0), kl0, vl0);
    __builtin_amdgcn_sched_barrier(0);
    wait_dma_keep<0>();
    block_sync_lds();
    auto step = [&](auto masked, int v, DSA_LDS uint8_t* kc, DSA_LDS uint8_t* vc, DSA_LDS uint8_t* kn, DSA_LDS uint8_t* vn) __attribute__((always_inline)) {
      if (v + 1 < walk.total) fetch(walk.tile(v + 1), kn, vn);
      __builtin_amdgcn_sched_barrier(0);
      const int s0 = walk.tile(v) * KT;
      if constexpr (!decltype(masked)::value) compute(std::false_type{}, s0, kc, vc);
      else if (s0 <= wave_last && (s0 + KT > tw - window + 1 || s0 < sinks)) compute(std::true_type{}, s0, kc, vc);
      wait_dma_keep<0>();
      block_sync_lds();
    };
    // Tiles that all queries of the block see whole are a loop of their own (in one with the
    // others, the compiler copies O, 64 registers, once a tile).
    const int w0 = walk.whole0, w1 = CAREFUL ? w0 : walk.whole1;
    int v = 0;
    auto edges = [&](int end) __attribute__((always_inline)) {
      for (; v < end; v += 2) {
        step(std::true_type{}, v, kl0, vl0, kl1, vl1);
        if (v + 1 < end) step(std::true_type{}, v + 1, kl1, vl1, kl0, vl0);
      }
    };
    for (int phase = 0; phase < 2; ++phase) {
      edges(phase ? walk.total : min(w0, walk.total));
      if (phase || w1 <= w0) continue;
      for (; v < w1; v += 2) {
        step(std::false_type{}, v, kl0, vl0, kl1, vl1);
        step(std::false_type{}, v + 1, kl1, vl1, kl0, vl0);
      }
    }
  };

  run(std::false_type{});
  bool odd = false;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float l = sum_xor32(sum_xor16(lpart[qt]));
    if (tq[qt] >= n) continue;
    odd |= !(l > 0.0f && finite_f32(l));
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) odd |= !finite_f32(o[dt][qt][r]);
  }
  if (__syncthreads_or(odd)) run(std::true_type{});

#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float l = sum_xor32(sum_xor16(lpart[qt]));
    if (tq[qt] >= T) continue;
    const float inv = tq[qt] < n ? 1.f / l : __builtin_nanf("");  // no token: sees nothing
    raw* to = out + static_cast<int64_t>(tq[qt]) * a.HQ * D;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) store4<Tag>(to + 16 * dt + 4 * g, o[dt][qt] * inv);
  }
}

// ---------------------------------------------------------------------------
// fp32: every operand as three bf16 pieces (8 bits each, to the nearest: 24 together),
// six of the nine products (those dropped are below 2^-25 of the whole) on the 16-bit
// matrix instructions: 96 cycles where the fp32 ones take 256.  K and V are split once for
// a block's queries, on the way into LDS; the next tile's rows wait in registers.
//
// Pieces of Inf are no numbers, and a p of 0 carries a NaN or Inf of V: a block whose result
// is not finite is run again on the fp32 matrix instructions, with V's non-finite elements
// taken out of the product and added to the rows that see them.
//
// Bound by the products: 2 x 4096 tokens, 8 heads of 64, window 1024, 15.0 GFLOP of pairs that are
// seen, take 107 us one after another, 140 TFLOP/s where a large fp32 product reaches 154 (125 in the
// first launches after a pause; 211 on the fp32 instructions); the matrix units are busy in 35 of
// 100 cycles, the rest goes to pieces of K and V (each block makes its own), of p, and the softmax.
// ---------------------------------------------------------------------------
struct Three {
  uint32_t h, m, l;  // two elements' pieces
};
__device__ __forceinline__ Three split3(float x, float y) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  Three t;
  t.h = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), bf16x2));
  x -= __uint_as_float(t.h << 16);
  y -= __uint_as_float(t.h & 0xffff0000u);
  t.m = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), bf16x2));
  x -= __uint_as_float(t.m << 16);
  y -= __uint_as_float(t.m & 0xffff0000u);
  t.l = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), bf16x2));
  return t;
}
// The six products, the small ones first; a chain of them waits for each before it, so callers
// take one of every chain in turn.
constexpr int kProducts = 6;
__device__ constexpr int kLeft[kProducts] = {0, 2, 1, 0, 1, 0}, kRight[kProducts] = {2, 0, 1, 1, 0, 0};

//
// TEAMS = 2, where blocks are so few that each has a compute unit to itself: two teams of four
// waves take every other tile for the same queries and join their sums at the end.
template <int D, int QT, int KT, int TEAMS>
__global__ __launch_bounds__(kNT * TEAMS, TEAMS == 2 || D * QT >= 256 ? 1 : 2) void window_f32_kernel(Win a) {
  using L = TileLds<D, KT>;
  using M = Mfma16x16x32<BF16>;
  constexpr int TQ = 64 * QT, NKS = D / 32, NDT = D / 16, NJ = KT / 16;
  constexpr int PER = KT * D / 8 / kNT;  // 8-element chunks of a tile a thread, of K and of V
  constexpr int LD = D + 4;              // fp32 rows of the careful pass
  static_assert(PER >= 1 && 16 * LD * 4 <= 3 * L::BYTES);
  __shared__ __align__(16) uint8_t k_lds[TEAMS * 3 * L::BYTES], v_lds[TEAMS * 3 * L::BYTES];
  const int team = TEAMS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kNT);
  uint8_t* const kl = k_lds + team * 3 * L::BYTES;
  uint8_t* const vl = v_lds + team * 3 * L::BYTES;
  const int tid = TEAMS == 1 ? threadIdx.x : threadIdx.x % kNT, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = lane_id(), g = lane >> 4, c16 = lane & 15;
  int t0, h, hk;
  int64_t b;
  place<TQ>(a, t0, b, h, hk);
  const Walk walk = walk_in<TQ, KT>(a, b, t0);
  const int T = a.T, n = walk.n, window = a.window, sinks = a.sinks;
  const int tw = t0 + 16 * QT * wave, wave_last = min(tw + 16 * QT - 1, n - 1);
  const float* const kb = static_cast<const float*>(a.K) + b * T * a.ldk + static_cast<int64_t>(hk) * D;
  const float* const vb = static_cast<const float*>(a.V) + b * T * a.ldv + static_cast<int64_t>(hk) * D;
  const float* const qb = static_cast<const float*>(a.Q) + b * T * a.ldq + static_cast<int64_t>(h) * D;

  f32x4 kx[PER][2], vx[PER][2];
  auto fetch = [&](int kt) __attribute__((always_inline)) {  // rows past the sequence: zeros
    const __amdgpu_buffer_rsrc_t kr = rows_rsrc(reinterpret_cast<const char*>(kb), kt * KT, n, static_cast<uint32_t>(a.ldk) * 4u);
    const __amdgpu_buffer_rsrc_t vr = rows_rsrc(reinterpret_cast<const char*>(vb), kt * KT, n, static_cast<uint32_t>(a.ldv) * 4u);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = tid + i * kNT, r = c / L::NCH, d = c % L::NCH * 32;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        kx[i][e] = buffer_load_f32x4(kr, static_cast<int>(r * static_cast<uint32_t>(a.ldk) * 4u) + d + 16 * e, 0, 0);
        vx[i][e] = buffer_load_f32x4(vr, static_cast<int>(r * static_cast<uint32_t>(a.ldv) * 4u) + d + 16 * e, 0, 0);
      }
    }
  };
  auto split = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = tid + i * kNT, r = c / L::NCH, ch = c % L::NCH;
      u32x4 k3[3], v3[3];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Three k = split3(kx[i][e >> 1][2 * (e & 1)], kx[i][e >> 1][2 * (e & 1) + 1]);
        const Three v = split3(vx[i][e >> 1][2 * (e & 1)], vx[i][e >> 1][2 * (e & 1) + 1]);
        k3[0][e] = k.h; k3[1][e] = k.m; k3[2][e] = k.l;
        v3[0][e] = v.h; v3[1][e] = v.m; v3[2][e] = v.l;
      }
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        *reinterpret_cast<u32x4*>(kl + p * L::BYTES + r * 2 * D + 16 * (ch ^ L::swz_k(r))) = k3[p];
        *reinterpret_cast<u32x4*>(vl + p * L::BYTES + r * 2 * D + 16 * (ch ^ L::swz_v(r))) = v3[p];
      }
    }
  };

  if (team < walk.total) fetch(walk.tile(team));
  u32x4 q[QT][NKS][3];
  int tq[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    tq[qt] = tw + 16 * qt + c16;
    const float* src = qb + min(tq[qt], T - 1) * a.ldq + 8 * g;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      float x[8];
      load_f32<8>(src + 32 * ks, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Three t = split3(__uint_as_float(__float_as_uint(x[2 * e]) ^ a.flip), __uint_as_float(__float_as_uint(x[2 * e + 1]) ^ a.flip));
        q[qt][ks][0][e] = t.h; q[qt][ks][1][e] = t.m; q[qt][ks][2][e] = t.l;
      }
    }
  }
  f32x4 o[NDT][QT];
  float m[QT], l[QT];
  auto clear = [&]() {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      m[qt] = -INFINITY;
      l[qt] = 0.0f;
#pragma unroll
      for (int d = 0; d < NDT; ++d) o[d][qt] = f32x4{0, 0, 0, 0};
    }
  };
  // Logits of nj 16-key tiles from s0 on into exponentials (of one: the careful pass), the sums
  // scaled by what the maximum moves.
  auto weigh = [&](auto nj, auto& st, uint32_t& ok, bool inner, int qt, int s0) __attribute__((always_inline)) {
    constexpr int E = 4 * decltype(nj)::value;
    ok = 0xffffu;
    if (!inner) {
      ok = 0;
      const int far = tq[qt] - s0 - 4 * g, near = far - window, sink = sinks - s0 - 4 * g;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int s = 16 * (e >> 2) + (e & 3);
        ok |= s <= far && (s > near || s < sink) ? 1u << e : 0u;
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (!inner) st[e >> 2][e & 3] = ok >> e & 1u ? st[e >> 2][e & 3] : -INFINITY;
      top = fmaxf(top, st[e >> 2][e & 3]);
    }
    top = mul(max_xor32(max_xor16(top)), a.scale_log2);
    if (ballot(top > m[qt] + 8.f)) {
      const float next = fmaxf(m[qt], top);
      const float fall = m[qt] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[qt] - next);
      m[qt] = next;
      l[qt] *= fall;
#pragma unroll
      for (int d = 0; d < NDT; ++d) o[d][qt] *= fall;
    }
    const float ref = m[qt] == -INFINITY ? 0.0f : m[qt];
#pragma unroll
    for (int e = 0; e < E; ++e) st[e >> 2][e & 3] = weight<E == 4>(st[e >> 2][e & 3], a.scale_log2, ref);
#pragma unroll
    for (int e = 0; e < E; ++e) l[qt] += st[e >> 2][e & 3];
  };
  auto seen = [&](int s0, int s1) { return s0 <= wave_last && (s1 > tw - window || s0 < sinks); };
  auto all_see = [&](int s0, int s1) { return s1 <= tw && (s0 > wave_last - window || s1 < sinks); };

  clear();
  for (int v0 = 0; v0 < walk.total; v0 += TEAMS) {
    const int v = v0 + team, s0 = walk.tile(v) * KT, s1 = s0 + KT - 1;
    block_sync_lds();  // the last tile has been read
    if (v < walk.total) split();
    if (v + TEAMS < walk.total) fetch(walk.tile(v + TEAMS));
    block_sync_lds();
    if (v >= walk.total || !seen(s0, s1)) continue;
    const bool inner = all_see(s0, s1);
    f32x4 st[QT][NJ];
    __builtin_amdgcn_s_setprio(1);
    const DSA_LDS uint8_t* const kp = (const DSA_LDS uint8_t*)kl + c16 * 2 * D;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) st[qt][j] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
      for (int j0 = 0; j0 < NJ; j0 += 2) {
        u32x4 x[2][3];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int p = 0; p < 3; ++p)
            x[j][p] = *reinterpret_cast<const DSA_LDS u32x4*>(kp + p * L::BYTES + 16 * (j0 + j) * 2 * D + 16 * ((4 * ks + g) ^ L::swz_k(c16)));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < kProducts; ++e)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) st[qt][j0 + j] = M::run(x[j][kLeft[e]], q[qt][ks][kRight[e]], st[qt][j0 + j]);
      }
    __builtin_amdgcn_s_setprio(0);
    u32x4 p3[QT][NJ / 2][3];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      uint32_t ok;
      weigh(std::integral_constant<int, NJ>{}, st[qt], ok, inner, qt, s0);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const Three t = split3(st[qt][j][2 * e], st[qt][j][2 * e + 1]);
          const int w = 2 * (j & 1) + e;
          p3[qt][j >> 1][0][w] = t.h; p3[qt][j >> 1][1][w] = t.m; p3[qt][j >> 1][2][w] = t.l;
        }
    }
    __builtin_amdgcn_s_setprio(1);
    const int vr = 4 * g + (c16 >> 2);
    const DSA_LDS uint8_t* const vp = (const DSA_LDS uint8_t*)vl + vr * 2 * D + 8 * (c16 & 1);
    constexpr int DG = QT == 1 ? 4 : 2;  // 16-dim tiles in turn
    static_assert(NDT % 2 == 0);
#pragma unroll
    for (int d0 = 0; d0 < NDT; d0 += DG)
#pragma unroll
      for (int jj = 0; jj < NJ / 2; ++jj) {
        u32x4 x[DG][3];
#pragma unroll
        for (int d = 0; d < DG; ++d)
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            if (d0 + d >= NDT) continue;
            const DSA_LDS uint8_t* at = vp + p * L::BYTES + 32 * jj * 2 * D + 16 * ((2 * (d0 + d) + ((c16 & 3) >> 1)) ^ L::swz_v(vr));
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DSA_LDS s16x4*)at);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DSA_LDS s16x4*)(at + 16 * 2 * D));
            const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
            x[d][p] = u32x4{l2.x, l2.y, h2.x, h2.y};
          }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < kProducts; ++e)
#pragma unroll
          for (int d = 0; d < DG; ++d)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
              if (d0 + d < NDT) o[d0 + d][qt] = M::run(x[d][kLeft[e]], p3[qt][jj][kRight[e]], o[d0 + d][qt]);
      }
    __builtin_amdgcn_s_setprio(0);
  }

  if constexpr (TEAMS == 2) {
    static_assert(QT == 1 && NDT * kNT * 16 <= TEAMS * 3 * L::BYTES);
    f32x4* const other_o = reinterpret_cast<f32x4*>(k_lds);
    float2* const other = reinterpret_cast<float2*>(v_lds);
    __syncthreads();
    if (team == 1) {
#pragma unroll
      for (int d = 0; d < NDT; ++d) other_o[d * kNT + tid] = o[d][0];
      other[tid] = make_float2(m[0], l[0]);
    }
    __syncthreads();
    if (team == 0) {
      const float2 x = other[tid];
      const float top = fmaxf(m[0], x.x), ref = top == -INFINITY ? 0.0f : top;
      const float f = __builtin_amdgcn_exp2f(m[0] - ref), g = __builtin_amdgcn_exp2f(x.x - ref);
      l[0] = l[0] * f + x.y * g;
#pragma unroll
      for (int d = 0; d < NDT; ++d) o[d][0] = o[d][0] * f + other_o[d * kNT + tid] * g;
    }
  }

  bool odd = false;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    if (team) break;  // its sums are in the first team's
    const float all = sum_xor32(sum_xor16(l[qt]));
    odd |= tq[qt] < n && !(all > 0.0f && finite_f32(all));
#pragma unroll
    for (int d = 0; d < NDT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) odd |= tq[qt] < n && !finite_f32(o[d][qt][r]);
  }
  if (__syncthreads_or(odd)) {
    // 16 keys at a time, fp32 rows as they are.  K-slots: element i of a lane's 16 bytes of K
    // is step i (dims 16kk + 4g + i), token 4g + r is step r of P's.
    float* const kf = reinterpret_cast<float*>(kl);
    float* const vf = reinterpret_cast<float*>(vl);
    clear();
    for (int v = 0; v < walk.total * NJ; ++v) {
      const int s0 = walk.tile(v / NJ) * KT + v % NJ * 16, s1 = s0 + 15;
      __syncthreads();
      for (int i = tid; i < 16 * D / 4; i += kNT) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        f32x4 x{0, 0, 0, 0}, y{0, 0, 0, 0};
        if (s0 + r < n) {
          x = *reinterpret_cast<const f32x4*>(kb + (s0 + r) * a.ldk + d);
          y = *reinterpret_cast<const f32x4*>(vb + (s0 + r) * a.ldv + d);
        }
        *reinterpret_cast<f32x4*>(kf + r * LD + d) = x;
        *reinterpret_cast<f32x4*>(vf + r * LD + d) = y;
      }
      __syncthreads();
      if (!seen(s0, s1)) continue;
      const bool inner = all_see(s0, s1);
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const float* src = qb + min(tq[qt], T - 1) * a.ldq + 4 * g;
        f32x4 st[1] = {f32x4{0, 0, 0, 0}};
        for (int kk = 0; kk < D / 16; ++kk) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(kf + c16 * LD + 16 * kk + 4 * g);
          const f32x4 y = *reinterpret_cast<const f32x4*>(src + 16 * kk);
#pragma unroll
          for (int i = 0; i < 4; ++i) st[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], __uint_as_float(__float_as_uint(y[i]) ^ a.flip), st[0], 0, 0, 0);
        }
        uint32_t ok;
        weigh(std::integral_constant<int, 1>{}, st, ok, inner, qt, s0);
        bool bad = false;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int d = 0; d < NDT; ++d) {
            const float x = vf[(4 * g + r) * LD + 16 * d + c16];
            bad |= !finite_f32(x);
            o[d][qt] = __builtin_amdgcn_mfma_f32_16x16x4f32(finite_f32(x) ? x : 0.0f, st[0][r], o[d][qt], 0, 0, 0);
          }
        if (!ballot(bad)) continue;
        for (int s = 0; s < min(16, n - s0); ++s) {
          const int from = (s >> 2) * 16 + c16, e0 = s & 3;
          const float mine = e0 == 0 ? st[0][0] : e0 == 1 ? st[0][1] : e0 == 2 ? st[0][2] : st[0][3];
          const float p = __shfl(mine, from, kWave);
          const bool yes = static_cast<uint32_t>(__shfl(static_cast<int>(ok), from, kWave)) >> e0 & 1u;
#pragma unroll
          for (int d = 0; d < NDT; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float x = vf[s * LD + 16 * d + 4 * g + r];
              if (yes && !finite_f32(x)) o[d][qt][r] += p * x;
            }
        }
      }
    }
  }

  if (team) return;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float sum = sum_xor32(sum_xor16(l[qt]));
    if (tq[qt] >= T) continue;
    const float inv = tq[qt] < n ? 1.0f / sum : __builtin_nanf("");
    float* to = static_cast<float*>(a.out) + ((b * T + tq[qt]) * a.HQ + h) * D;
#pragma unroll
    for (int d = 0; d < NDT; ++d) store4<F32>(to + 16 * d + 4 * g, o[d][qt] * inv);
  }
}

// 128 queries a block where that leaves four blocks a compute unit, else 64 (us with 128 / 64,
// bf16: 8 heads of 128, 2048 tokens, window 1024 33.6 / 22.3; 16 of 64, 4 x 1777, window 500
// 32.8 / 31.0; 32 on 8 of 128, 4096 tokens, window 1024 84 / 93).
// fp32, whose tiles take longer to make, needs two (8 heads of 64, 2 x 4096 tokens, window 1024:
// 109 / 133).
bool wide_tiles(const Win& w, int a_unit) {
  return blocks_of<128>(w) >= a_unit * int64_t{device_cus() > 0 ? device_cus() : 256};
}

template <typename Tag, int D>
void launch_16(const Win& w, hipStream_t stream) {
  if constexpr (D <= 128)  // registers
    if (wide_tiles(w, 4)) return (void)(window_kernel<Tag, D, 2><<<static_cast<uint32_t>(blocks_of<128>(w)), kNT, 0, stream>>>(w));
  window_kernel<Tag, D, 1><<<static_cast<uint32_t>(blocks_of<64>(w)), kNT, 0, stream>>>(w);
}
template <int D, int KT>
void launch_32(const Win& w, hipStream_t stream) {
  if constexpr (D <= 64)  // registers
    if (wide_tiles(w, 2)) return (void)(window_f32_kernel<D, 2, KT, 1><<<static_cast<uint32_t>(blocks_of<128>(w)), kNT, 0, stream>>>(w));
  const uint32_t blocks = static_cast<uint32_t>(blocks_of<64>(w));
  // one / two teams, us: 8 heads of 128, 2 x 1000 tokens 77 / 56, 4 heads of 64, 2 x 438 tokens 23 / 18;
  // past a block a compute unit the other block is the better neighbour (512 blocks of 128: 58 / 65)
  if constexpr (D <= 128)  // LDS
    if (w.T > KT && blocks <= static_cast<uint32_t>(device_cus() > 0 ? device_cus() : 256)) return (void)(window_f32_kernel<D, 1, KT, 2><<<blocks, 2 * kNT, 0, stream>>>(w));
  window_f32_kernel<D, 1, KT, 1><<<blocks, kNT, 0, stream>>>(w);
}
template <int D>
hipError_t launch_dims(const Win& w, int dtype, hipStream_t stream) {
  if (dtype == 1) launch_16<BF16, D>(w, stream);
  else if (dtype == 2) launch_16<F16, D>(w, stream);
  else launch_32<D, (D <= 64 ? 64 : 32)>(w, stream);
  return hipGetLastError();
}

}  // namespace

bool window_attn_supported(int D) { return D == 32 || D == 64 || D == 128 || D == 256; }

hipError_t launch_window_attn(const WindowArgs& a, int dtype, hipStream_t stream) {
  if (a.B == 0 || a.T == 0) return hipSuccess;
  Win w;
  w.Q = a.Q;
  w.K = a.K;
  w.V = a.V;
  w.out = a.out;
  w.count = a.count;
  w.B = a.B;
  w.ldq = a.ldq;
  w.ldk = a.ldk;
  w.ldv = a.ldv;
  w.T = a.T;
  w.HQ = a.HQ;
  w.HKV = a.HKV;
  w.G = a.HQ / a.HKV;
  w.window = a.window;
  w.sinks = a.sinks;
  w.scale_log2 = std::max(std::fabs(a.scale * 1.4426950408889634f), 0x1p-126f);
  w.flip = a.scale < 0.0f ? dtype == 0 ? 0x80000000u : 0x80008000u : 0u;
  switch (a.D) {
    case 32: return launch_dims<32>(w, dtype, stream);
    case 64: return launch_dims<64>(w, dtype, stream);
    case 128: return launch_dims<128>(w, dtype, stream);
    default: return launch_dims<256>(w, dtype, stream);
  }
}

}  // namespace dsa
