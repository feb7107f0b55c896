// kv4_attn.hip -- attention of new tokens over the 4-bit decode cache (gfx950):
//   p = softmax over the visible (or listed) slots of <Q, K> * scale
//   O = sum p V,   weight[b, slot] += sum over queries and heads of p
#include "kv4.h"

namespace dsa {
namespace {

constexpr int kNT = 256;

__device__ __forceinline__ int32_t slot_of(const int32_t* slots, int64_t row, int64_t n, int64_t j) {
  return slots ? slots[row * n + j] : static_cast<int32_t>(j);
}

// Logits of one query head: a thread a slot.
template <typename Tag>
__global__ __launch_bounds__(kNT) void logits_kernel(Kv4 c, const typename Tag::raw* __restrict__ Q,
                                                     const int32_t* __restrict__ slots,
                                                     const int32_t* __restrict__ count, int Tq, int HQ,
                                                     int64_t n, float scale, float* __restrict__ logits) {
  __shared__ float q[256];
  const int64_t bt = blockIdx.z, b = bt / Tq, j = static_cast<int64_t>(blockIdx.x) * kNT + threadIdx.x;
  const int h = blockIdx.y, hk = h / (HQ / c.HKV);
  if (static_cast<int>(threadIdx.x) < c.DK) q[threadIdx.x] = to_f32(Tag{}, Q[(bt * HQ + h) * c.DK + threadIdx.x]);
  __syncthreads();
  if (j >= n) return;
  const int32_t seen = kv4_visible(c.length, count, b, c.S, static_cast<int>(bt % Tq), Tq);
  const int32_t s = slot_of(slots, bt, n, j);
  if (s < 0 || s >= seen) return;
  const int64_t slot = b * c.S + s;
  const int u0 = hk * (c.DK + c.DV) / 8;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(c.codes) + slot * c.words() + u0;
  const uint8_t* e = c.scales + slot * c.scale_bytes() + u0 / 4;
  float dot = 0.0f;
  for (int u = 0; u < c.DK / 8; ++u) {
    float x[8];
    e2m1_unpack8(w[u], e8m0(e[u / 4]), x);
#pragma unroll
    for (int i = 0; i < 8; ++i) dot += q[u * 8 + i] * x[i];
  }
  logits[(bt * HQ + h) * n + j] = dot * scale;
}

// Softmax and the sum over V of one query head; its probabilities replace the logits.
__global__ __launch_bounds__(kNT) void rows_kernel(Kv4 c, const int32_t* __restrict__ slots,
                                                   const int32_t* __restrict__ count, int Tq, int HQ,
                                                   int64_t n, float* __restrict__ logits,
                                                   float* __restrict__ out) {
  __shared__ float red[kNT / kWave];
  const int64_t bt = blockIdx.y, b = bt / Tq;
  const int h = blockIdx.x, hk = h / (HQ / c.HKV);
  const int32_t seen = kv4_visible(c.length, count, b, c.S, static_cast<int>(bt % Tq), Tq);
  float* row = logits + (bt * HQ + h) * n;
  auto ok = [&](int64_t j) {
    const int32_t s = slot_of(slots, bt, n, j);
    return s >= 0 && s < seen;
  };
  float m = -INFINITY;
  for (int64_t j = threadIdx.x; j < n; j += kNT)
    if (ok(j)) m = fmaxf(m, row[j]);
  m = wave_max(m);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  if (m == -INFINITY) m = 0.0f;
  __syncthreads();
  float l = 0.0f;
  for (int64_t j = threadIdx.x; j < n; j += kNT)
    if (ok(j)) l += expf(row[j] - m);
  l = wave_sum(l);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = l;
  __syncthreads();
  l = red[0] + red[1] + red[2] + red[3];
  for (int64_t j = threadIdx.x; j < n; j += kNT)
    if (ok(j)) row[j] = expf(row[j] - m) / l;
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= c.DV) return;
  const int u = hk * (c.DK + c.DV) / 8 + (c.DK + d) / 8;
  float o = 0.0f;
  for (int64_t j = 0; j < n; ++j) {
    const int32_t s = slot_of(slots, bt, n, j);
    if (s < 0 || s >= seen) continue;
    const int64_t slot = b * c.S + s;
    float x[8];
    e2m1_unpack8(reinterpret_cast<const uint32_t*>(c.codes)[slot * c.words() + u],
                 e8m0(c.scales[slot * c.scale_bytes() + u / 4]), x);
    float v = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) v = (d & 7) == i ? x[i] : v;
    o += row[j] * v;
  }
  out[(bt * HQ + h) * c.DV + d] = l == 0.0f ? __builtin_nanf("") : o;
}

// weight += the probabilities of query t's heads.  Queries come in launches of
// their own, so that no two of them add to one slot at once; a slot that one
// query lists twice takes the same addend twice, in whatever order.
__global__ __launch_bounds__(kNT) void weight_kernel(Kv4 c, const int32_t* __restrict__ slots,
                                                     const int32_t* __restrict__ count, int t, int Tq,
                                                     int HQ, int64_t n, const float* __restrict__ p) {
  const int64_t b = blockIdx.y, bt = b * Tq + t, j = static_cast<int64_t>(blockIdx.x) * kNT + threadIdx.x;
  if (j >= n) return;
  const int32_t s = slot_of(slots, bt, n, j);
  if (s < 0 || s >= kv4_visible(c.length, count, b, c.S, t, Tq)) return;
  float sum = 0.0f;
  for (int h = 0; h < HQ; ++h) sum += p[(bt * HQ + h) * n + j];
  atomicAdd(c.weight + b * c.S + s, sum);
}

}  // namespace

bool kv4_attn_supported(int DK, int DV) {
  if (DK == 192 && DV == 128) return true;
  return DK == DV && (DK == 32 || DK == 64 || DK == 96 || DK == 128 || DK == 192 || DK == 256);
}

int64_t kv4_attn_workspace(const Kv4& c, int64_t Tq, int HQ, int64_t n, bool) { return c.B * Tq * HQ * n * 4; }

hipError_t launch_kv4_attn(const Kv4& c, const void* Q, int dtype, const int32_t* slots,
                           const int32_t* count, int64_t Tq, int HQ, int64_t n, bool accumulate,
                           float scale, float* out, void* ws, hipStream_t stream) {
  const int tq = static_cast<int>(Tq);
  float* logits = static_cast<float*>(ws);
  const dim3 g1(static_cast<uint32_t>((n + kNT - 1) / kNT), HQ, static_cast<uint32_t>(c.B * Tq));
  if (n > 0) {
    if (dtype == 0)
      logits_kernel<F32><<<g1, kNT, 0, stream>>>(c, static_cast<const float*>(Q), slots, count, tq, HQ, n, scale, logits);
    else if (dtype == 1)
      logits_kernel<BF16><<<g1, kNT, 0, stream>>>(c, static_cast<const uint16_t*>(Q), slots, count, tq, HQ, n, scale, logits);
    else
      logits_kernel<F16><<<g1, kNT, 0, stream>>>(c, static_cast<const uint16_t*>(Q), slots, count, tq, HQ, n, scale, logits);
  }
  rows_kernel<<<dim3(HQ, static_cast<uint32_t>(c.B * Tq)), kNT, 0, stream>>>(c, slots, count, tq, HQ, n, logits, out);
  if (accumulate && n > 0)
    for (int t = 0; t < tq; ++t)
      weight_kernel<<<dim3(static_cast<uint32_t>((n + kNT - 1) / kNT), static_cast<uint32_t>(c.B)), kNT, 0, stream>>>(c, slots, count, t, tq, HQ, n, logits);
  return hipGetLastError();
}

}  // namespace dsa
