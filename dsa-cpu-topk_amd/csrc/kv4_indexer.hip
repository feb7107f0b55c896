// kv4_indexer.hip -- lightning indexer of new tokens against the cached index
// keys (gfx950):
//   I[b,t,s] = sum_j w[b,t,j] * ReLU(<q[b,t,j,:], k[b,s,:]>)  for visible s, else -inf
#include "kv4.h"

namespace dsa {
namespace {

constexpr int kNT = 256;

// One thread a slot, the query row in LDS head by head.
template <typename Tag>
__global__ __launch_bounds__(kNT) void indexer_kernel(Kv4 c, const typename Tag::raw* __restrict__ q,
                                                      const typename Tag::raw* __restrict__ w,
                                                      const int32_t* __restrict__ count, int Tq, int HI,
                                                      int64_t span, float* __restrict__ scores) {
  __shared__ float qs[256];
  const int64_t bt = blockIdx.y, b = bt / Tq;
  const int64_t s = static_cast<int64_t>(blockIdx.x) * kNT + threadIdx.x;
  const int32_t seen = kv4_visible(c.length, count, b, c.S, static_cast<int>(bt % Tq), Tq);
  const bool ok = s < seen && s < span;
  const typename Tag::raw* k = static_cast<const typename Tag::raw*>(c.k_idx) + (b * c.S + (ok ? s : 0)) * c.DI;
  float total = 0.0f;
  for (int j = 0; j < HI; ++j) {
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < c.DI) qs[threadIdx.x] = to_f32(Tag{}, q[(bt * HI + j) * c.DI + threadIdx.x]);
    __syncthreads();
    float dot = 0.0f;
    if (ok)
      for (int d = 0; d < c.DI; ++d) dot += qs[d] * to_f32(Tag{}, k[d]);
    total += to_f32(Tag{}, w[bt * HI + j]) * relu_f32(dot);
  }
  if (s < span) scores[bt * span + s] = ok ? total : -INFINITY;
}

}  // namespace

hipError_t launch_kv4_indexer(const Kv4& c, const void* q, const void* w, int dtype, const int32_t* count,
                              int64_t Tq, int HI, int64_t span, float* scores, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>((span + kNT - 1) / kNT), static_cast<uint32_t>(c.B * Tq));
  const int tq = static_cast<int>(Tq);
  if (dtype == 0)
    indexer_kernel<F32><<<grid, kNT, 0, stream>>>(c, static_cast<const float*>(q), static_cast<const float*>(w), count, tq, HI, span, scores);
  else if (dtype == 1)
    indexer_kernel<BF16><<<grid, kNT, 0, stream>>>(c, static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(w), count, tq, HI, span, scores);
  else
    indexer_kernel<F16><<<grid, kNT, 0, stream>>>(c, static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(w), count, tq, HI, span, scores);
  return hipGetLastError();
}

}  // namespace dsa
