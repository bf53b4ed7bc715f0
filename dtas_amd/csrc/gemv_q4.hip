// 4-bit weights with group scales for gfx950: products of one row, or of the few rows of a tree of drafted tokens.
//
//   Wq[N, K/8] uint32: element k of a row is bits 4 (k % 8) .. + 3 of word k / 8;  S[N, K/G] fp16, one scale per G = 32, 64 or 128
//   y[m, n] = epilogue(sum_g S[n, g] * sum_{k in g} x[m, k] * (nibble(n, k) - 7))
//
// nibble - 7 is exact in fp16, so a group's sum is formed of exact products in fp32 and scaled once, in fp32: no weight is ever
// rounded.  The epilogue is fp32 as well; its result is rounded once, to the type of y.
#include "dtas_device.h"
#include "dtas_host.h"

namespace dtas {
namespace {

struct Q4Epilogue {
  const half_t* bias;  // [N] or NULL
  const half_t* res1;  // [M, N]: ADD2 kinds
  const half_t* res2;
  int kind;
};

// erfc keeps the tail of a large negative argument, where 1 + erf cancels
__device__ __forceinline__ float gelu_f32(float t) { return 0.5f * t * erfcf(-0.70710678118654752f * t); }

__device__ __forceinline__ void finish_q4(float acc, const Q4Epilogue& ep, void* y, int64_t m, int64_t n, int64_t N) {
  if (ep.bias) acc += static_cast<float>(ep.bias[n]);
  const int64_t at = m * N + n;
  if (ep.kind == DTAS_EPI_BIAS_GELU) acc = gelu_f32(acc);
  if (ep.res1) acc += static_cast<float>(ep.res1[at]) + static_cast<float>(ep.res2[at]);
  if (ep.kind == DTAS_EPI_BIAS_ADD2_CAST_F32) static_cast<float*>(y)[at] = acc;
  else static_cast<half_t*>(y)[at] = static_cast<half_t>(acc);
}

// any alignment: one wavefront per element of y
__global__ void __launch_bounds__(256) gemv_q4_scalar_kernel(const half_t* __restrict__ x, const unsigned char* __restrict__ Wq,
                                                             const half_t* __restrict__ S, Q4Epilogue ep, void* __restrict__ y, int64_t N,
                                                             int64_t K, int group_shift, int64_t total) {
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); t < total; t += static_cast<int64_t>(gridDim.x) * 4) {
    const int64_t m = t / N, n = t % N;
    float acc = 0.f;
    for (int64_t k = threadIdx.x & 63; k < K; k += 64) {
      const int nibble = (Wq[(n * K + k) >> 1] >> (4 * (k & 1))) & 15;
      acc = fmaf(static_cast<float>(x[m * K + k]) * static_cast<float>(nibble - 7),
                 static_cast<float>(S[n * (K >> group_shift) + (k >> group_shift)]), acc);
    }
    acc = wave_sum(acc);
    if ((threadIdx.x & 63) == 0) finish_q4(acc, ep, y, m, n, N);
  }
}

}  // namespace
}  // namespace dtas

extern "C" int dtas_gemv_q4_f16(const void* x, const void* Wq, const void* scale, const void* bias, const void* res1, const void* res2,
                                void* y, int64_t M, int64_t N, int64_t K, int32_t group, int32_t epilogue, void* stream) {
  using namespace dtas;
  clear_error();
  if (M < 0 || N < 0 || K < 0) return fail("gemv_q4: negative extent M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (group != 32 && group != 64 && group != 128) return fail("gemv_q4: scale groups are of 32, 64 or 128 weights, got %d", group);
  if (K % group != 0) return fail("gemv_q4: K must be a multiple of the scale group, %d (K=%lld)", group, (long long)K);
  if (epilogue < DTAS_EPI_BIAS || epilogue > DTAS_EPI_BIAS_GELU) return fail("gemv_q4: unknown epilogue %d", epilogue);
  const bool two = epilogue == DTAS_EPI_BIAS_ADD2 || epilogue == DTAS_EPI_BIAS_ADD2_CAST_F32;
  constexpr int64_t kMost = int64_t{1} << 60;
  if ((K != 0 && (N > kMost / K || M > kMost / K)) || (N != 0 && M > kMost / N)) return fail("gemv_q4: the extents overflow");
  if (M == 0 || N == 0) return 0;
  if (!y || (K > 0 && (!x || !Wq || !scale))) return fail("gemv_q4: NULL buffer");
  if (two != (res1 != nullptr) || two != (res2 != nullptr)) return fail("gemv_q4: residuals go with the epilogues that add them, both of them");
  const int64_t out_bytes = M * N * (epilogue == DTAS_EPI_BIAS_ADD2_CAST_F32 ? 4 : 2);
  if (overlaps(y, out_bytes, Wq, N * (K / 2)) || overlaps(y, out_bytes, x, M * K * 2) || overlaps(y, out_bytes, scale, N * (K / group) * 2) ||
      (bias && overlaps(y, out_bytes, bias, N * 2)) || (two && (overlaps(y, out_bytes, res1, M * N * 2) || overlaps(y, out_bytes, res2, M * N * 2))))
    return fail("gemv_q4: output overlaps an input");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Q4Epilogue ep{static_cast<const half_t*>(bias), static_cast<const half_t*>(res1), static_cast<const half_t*>(res2), epilogue};
  const half_t* xp = static_cast<const half_t*>(x);
  const half_t* sp = static_cast<const half_t*>(scale);
  const int group_shift = group == 32 ? 5 : group == 64 ? 6 : 7;
  const int64_t grid = ceil_div(M * N, 4) < (int64_t{1} << 20) ? ceil_div(M * N, 4) : int64_t{1} << 20;
  hipLaunchKernelGGL(gemv_q4_scalar_kernel, dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, xp, static_cast<const unsigned char*>(Wq), sp, ep,
                     y, N, K, group_shift, M * N);
  return check_launch("gemv_q4");
}
