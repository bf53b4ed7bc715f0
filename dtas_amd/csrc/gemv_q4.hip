// 4-bit weights with group scales for gfx950: products of one row, or of the few rows of a tree of drafted tokens.
//
//   Wq[N, K/8] uint32: element k of a row is bits 4 (k % 8) .. + 3 of word k / 8;  S[N, K/G] fp16, one scale per G = 32, 64 or 128
//   y[m, n] = epilogue(sum_g S[n, g] * sum_{k in g} x[m, k] * (nibble(n, k) - 7))
//
// nibble - 7 is exact in fp16, so a group's sum is formed of exact products in fp32 and scaled once, in fp32: no weight is ever
// rounded.  The epilogue is fp32 as well; its result is rounded once, to the type of y.
#include "gemm_common.h"

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

// ---- rows on 16-byte boundaries: the matrix cores -------------------------------------------------------------------------------
// A wavefront takes 16 NT columns and every W-th chunk of 128 k; the W wavefronts of a workgroup (and the workgroups that share a long K) join their sums at
// the end.  A lane loads 16 bytes of one row of W, 32 weights: the four lanes of a column hold 128.  Two exchanges of halves and two of quarters
// turn the four words around, so that word i of the four lanes is the i-th 32 weights in order, which is an operand of
// v_mfma_f32_16x16x32_f16 once it is fp16.  Seven instructions do that: the bytes' nibbles, even and odd, and four permutes that put
// them into halves.  A nibble as the bits of an fp16 number is nibble * 2^-24, a subnormal, which the matrix cores take as it is: no
// conversion, and the offset goes through them as well, as the accumulator that a first MFMA fills with -7 * 2^-24 * (the sum of x over the group) --
// both exact, and 2^24 is part of the scale.  The group's sum leaves the accumulator with one multiply-add per row of x and group.
// Rows of x lie at 4 (r % 4) + r / 4 of the operand: up to four rows fill one accumulator register of the lanes, up to eight two.
constexpr int kChunk = 128;

__device__ __forceinline__ f16x8 halves_of(unsigned word) {
  const unsigned even = word & 0x0f0f0f0fu, odd = (word >> 4) & 0x0f0f0f0fu;
  const u32x4 h = {__builtin_amdgcn_perm(odd, even, 0x0c040c00u), __builtin_amdgcn_perm(odd, even, 0x0c050c01u),
                   __builtin_amdgcn_perm(odd, even, 0x0c060c02u), __builtin_amdgcn_perm(odd, even, 0x0c070c03u)};
  return __builtin_bit_cast(f16x8, h);
}
__device__ __forceinline__ void turn(u32x4& w) {
  unsigned a = w[0], b = w[1], c = w[2], d = w[3];
  const auto ac = __builtin_amdgcn_permlane32_swap(a, c, false, false), bd = __builtin_amdgcn_permlane32_swap(b, d, false, false);
  const auto ab = __builtin_amdgcn_permlane16_swap(ac[0], bd[0], false, false), cd = __builtin_amdgcn_permlane16_swap(ac[1], bd[1], false, false);
  w = u32x4{static_cast<unsigned>(ab[0]), static_cast<unsigned>(ab[1]), static_cast<unsigned>(cd[0]), static_cast<unsigned>(cd[1])};
}

struct Q4Args {
  const half_t* x;
  const unsigned char* Wq;
  const half_t* S;
  void* y;
  int64_t M, N, K;
  int splits;
  float* ws;
  unsigned* arrivals;
};

// MT row tiles of x, NT column tiles, JN registers of a tile that hold rows, GS 32-blocks of k to a scale, W wavefronts
template <int MT, int NT, int JN, int GS, int W>
__global__ void __launch_bounds__(64 * W) gemv_q4_kernel(Q4Args a, Q4Epilogue ep) {
  constexpr int kRows = 16 * MT, kCols = 16 * NT, kScales = 4 / GS;
  __shared__ float sums[W][MT][NT][JN][64];
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quarter = lane >> 4, i16 = lane & 15;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kCols, m0 = static_cast<int64_t>(blockIdx.z) * kRows;
  const int64_t chunks = (a.K + kChunk - 1) / kChunk, lo = chunks * blockIdx.y / a.splits, hi = chunks * (blockIdx.y + 1) / a.splits;
  const int64_t groups = a.K / (32 * GS);

  const unsigned char* w_at[NT];
  const half_t* s_at[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int64_t n = n0 + nt * 16 + i16 < a.N ? n0 + nt * 16 + i16 : a.N - 1;  // columns past N repeat the last; never stored
    w_at[nt] = a.Wq + n * (a.K / 2) + quarter * 16;
    s_at[nt] = a.S + n * groups;
  }
  const half_t* x_at[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int64_t r = m0 + mt * 16 + (i16 >> 2) + 4 * (i16 & 3);
    x_at[mt] = a.x + (r < a.M ? r : a.M - 1) * a.K + quarter * 8;  // (rows past M repeat the last; never stored)
  }
  struct Chunk {
    u32x4 w[NT];
    f16x8 x[MT][4];
    half_t s[NT][kScales];
  };
  auto load = [&](Chunk& c, int64_t at) {
    const int64_t k = at * kChunk;
    if (k + kChunk <= a.K) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        c.w[nt] = load_stream(reinterpret_cast<const u32x4*>(w_at[nt] + k / 2));
        __builtin_memcpy(c.s[nt], s_at[nt] + at * kScales, sizeof c.s[nt]);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) c.x[mt][i] = *reinterpret_cast<const f16x8*>(x_at[mt] + k + 32 * i);
    } else {  // the last 32, 64 or 96: what lies behind them is read from the last 32 again and meets zeros of x
      const int blocks = static_cast<int>((a.K - k) / 32);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        c.w[nt] = load_stream(reinterpret_cast<const u32x4*>(w_at[nt] + k / 2 - (quarter < blocks ? 0 : (quarter - blocks + 1) * 16)));
#pragma unroll
        for (int i = 0; i < kScales; ++i) c.s[nt][i] = s_at[nt][at * kScales + i < groups ? at * kScales + i : groups - 1];
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) c.x[mt][i] = i < blocks ? *reinterpret_cast<const f16x8*>(x_at[mt] + k + 32 * i) : f16x8{};
    }
  };
  f32x4 acc[MT][NT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr unsigned short kSeven = 0x8007;  // -7 * 2^-24
  const half_t seven = __builtin_bit_cast(half_t, kSeven);
  const f16x8 offset = {seven, seven, seven, seven, seven, seven, seven, seven};
  auto use = [&](Chunk& c) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) turn(c.w[nt]);
    f32x4 part[MT][NT];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i % GS == 0) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          f32x4 from = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int u = 0; u < GS; ++u) from = __builtin_amdgcn_mfma_f32_16x16x32_f16(c.x[mt][i + u], offset, from, 0, 0, 0);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) part[mt][nt] = from;
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const f16x8 w = halves_of(c.w[nt][i]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) part[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c.x[mt][i], w, part[mt][nt], 0, 0, 0);
      }
      if (i % GS == GS - 1) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float s = static_cast<float>(c.s[nt][i / GS]) * 16777216.f;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < JN; ++j) acc[mt][nt][j] = fmaf(s, part[mt][nt][j], acc[mt][nt][j]);
        }
      }
    }
  };
  Chunk now, next;
  int64_t at = lo + wave;
  if (at < hi) load(now, at);
  for (; at < hi; at += W) {
    if (at + W < hi) load(next, at + W);
    use(now);
    now = next;
  }

  // ---- the wavefronts' sums, in their order; a thread holds output (m, n) of register j, lane l of tile (mt, nt)
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < JN; ++j) sums[wave][mt][nt][j][lane] = acc[mt][nt][j];
  __syncthreads();
  constexpr int kValues = MT * NT * JN * 64;
  const int64_t tile = static_cast<int64_t>(blockIdx.z) * gridDim.x + blockIdx.x;
  float* shares = a.ws + tile * a.splits * kValues;
  auto finish = [&](int v, float sum) {
    const int l = v & 63, j = v / 64 % JN, nt = v / (64 * JN) % NT, mt = v / (64 * JN * NT);
    const int64_t m = m0 + mt * 16 + (l >> 4) + 4 * j, n = n0 + nt * 16 + (l & 15);
    if (m < a.M && n < a.N) finish_q4(sum, ep, a.y, m, n, a.N);
  };
  for (int v = tid; v < kValues; v += 64 * W) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) sum += (&sums[w][0][0][0][0])[v];
    if (a.splits == 1) finish(v, sum);
    else __hip_atomic_store(shares + static_cast<int64_t>(blockIdx.y) * kValues + v, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (a.splits == 1) return;
  // ---- a long K shared by workgroups: their sums pass the L2 (the XCDs' are not coherent) and are counted once they have drained; whoever
  // arrives last adds them up in their order
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const unsigned before = __hip_atomic_fetch_add(a.arrivals + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    flag = before == static_cast<unsigned>(a.splits) - 1;
    if (flag) __hip_atomic_store(a.arrivals + tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // re-armed for the next launch
  }
  __syncthreads();
  if (!flag) return;
  for (int v = tid; v < kValues; v += 64 * W) {
    float sum = 0.f;
    for (int z0 = 0; z0 < a.splits; z0 += 8) {
      float some[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        some[u] = __hip_atomic_load(shares + static_cast<int64_t>(z0 + u < a.splits ? z0 + u : a.splits - 1) * kValues + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
      for (int u = 0; u < 8; ++u) sum += z0 + u < a.splits ? some[u] : 0.f;
    }
    finish(v, sum);
  }
}

template <int MT, int NT, int JN, int GS, int W>
int launch_q4(Q4Args a, const Q4Epilogue& ep, hipStream_t s) {
  const int64_t cols = ceil_div(a.N, 16 * NT), rows = ceil_div(a.M, 16 * MT), tiles = cols * rows, chunks = ceil_div(a.K, kChunk);
  // K shared by workgroups where the columns alone leave CUs idle, at two chunks per wavefront at least
  int64_t splits = kNumCU / tiles;
  const int64_t most = chunks / (2 * W);
  splits = splits > most ? most : splits;
  splits = splits > 16 ? 16 : splits;
  a.splits = static_cast<int>(splits < 1 ? 1 : splits);
  if (cols > INT32_MAX || rows > 65535) return fail("gemv_q4: the launch has too many workgroups");
  std::unique_lock<std::recursive_mutex> lock;
  if (a.splits > 1 && split_scratch(s, static_cast<size_t>(tiles * a.splits) * (MT * NT * JN * 64) * sizeof(float), static_cast<size_t>(tiles), a.splits, &a.ws, &a.arrivals, &lock) != 0)
    return -1;
  hipLaunchKernelGGL((gemv_q4_kernel<MT, NT, JN, GS, W>), dim3(static_cast<unsigned>(cols), static_cast<unsigned>(a.splits), static_cast<unsigned>(rows)), dim3(64 * W), 0, s, a, ep);
  return check_launch("gemv_q4");
}
template <int GS>
int launch_q4_rows(const Q4Args& a, const Q4Epilogue& ep, hipStream_t s) {
  if (a.M <= 4) return launch_q4<1, 1, 1, GS, 4>(a, ep, s);
  if (a.M <= 8) return launch_q4<1, 1, 2, GS, 4>(a, ep, s);
  if (a.M <= 16) return launch_q4<1, 1, 4, GS, 4>(a, ep, s);
  if (a.M <= 32) return launch_q4<2, 2, 4, GS, 4>(a, ep, s);
  return launch_q4<4, 2, 4, GS, 4>(a, ep, s);
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
  if (K > 0 && aligned(x, 16) && aligned(Wq, 16) && M <= 64 * int64_t{65535}) {
    const Q4Args a{xp, static_cast<const unsigned char*>(Wq), sp, y, M, N, K, 1, nullptr, nullptr};
    return group == 32 ? launch_q4_rows<1>(a, ep, s) : group == 64 ? launch_q4_rows<2>(a, ep, s) : launch_q4_rows<4>(a, ep, s);
  }
  const int64_t grid = ceil_div(M * N, 4) < (int64_t{1} << 20) ? ceil_div(M * N, 4) : int64_t{1} << 20;
  hipLaunchKernelGGL(gemv_q4_scalar_kernel, dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, xp, static_cast<const unsigned char*>(Wq), sp, ep,
                     y, N, K, group_shift, M * N);
  return check_launch("gemv_q4");
}
