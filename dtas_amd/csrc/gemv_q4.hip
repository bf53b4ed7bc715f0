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
// A wavefront takes 16 columns and chunks of 128 k.  A lane loads 16 bytes of one row of W, 32 weights: the four lanes of a column hold a chunk.  Two
// exchanges of halves and two of quarters turn the four words around, so that word i of the four lanes is the i-th 32 weights in order, which is an
// operand of v_mfma_f32_16x16x32_f16 once it is fp16.  Nine instructions do that: a nibble in the low bits of the fp16 number 1024 is 1024 + nibble, or
// 1024 + 16 nibble four bits up; one packed add (or multiply-add) leaves nibble - 7, exactly.  That pairs the weights k and k + 4 of a word, so x lies in
// the LDS in the same order.  (The nibble as a subnormal, its offset through the matrix cores as well, takes fewer instructions and loses the sum's
// low bits: products are aligned by the exponents of their factors, a subnormal's being 2^-14 whatever its size, and ten bits fall off.)
// The group's sum leaves the accumulator with one multiply-add per row of x and group.
// Rows of x lie at 4 (r % 4) + r / 4 of the operand: up to four rows fill one accumulator register of the lanes.
// The scales pass through the LDS: eight bytes of each of sixteen rows, chunk by chunk, take more lines from the caches than W does
// (1 x 50280 x 4096: 34 us).  W's loads are plain: what fits the Infinity Cache is read from there (streamed: 5 .. 10 % longer).
constexpr int kChunk = 128;

// weights 0 4 1 5 2 6 3 7 of a word
__device__ __forceinline__ f16x8 halves_of(unsigned word) {
  constexpr unsigned kLow = 0x000f000fu, kHigh = 0x00f000f0u;
  unsigned k1024 = 0x64006400u;
  asm("" : "+v"(k1024));  // (a register: two constants of one instruction would make it two)
  const f16x2 less = {-1031.f16, -1031.f16}, sixteenth = {0.0625f16, 0.0625f16}, less_high = {-71.f16, -71.f16};
  const unsigned next = word >> 8;
  const f16x2 a = __builtin_bit_cast(f16x2, (word & kLow) | k1024) + less;
  const f16x2 b = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (word & kHigh) | k1024), sixteenth, less_high);
  const f16x2 c = __builtin_bit_cast(f16x2, (next & kLow) | k1024) + less;
  const f16x2 d = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (next & kHigh) | k1024), sixteenth, less_high);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// eight of x in the weights' order
__device__ __forceinline__ u32x4 in_order(u32x4 x) {
  return u32x4{__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
               __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)};
}
__device__ __forceinline__ void turn(u32x4& w) {
  const auto ac = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), bd = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
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

// What a workgroup has of K, counted from its first chunk (the LDS holds all its scales: few)
struct Q4Part {
  int64_t lo;       // its first chunk
  int chunks, len;  // its chunks and k
};
__device__ __forceinline__ Q4Part part_of(const Q4Args& a) {
  const int64_t chunks = (a.K + kChunk - 1) / kChunk, lo = chunks * blockIdx.y / a.splits, hi = chunks * (blockIdx.y + 1) / a.splits;
  const int64_t end = hi * kChunk < a.K ? hi * kChunk : a.K;
  return {lo, static_cast<int>(hi - lo), static_cast<int>(end - lo * kChunk)};
}
// One chunk of a row of W (from the part's first on).  In the last chunk, of 32, 64 or 96, the lanes behind its end read the last 32 again: they meet zeros of x.
__device__ __forceinline__ u32x4 load_w(const unsigned char* row, int chunk, int len, int quarter) {
  const int left = (len - chunk * kChunk) / 32;
  return *reinterpret_cast<const u32x4*>(row + (chunk * (kChunk / 2) + (quarter < left ? quarter : left - 1) * 16));
}
// Scales of `cols` rows from n0 on, of one part of K, into the LDS: a row is an odd number of 8-byte pieces (sixteen rows fall on different banks).
// What lies behind the row's last scale is zero (it meets sums of zero, and the last scale itself may be no number).
template <int GS>
__host__ __device__ constexpr int scale_pitch(int64_t chunks) {
  return static_cast<int>((chunks * (4 / GS) + 3) / 4) | 1;
}
template <int GS, int THREADS>
__device__ __forceinline__ void stage_scales(char* lds, const Q4Args& a, int64_t n0, int cols, const Q4Part& part) {
  constexpr int kScales = 4 / GS;
  const int64_t row = a.K / (32 * GS), first = part.lo * kScales;
  const int pieces = (part.chunks * kScales + 3) / 4, pitch = scale_pitch<GS>(part.chunks);
  const int groups = static_cast<int>(row - first < 4 * pieces ? row - first : 4 * pieces);  // those there are
  for (int t = threadIdx.x; t < cols * pieces; t += THREADS) {
    const int r = t / pieces, c = t % pieces, g = 4 * c;
    const half_t* from = a.S + (n0 + r < a.N ? n0 + r : a.N - 1) * row + first;
    f16x4 v;
    if (g + 4 <= groups) {
      __builtin_memcpy(&v, from + g, 8);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = g + i < groups ? from[g + i] : half_t{0};
    }
    *reinterpret_cast<f16x4*>(lds + (r * pitch + c) * 8) = v;
  }
}
// The products of one chunk for MT row tiles and one column tile, onto acc; x(mt, i): the operand of its i-th 32 k
template <int MT, int JN, int GS, typename X>
__device__ __forceinline__ void multiply(u32x4 w, X x, const char* scales, f32x4 (&acc)[MT]) {
  turn(w);
  half_t s[4 / GS];
  __builtin_memcpy(s, __builtin_assume_aligned(scales, 8 / GS), sizeof s);
#pragma unroll
  for (int g = 0; g < 4 / GS; ++g) {
    f32x4 part[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) part[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < GS; ++u) {
      const f16x8 h = halves_of(w[g * GS + u]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) part[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x(mt, g * GS + u), h, part[mt], 0, 0, 0);
    }
    const float scale = static_cast<float>(s[g]);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < JN; ++j) acc[mt][j] = fmaf(scale, part[mt][j], acc[mt][j]);
  }
}
// Workgroups that share a long K leave their sums in the workspace; they pass the L2 (the XCDs' are not coherent) and are counted once they have drained.
// True for whoever arrives last, and adds them up in their order.
__device__ __forceinline__ bool last_to_arrive(const Q4Args& a, int64_t tile, int* flag) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned before = __hip_atomic_fetch_add(a.arrivals + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = before == static_cast<unsigned>(a.splits) - 1;
    if (*flag) __hip_atomic_store(a.arrivals + tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // re-armed for the next launch
  }
  __syncthreads();
  return *flag != 0;
}

// ---- up to four rows: the W wavefronts of a workgroup share the K of 16 columns, by pairs of chunks (the 128 bytes of a row that make a line), and
// request D chunks before they use the first; x and the scales lie in the LDS.
template <int GS, int W, int D>
__global__ void __launch_bounds__(64 * W) gemv_q4_kernel(Q4Args a, Q4Epilogue ep) {
  static_assert(D % 2 == 0, "pairs");
  __shared__ float sums[W][64];
  __shared__ int flag;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quarter = lane >> 4, i16 = lane & 15, M = static_cast<int>(a.M);
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const Q4Part part = part_of(a);
  const unsigned char* w_at = a.Wq + (n0 + i16 < a.N ? n0 + i16 : a.N - 1) * (a.K / 2) + part.lo * (kChunk / 2);  // columns past N repeat the last; never stored
  u32x4 some[D];
  auto chunk_of = [&](int base, int d) { return base + (d / 2 * W + wave) * 2 + d % 2; };
  auto load_all = [&](int base) {
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (chunk_of(base, d) < part.chunks) some[d] = load_w(w_at, chunk_of(base, d), part.len, quarter);
  };
  load_all(0);
  const int row_bytes = part.chunks * (kChunk * 2), pieces = row_bytes / 16;
  const half_t* x_from = a.x + part.lo * kChunk;
  for (int t = tid; t < pieces * M; t += 64 * W) {
    const int r = t / pieces, c = t % pieces;
    reinterpret_cast<u32x4*>(lds)[t] = c * 8 < part.len ? in_order(*reinterpret_cast<const u32x4*>(x_from + r * a.K + c * 8)) : u32x4{0u, 0u, 0u, 0u};
  }
  char* lds_s = lds + row_bytes * M;
  stage_scales<GS, 64 * W>(lds_s, a, n0, 16, part);
  __syncthreads();
  // row r of x is row 4 r of the operand; the others, never stored, repeat the last
  const char* x_at = lds + ((i16 >> 2) < M ? i16 >> 2 : M - 1) * row_bytes + quarter * 16;
  const char* s_at = lds_s + i16 * scale_pitch<GS>(part.chunks) * 8;
  f32x4 acc[1] = {f32x4{0.f, 0.f, 0.f, 0.f}};
  for (int base = 0; base < part.chunks; base += W * D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int at = chunk_of(base, d);
      if (at >= part.chunks) break;
      multiply<1, 1, GS>(some[d], [&](int, int i) { return *reinterpret_cast<const f16x8*>(x_at + at * (kChunk * 2) + i * 64); }, s_at + at * (8 / GS), acc);
    }
    if (base + W * D < part.chunks) load_all(base + W * D);
  }
  sums[wave][lane] = acc[0][0];
  __syncthreads();
  if (a.splits == 1 && tid >= 64) return;
  float sum = 0.f;
  const int64_t n = n0 + i16;
  float* shares = a.ws + static_cast<int64_t>(blockIdx.x) * a.splits * 64;
  if (tid < 64) {
#pragma unroll
    for (int w = 0; w < W; ++w) sum += sums[w][lane];
    if (a.splits > 1) __hip_atomic_store(shares + blockIdx.y * 64 + lane, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (a.splits > 1) {
    if (!last_to_arrive(a, blockIdx.x, &flag) || tid >= 64) return;
    sum = 0.f;
    for (int z0 = 0; z0 < a.splits; z0 += 8) {
      float part[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) part[u] = __hip_atomic_load(shares + (z0 + u < a.splits ? z0 + u : a.splits - 1) * 64 + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
      for (int u = 0; u < 8; ++u) sum += z0 + u < a.splits ? part[u] : 0.f;
    }
  }
  if (quarter < M && n < a.N) finish_q4(sum, ep, a.y, quarter, n, a.N);
}

// ---- more rows: CT x KG wavefronts, CT column tiles and KG parts of every KG SL chunks.  x passes through the LDS, KG SL chunks at a time in two stages; a
// wavefront requests W's next SL chunks, and its share of x's next stage, before it works on the present ones.
template <int MT, int GS, int CT, int KG, int SL>
__global__ void __launch_bounds__(64 * CT * KG) gemv_q4_rows_kernel(Q4Args a, Q4Epilogue ep) {
  constexpr int W = CT * KG, kRows = 16 * MT, kCols = 16 * CT, kAll = KG * SL, kPitch = kChunk * 2 + 16;  // (the same 16 bytes of sixteen rows fall on different banks)
  constexpr int kStage = kRows * kAll * kPitch, kPieces = kRows * kAll * (kChunk / 8) / (64 * W), kSums = KG * kRows * kCols * 4;
  static_assert(kRows * kAll * (kChunk / 8) % (64 * W) == 0, "whole pieces");
  __shared__ __attribute__((aligned(16))) char lds[2 * kStage > kSums ? 2 * kStage : kSums];
  __shared__ int flag;
  extern __shared__ __attribute__((aligned(16))) char lds_s[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quarter = lane >> 4, i16 = lane & 15;
  const int ct = wave % CT, kg = wave / CT;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kCols, m0 = static_cast<int64_t>(blockIdx.z) * kRows;
  const Q4Part part = part_of(a);
  const int64_t col = n0 + ct * 16 + i16;
  const unsigned char* w_at = a.Wq + (col < a.N ? col : a.N - 1) * (a.K / 2) + part.lo * (kChunk / 2);  // columns past N repeat the last; never stored
  u32x4 w[SL], xr[kPieces];
  const half_t* x_from[kPieces];
  int x_k[kPieces];
#pragma unroll
  for (int n = 0; n < kPieces; ++n) {
    // piece: row, then chunk, then 16 bytes; rows past M repeat the last, never stored
    const int id = n * 64 * W + tid, r = id / (kChunk / 8 * kAll);
    x_k[n] = id % (kChunk / 8 * kAll) * 8;
    x_from[n] = a.x + (m0 + r < a.M ? m0 + r : a.M - 1) * a.K + part.lo * kChunk + x_k[n];
  }
  auto load_all = [&](int base) {
#pragma unroll
    for (int sl = 0; sl < SL; ++sl)
      if (base + kg * SL + sl < part.chunks) w[sl] = load_w(w_at, base + kg * SL + sl, part.len, quarter);
#pragma unroll
    for (int n = 0; n < kPieces; ++n)
      xr[n] = base * kChunk + x_k[n] < part.len ? *reinterpret_cast<const u32x4*>(x_from[n] + base * kChunk) : u32x4{0u, 0u, 0u, 0u};
  };
  auto keep_x = [&](int stage) {
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
      const int id = n * 64 * W + tid, c = id % (kChunk / 8), sl = id / (kChunk / 8) % kAll, r = id / (kChunk / 8 * kAll);
      *reinterpret_cast<u32x4*>(lds + stage * kStage + (sl * kRows + r) * kPitch + c * 16) = in_order(xr[n]);
    }
  };
  load_all(0);
  stage_scales<GS, 64 * W>(lds_s, a, n0, kCols, part);
  keep_x(0);
  __syncthreads();
  const char* s_at = lds_s + (ct * 16 + i16) * scale_pitch<GS>(part.chunks) * 8;
  const char* x_at = lds + (kg * SL * kRows + (i16 >> 2) + 4 * (i16 & 3)) * kPitch + quarter * 16;
  f32x4 acc[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) acc[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  int stage = 0;
  for (int base = 0; base < part.chunks; base += kAll, stage ^= 1) {
    u32x4 now[SL];
#pragma unroll
    for (int sl = 0; sl < SL; ++sl) now[sl] = w[sl];
    const bool more = base + kAll < part.chunks;
    if (more) load_all(base + kAll);
#pragma unroll
    for (int sl = 0; sl < SL; ++sl) {
      const int at = base + kg * SL + sl;
      if (at >= part.chunks) break;
      multiply<MT, 4, GS>(now[sl], [&](int mt, int i) { return *reinterpret_cast<const f16x8*>(x_at + stage * kStage + (sl * kRows + mt * 16) * kPitch + i * 64); },
                          s_at + at * (8 / GS), acc);
    }
    if (more) {
      keep_x(stage ^ 1);
      __syncthreads();
    }
  }
  // the parts of K joined in their order, and into rows of columns
  __syncthreads();
  float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[(kg * kRows + mt * 16 + quarter + 4 * j) * kCols + ct * 16 + i16] = acc[mt][j];
  __syncthreads();
  const int64_t tile = static_cast<int64_t>(blockIdx.z) * gridDim.x + blockIdx.x;
  constexpr int kFours = kRows * kCols / 4, kMine = (kFours + 64 * W - 1) / (64 * W);
  f32x4 sum[kMine];
  auto finish = [&] {
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int at = 4 * (i * 64 * W + tid);
      const int64_t m = m0 + at / kCols, n = n0 + at % kCols;
      if (at >= 4 * kFours || m >= a.M) break;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < a.N) finish_q4(sum[i][j], ep, a.y, m, n + j, a.N);
    }
  };
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int at = 4 * (i * 64 * W + tid);
    if (at >= 4 * kFours) break;
    sum[i] = *reinterpret_cast<const f32x4*>(sums + at);
#pragma unroll
    for (int k = 1; k < KG; ++k) {
      const f32x4 part = *reinterpret_cast<const f32x4*>(sums + k * kRows * kCols + at);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[i][j] += part[j];
    }
  }
  if (a.splits == 1) return finish();
  float* shares = a.ws + tile * a.splits * (kRows * kCols);
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int at = 4 * (i * 64 * W + tid);
    if (at < 4 * kFours) store_out(sum[i], reinterpret_cast<f32x4*>(shares + static_cast<int64_t>(blockIdx.y) * (kRows * kCols) + at), true);
  }
  if (!last_to_arrive(a, tile, &flag)) return;
#pragma unroll
  for (int i = 0; i < kMine; ++i) sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int kAtOnce = kMine >= 8 ? 1 : 8 / kMine;  // splits requested before the first is used: eight 16-byte pieces
  for (int z0 = 0; z0 < a.splits; z0 += kAtOnce) {
    uint64_t part[kAtOnce][kMine][2];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const float* from = shares + static_cast<int64_t>(z0 + u < a.splits ? z0 + u : a.splits - 1) * (kRows * kCols);
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int at = 4 * (i * 64 * W + tid);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          part[u][i][h] = __hip_atomic_load(reinterpret_cast<const uint64_t*>(from + (at < 4 * kFours ? at : 0)) + h, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (z0 + u >= a.splits) break;
#pragma unroll
      for (int i = 0; i < kMine; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] += __builtin_bit_cast(float, static_cast<unsigned>(part[u][i][j / 2] >> (32 * (j % 2))));
    }
  }
  finish();
}

// `cols` x `rows` per workgroup and K shared by workgroups: while the tiles alone are fewer than `fill`, at `least` chunks each, and as the LDS needs it
template <typename Kernel>
int launch_q4(Kernel kernel, Q4Args a, const Q4Epilogue& ep, int cols, int rows, int threads, int values, int64_t fill, int64_t least, int64_t lds_per_chunk, int64_t lds_fixed,
              int64_t lds_most, hipStream_t s) {
  const int64_t across = ceil_div(a.N, cols), down = ceil_div(a.M, rows), tiles = across * down, chunks = ceil_div(a.K, kChunk);
  int64_t splits = fill / tiles;
  splits = splits > chunks / least ? chunks / least : splits;
  splits = splits > 16 ? 16 : splits;
  const int64_t needed = ceil_div(chunks, (lds_most - lds_fixed) / lds_per_chunk);
  splits = splits < needed ? needed : splits;
  splits = splits < 1 ? 1 : splits;
  // many rows of a long K: in slabs whose parts fit the workspace well
  constexpr int64_t kMostBytes = int64_t{256} << 20;
  const int64_t bytes = splits > 1 ? tiles * splits * values * 4 : 0, by_bytes = ceil_div(bytes, kMostBytes), by_grid = ceil_div(down, 65535);
  const int64_t slabs = by_bytes > by_grid ? by_bytes : by_grid;
  if (slabs > 1 && down > 1) {
    const int64_t step = (down / slabs > 1 ? down / slabs : 1) * rows;
    for (int64_t m = 0; m < a.M; m += step) {
      Q4Args part = a;
      Q4Epilogue at = ep;
      part.M = a.M - m < step ? a.M - m : step;
      part.x = a.x + m * a.K;
      part.y = static_cast<char*>(a.y) + m * a.N * (ep.kind == DTAS_EPI_BIAS_ADD2_CAST_F32 ? 4 : 2);
      if (ep.res1) at.res1 = ep.res1 + m * a.N, at.res2 = ep.res2 + m * a.N;
      if (launch_q4(kernel, part, at, cols, rows, threads, values, fill, least, lds_per_chunk, lds_fixed, lds_most, s) != 0) return -1;
    }
    return 0;
  }
  if (across > INT32_MAX || splits > 65535) return fail("gemv_q4: the launch has too many workgroups");
  a.splits = static_cast<int>(splits);
  std::unique_lock<std::recursive_mutex> lock;
  if (splits > 1 && split_scratch(s, static_cast<size_t>(tiles * splits) * values * sizeof(float), static_cast<size_t>(tiles), a.splits, &a.ws, &a.arrivals, &lock) != 0) return -1;
  const unsigned lds = static_cast<unsigned>(ceil_div(chunks, splits) * lds_per_chunk + lds_fixed);
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(across), static_cast<unsigned>(splits), static_cast<unsigned>(down)), dim3(threads), lds, s, a, ep);
  return check_launch("gemv_q4");
}
template <int GS, int W, int D>
int launch_q4_few(const Q4Args& a, const Q4Epilogue& ep, hipStream_t s) {
  return launch_q4(gemv_q4_kernel<GS, W, D>, a, ep, 16, 4, 64 * W, 64, kNumCU, 2 * W, a.M * kChunk * 2 + 16 * (8 / GS), 16 * 16, 60 * 1024, s);
}
template <int MT, int GS, int CT, int KG, int SL>
int launch_q4_many(const Q4Args& a, const Q4Epilogue& ep, hipStream_t s, int least = KG * SL) {
  constexpr int kRows = 16 * MT, kCols = 16 * CT;
  return launch_q4(gemv_q4_rows_kernel<MT, GS, CT, KG, SL>, a, ep, kCols, kRows, 64 * CT * KG, kRows * kCols, kNumCU, least, kCols * (8 / GS), kCols * 16, 20 * 1024, s);
}
template <int GS>
int launch_q4_rows(const Q4Args& a, const Q4Epilogue& ep, hipStream_t s) {
  // few columns: more wavefronts to each sixteen.  2560 x 10240 (160 workgroups) on 4 / 8 / 16 wavefronts 14.9 / 10.4 / 7.9 us, 7680 x 2560 (480) 7.2 / 6.2 / 6.3,
  // 50280 x 4096 (3143) 27.0 (28.8 when the others were measured) / 31.5 / 40.5; four chunks requested at once instead of two are level to 10 % longer
  if (a.M <= 4) return a.N <= 16 * 256 ? launch_q4_few<GS, 16, 2>(a, ep, s) : a.N <= 16 * 1024 ? launch_q4_few<GS, 8, 2>(a, ep, s) : launch_q4_few<GS, 4, 2>(a, ep, s);
  // Where blocks of 32 columns fill one round of the CUs at most, and K is not long: those, with all of K, instead of 64 columns and parts of K that are handed
  // over.  16 x 2560 x 2560 9.0 -> 6.4 us, 16 x 7680 x 2560 9.9 -> 7.1, 64 x 4096 x 4096 12.4 -> 10.5, 64 x 4096 x 6144 14.9 -> 13.6; 16 x 2560 x 10240 would
  // take 12.6 instead of 10.9, 64 x 10240 x 2560 (two rounds) 21.6 instead of 16.6.
  const int rows = a.M <= 16 ? 16 : 32;
  if (ceil_div(a.N, 32) * ceil_div(a.M, rows) <= kNumCU && a.K <= 6144) {
    constexpr int kWhole = 64;  // chunks: more than there are
    return a.M <= 16 ? launch_q4_many<1, GS, 2, 8, 1>(a, ep, s, kWhole) : launch_q4_many<2, GS, 2, 8, 1>(a, ep, s, kWhole);
  }
  if (a.M <= 16) return launch_q4_many<1, GS, 4, 4, 2>(a, ep, s);
  // by 32 rows, W again for the next 32: 64 rows at once are behind but for the widest W (64 x 2560 x 10240 25.4 us against 18.3,
  // 64 x 10240 x 2560 23.0 / 17.8, 48 x 11008 x 4096 20.9 / 22.9).  Sixteen wavefronts where the columns are few, eight beyond (10240 x 2560 20.5 / 17.8, 2560 x 10240 18.3 / 20.3)
  return a.N <= 8192 ? launch_q4_many<2, GS, 4, 4, 1>(a, ep, s) : launch_q4_many<2, GS, 4, 2, 2>(a, ep, s);
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
  if (K > 0 && aligned(x, 16) && aligned(Wq, 16)) {
    const Q4Args a{xp, static_cast<const unsigned char*>(Wq), sp, y, M, N, K, 1, nullptr, nullptr};
    return group == 32 ? launch_q4_rows<1>(a, ep, s) : group == 64 ? launch_q4_rows<2>(a, ep, s) : launch_q4_rows<4>(a, ep, s);
  }
  const int64_t grid = ceil_div(M * N, 4) < (int64_t{1} << 20) ? ceil_div(M * N, 4) : int64_t{1} << 20;
  hipLaunchKernelGGL(gemv_q4_scalar_kernel, dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, xp, static_cast<const unsigned char*>(Wq), sp, ep,
                     y, N, K, group_shift, M * N);
  return check_launch("gemv_q4");
}
