// What the kernels have in common that attend with few query rows per key head (attn_tree.hip, attn_paged.hip): 16 keys or rows to a matrix instruction, P and O^T as
// the lanes hold them, weights in fp16 (one or two of them), parts of the keys joined through the workspace.  Internal to libdtas_gfx950.so.
#pragma once
#include "gemm_common.h"

namespace dtas {
namespace {

constexpr int v_row_bytes(int DP) { return 2 * DP + 32; }
// A kernel for DP channels serves head dimensions above `below(DP)`: a lane whose channels lie behind the head's last reads that head's last
// ones instead, and what it read of K and Q is cleared (of V it only reaches sums that are not stored).
constexpr int below(int DP) { return DP == 64 ? 0 : DP == 96 ? 64 : DP == 128 ? 96 : DP == 192 ? 128 : 192; }

// a value's maximum (sum) over the four lanes that hold the same row, l, l ^ 16, l ^ 32, l ^ 48.  The swaps exchange halves (and
// quarters) of two registers; of a value and its copy, whose origin is hidden (given one value twice the compiler takes the two results for one)
template <typename Join>
__device__ __forceinline__ float over_row(float v, Join join) {
  unsigned x = __builtin_bit_cast(unsigned, v), y = x;
  asm("" : "+v"(y));
  const auto a = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  x = y = __builtin_bit_cast(unsigned, join(__builtin_bit_cast(float, static_cast<unsigned>(a[0])), __builtin_bit_cast(float, static_cast<unsigned>(a[1]))));
  asm("" : "+v"(y));
  const auto b = __builtin_amdgcn_permlane16_swap(x, y, false, false);
  return join(__builtin_bit_cast(float, static_cast<unsigned>(b[0])), __builtin_bit_cast(float, static_cast<unsigned>(b[1])));
}
__device__ __forceinline__ float max_of_row(float v) { return over_row(v, [](float p, float q) { return fmaxf(p, q); }); }
__device__ __forceinline__ float sum_of_row(float v) { return over_row(v, [](float p, float q) { return p + q; }); }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// N (4 or 2) channel tiles of V^T: transposing reads of the block's two halves, and the wait for them, in one statement
template <int DP, int N>
__device__ __forceinline__ void read_v(unsigned at, f16x4 (&lo)[N], f16x4 (&hi)[N]) {
  constexpr int kHalf = 16 * v_row_bytes(DP);
  if constexpr (N == 4)
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n"
        "ds_read_b64_tr_b16 %1, %8 offset:32\n"
        "ds_read_b64_tr_b16 %2, %8 offset:64\n"
        "ds_read_b64_tr_b16 %3, %8 offset:96\n"
        "ds_read_b64_tr_b16 %4, %8 offset:%9\n"
        "ds_read_b64_tr_b16 %5, %8 offset:%10\n"
        "ds_read_b64_tr_b16 %6, %8 offset:%11\n"
        "ds_read_b64_tr_b16 %7, %8 offset:%12\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(lo[2]), "=&v"(lo[3]), "=&v"(hi[0]), "=&v"(hi[1]), "=&v"(hi[2]), "=&v"(hi[3])
        : "v"(at), "n"(kHalf), "n"(kHalf + 32), "n"(kHalf + 64), "n"(kHalf + 96)
        : "memory");
  else
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4\n"
        "ds_read_b64_tr_b16 %1, %4 offset:32\n"
        "ds_read_b64_tr_b16 %2, %4 offset:%5\n"
        "ds_read_b64_tr_b16 %3, %4 offset:%6\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(hi[0]), "=&v"(hi[1])
        : "v"(at), "n"(kHalf), "n"(kHalf + 32)
        : "memory");
}

// (maxima are those of the products, before the scale)
__device__ __forceinline__ float weight_of(float m, float best, float scale_log2) { return best == -INFINITY ? 0.f : exp2_fast((m - best) * scale_log2); }

// sums over the lanes up to this one
__device__ __forceinline__ int sum_upto(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, true);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, true);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(sum_upto(v), 63); }
__device__ __forceinline__ int wave_most(int v) {
  auto join = [&](int w) { v = v > w ? v : w; };
  join(__builtin_amdgcn_update_dpp(v, v, 0x111, 0xf, 0xf, false));
  join(__builtin_amdgcn_update_dpp(v, v, 0x112, 0xf, 0xf, false));
  join(__builtin_amdgcn_update_dpp(v, v, 0x114, 0xf, 0xf, false));
  join(__builtin_amdgcn_update_dpp(v, v, 0x118, 0xf, 0xf, false));
  join(__builtin_amdgcn_update_dpp(v, v, 0x142, 0xa, 0xf, false));
  join(__builtin_amdgcn_update_dpp(v, v, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(v, 63);
}

// The 8 channels of k step `ks` that a lane of `quarter` holds
template <int DP>
__device__ __forceinline__ f16x8 load_channels(const char* row, int ks, int quarter, int d) {
  const int at = ks * 32 + quarter * 8;
  if (ks * 32 + 32 <= below(DP)) return *reinterpret_cast<const f16x8*>(row + at * 2);
  const f16x8 v = *reinterpret_cast<const f16x8*>(row + (at < d ? at : d - 8) * 2);
  return at < d ? v : f16x8{};
}

// Q's 8 channels, with the scale's sign: the scale itself is positive (one, where it was nought), so that a row's largest product has its largest score
template <int DP>
__device__ __forceinline__ f16x8 load_query(const half_t* row, int ks, int quarter, int d, half_t sign) {
  return load_channels<DP>(reinterpret_cast<const char*>(row), ks, quarter, d) * sign;
}

// P in fp16: a weight is 2^kRoom at the running maximum and 2^(kRoom + kAhead) = 2^15 at most.  The type's whole steps reach down to 2^-14, which is 2^-25 of the
// maximum's weight (17.3 below it in the score): down to there a weight is off by half a step, 2^-11 of itself, below by 2^-36 of the maximum's, and what is less than
// that is lost to the product with the values (not to the sum of the weights, in fp32): 2^-20 of the largest value at most after 65536 keys.  The maximum itself moves only when a
// row's largest score leaves it behind by more than 2^kAhead: O is rescaled in few tiles instead of in most.  64 nodes after 65533 keys: 2^8 and 2^7 104 .. 107 us, 2^4 and
// 2^11 level, 2^2 and 2^13 111.
constexpr float kAhead = 4.f, kRoom = 11.f;

// A weight per key from the products of one row tile, NK key tiles: mask, running maximum and sum, O rescaled where the maximum moved.
// `shown` says which of the keys 16 kt + 4 (lane >> 4) + j the row sees (bit 16 kt + ..), all: none is hidden.
template <int NK, int DT>
__device__ __forceinline__ void weigh(f32x4 (&s)[NK], bool all, uint64_t shown, int quarter, float scale_log2, float& top, float& sum, f32x4 (&o)[DT]) {
  float best = -INFINITY;
  if (!all) {
    const uint64_t mine = shown >> (4 * quarter);
#pragma unroll
    for (int kt = 0; kt < NK; ++kt)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[kt][j] = (mine >> (16 * kt + j)) & 1 ? s[kt][j] : -INFINITY;
  }
#pragma unroll
  for (int kt = 0; kt < NK; ++kt)
#pragma unroll
    for (int j = 0; j < 4; ++j) best = fmaxf(best, s[kt][j]);
  best = fmaxf(max_of_row(best), top);
  if (__builtin_amdgcn_ballot_w64((best - top) * scale_log2 > kAhead) != 0) {
    const float keep = best == -INFINITY ? 1.f : exp2_fast((top - best) * scale_log2);
    sum *= keep;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[dt][j] *= keep;
    top = best;
  }
  // (s - top) scale as one multiply-add, s scale - top scale, which is off by the rounding of top scale, up to 2^-17 (weights that much of themselves) while that
  // is 256 at most.  Where a row is beyond, that would be more than the products' own rounding, and overflow in the end: the difference is taken first.
  const float base = top == -INFINITY ? 0.f : top;
  float from = fmaf(-base, scale_log2, kRoom);
  if (__builtin_amdgcn_ballot_w64(!(fabsf(from) <= 256.f)) != 0) {
#pragma unroll
    for (int kt = 0; kt < NK; ++kt)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[kt][j] -= base;
    from = kRoom;
  }
#pragma unroll
  for (int kt = 0; kt < NK; ++kt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[kt][j] = exp2_fast(fmaf(s[kt][j], scale_log2, from));
      sum += s[kt][j];
    }
}
__device__ __forceinline__ f16x8 weights_f16(const f32x4& a, const f32x4& b) {
  return f16x8{static_cast<half_t>(a[0]), static_cast<half_t>(a[1]), static_cast<half_t>(a[2]), static_cast<half_t>(a[3]),
               static_cast<half_t>(b[0]), static_cast<half_t>(b[1]), static_cast<half_t>(b[2]), static_cast<half_t>(b[3])};
}
// ... and what is left of them beside that, in fp16 as well: the two together have 22 bits, and steps of 2^-36 of the maximum's weight at least
__device__ __forceinline__ f16x8 weights_rest(const f32x4& a, const f32x4& b, const f16x8& p) {
  f16x8 rest;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    rest[j] = static_cast<half_t>(a[j] - static_cast<float>(p[j]));
    rest[4 + j] = static_cast<half_t>(b[j] - static_cast<float>(p[4 + j]));
  }
  return rest;
}
__device__ __forceinline__ uint64_t first_bits(int n) { return n >= 64 ? ~uint64_t{0} : (uint64_t{1} << n) - 1; }

// A value that is no number, in the 16 bytes of a piece
__device__ __forceinline__ bool no_number(const u32x4& v) {
  bool bad = false;
#pragma unroll
  for (int w = 0; w < 4; ++w) bad = bad || (v[w] & 0x7c00u) == 0x7c00u || (v[w] & 0x7c000000u) == 0x7c000000u;
  return bad;
}

__device__ __forceinline__ void store_row4(half_t* to, const f32x4& v, float inv) {
  *reinterpret_cast<f16x4*>(to) = f16x4{static_cast<half_t>(v[0] * inv), static_cast<half_t>(v[1] * inv), static_cast<half_t>(v[2] * inv), static_cast<half_t>(v[3] * inv)};
}

// ---- parts of a sequence's keys: each leaves its rows' sums, and behind them their maxima and weights, in the workspace; whoever arrives last
// joins them in their order.  The shares pass the L2 (the XCDs' are not coherent): once a part's stores have drained they are visible everywhere, and
// only then is its arrival counted.
__device__ __forceinline__ void store_stat(float* share, int rows, int DP, int r, float top, float sum) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(share + rows * DP) + r,
                     static_cast<uint64_t>(__builtin_bit_cast(unsigned, top)) | static_cast<uint64_t>(__builtin_bit_cast(unsigned, sum)) << 32, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ bool last_to_arrive(unsigned* counter, int parts, int* flag) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = before == static_cast<unsigned>(parts) - 1;
    if (*flag) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // re-armed for the next launch
  }
  __syncthreads();
  return *flag != 0;
}

}  // namespace
}  // namespace dtas
