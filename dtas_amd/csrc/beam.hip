// Beam search's selection over beams and vocabulary, for gfx950.
//
//   candidate (w, v) of a group: scores[w] + logits[w][v] - log sum_u exp(logits[w][u]); of a beam that is done: (w, eos) with scores[w]
//   the `beams` best, by (score descending, w, v ascending); what is no finite number counts as -inf
//
// Within a beam the order is that of the logits, so one pass over them is enough: a workgroup goes through a part of one beam's logits and keeps its maximum, its sum of
// exponentials (sixteen terms added in 32 bits, their sums in 64) and its W best so far; whoever is last among a group's workgroups has the
// sums of all and compares what is left, in 64 bits.
// The W best of many are found without sorting them: every eight lanes have the best of their own, the W-th best of these is as good as W of all at least, so only what is not
// below that can be among the W.  These few are counted out against each other; behind the first piece of a part only what beats the W-th best so far is left.
// Measured (vocabulary 50280): one group of 4 beams 11.6 us, 32 groups of 8 23.4 us (51 MB: 2.2 TB/s; 10 us at a copy's rate), one group of 32 20.5 us.  What binds is the chain of one
// workgroup: its load's trip, bound, counting, the hand-over and the last one's comparison (5 to 8 us), each behind the one before.  One search after the other, W of them, took 36.7 and
// 181 us; the W-th best lanes of each wavefront as the bound 14.4, 30.8 and 39.2.  (Candidates behind the first piece counted out behind the last alone: 24.6 for 32 groups, but 12.9 for one.)
#include "gemm_common.h"

namespace dtas {
namespace {

struct BeamArgs {
  const float *logits, *scores;
  const int* done;
  int *tokens, *parents;
  float* new_scores;
  int* new_done;
  int beams, parts, per;  // logits per part, a multiple of 4
  int64_t V, eos;
  uint64_t* room;      // [groups][beams][parts][2 + beams]: maximum and number of candidates, sum, candidates (logit, token)
  unsigned* arrivals;  // [groups]
};
template <typename T>
__device__ __forceinline__ void put(T* at, T v) { __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename T>
__device__ __forceinline__ T get(const T* at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint64_t pair_of(float x, unsigned y) { return static_cast<uint64_t>(__builtin_bit_cast(unsigned, x)) | static_cast<uint64_t>(y) << 32; }
__device__ __forceinline__ float first_of(uint64_t v) { return __builtin_bit_cast(float, static_cast<unsigned>(v)); }
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

typedef double f64x4 __attribute__((ext_vector_type(4)));

constexpr int kBeamThreads = 512, kBeamWaves = kBeamThreads / 64;

// Terms exp(x - m), x <= m, as 2^(x k - c) with k = log2 e in fp32 and c = m k rounded: in one operation x k - c = (x - m) k + (m k - c), whose last part is the same for all of
// them, exact in fp32, and small while m is (below 2^20: 0.1).  Its own rounding and k's leave y 2^-24 and 0.23 y 2^-24 of a term, y = m - x.
constexpr float kLog2e = 1.44269502f;
// For m beyond: the exponent as the rounded product with log2 e and what that rounding left; nought for -inf and for what is no number
__device__ __forceinline__ float exp_below(float x, float m) {
  constexpr float kLow = 1.92596299e-8f, kLn2 = 0.693147182f;
  const float d = fmaxf(x - m, -150.f), t = d * kLog2e;
  const float e = __builtin_amdgcn_exp2f(t), r = fmaf(d, kLow, fmaf(d, kLog2e, -t));
  return fmaf(e, r * kLn2, e);
}
// the next number below (-inf: itself)
__device__ __forceinline__ float below_of(float v) {
  const int bits = __builtin_bit_cast(int, v);
  return v == -INFINITY ? v : v == 0.f ? -__builtin_bit_cast(float, 1) : __builtin_bit_cast(float, v > 0.f ? bits - 1 : bits + 1);
}

// sums over the lanes whose numbers agree but for the bits below `width` (a power of two up to 64)
__device__ __forceinline__ double sum_over(double v, int width) {
  for (int k = 1; k < width; k *= 2) v += __shfl_xor(v, k);
  return v;
}
__device__ __forceinline__ float max_over(float v, int width) {
  for (int k = 1; k < width; k *= 2) v = fmaxf(v, __shfl_xor(v, k));
  return v;
}
// Numbers as whole ones in the same order, and back (what is not above -inf: -inf)
__device__ __forceinline__ unsigned key_bits(float v) {
  const unsigned bits = __builtin_bit_cast(unsigned, v);
  return bits >> 31 != 0 ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float of_key_bits(unsigned key) {
  return key <= 0x007fffffu ? -INFINITY : __builtin_bit_cast(float, key >> 31 != 0 ? key & 0x7fffffffu : ~key);
}
constexpr int kLastBit = 12;  // of a bound: 20 bits are near enough
// The W-th largest of the lanes' values, or a little less: its first bits, found one by one
__device__ __forceinline__ float nth_in_wave(float v, int W) {
  const unsigned key = key_bits(v);
  unsigned found = 0;
#pragma unroll 4
  for (int i = 31; i >= kLastBit; --i) {
    const unsigned next = found | 1u << i;
    found = __builtin_popcountll(__builtin_amdgcn_ballot_w64(key >= next)) >= W ? next : found;
  }
  return of_key_bits(found);
}
// the sum of all lanes, in the last
template <int CTRL, int ROWS>
__device__ __forceinline__ double add_dpp(double v) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const unsigned low = static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(bits), CTRL, ROWS, 0xf, true));
  const unsigned high = static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(bits >> 32), CTRL, ROWS, 0xf, true));
  return v + __builtin_bit_cast(double, static_cast<uint64_t>(low) | static_cast<uint64_t>(high) << 32);
}
__device__ __forceinline__ double sum_in_last(double v) {
  v = add_dpp<0x118, 0xf>(add_dpp<0x114, 0xf>(add_dpp<0x112, 0xf>(add_dpp<0x111, 0xf>(v))));  // row_shr:1, 2, 4, 8
  return add_dpp<0x143, 0xc>(add_dpp<0x142, 0xa>(v));                                         // row_bcast:15, :31
}
template <int CTRL>
__device__ __forceinline__ float max_dpp(float v) {
  const int bits = __builtin_bit_cast(int, v);
  return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(bits, bits, CTRL, 0xf, 0xf, true)));
}
__device__ __forceinline__ float max_of_eight(float v) { return max_dpp<0x141>(max_dpp<0x4E>(max_dpp<0xB1>(v))); }  // quad_perm xor 1, xor 2, row_half_mirror

// A candidate's place in the order: score, then the beam, then the logit, then the token (of one beam's candidates the sum may be the same where the logits are not)
struct Key {
  double score;
  float logit;
  int beam, token;
};
__device__ __forceinline__ bool before(const Key& a, const Key& b) {
  if (a.score != b.score) return a.score > b.score;
  if (a.beam != b.beam) return a.beam < b.beam;
  if (a.logit != b.logit) return a.logit > b.logit;
  return a.token < b.token;
}
__device__ __forceinline__ Key other(const Key& k, int lane_mask) {
  return Key{__shfl_xor(k.score, lane_mask), __shfl_xor(k.logit, lane_mask), __shfl_xor(k.beam, lane_mask), __shfl_xor(k.token, lane_mask)};
}
__device__ __forceinline__ Key no_key() { return Key{-INFINITY, -INFINITY, INT32_MAX, INT32_MAX}; }
__device__ Key first_in_block(Key k, Key* slots) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    const Key o = other(k, m);
    if (before(o, k)) k = o;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = k;
  __syncthreads();
  k = slots[0];
  for (int w = 1; w < kBeamWaves; ++w)
    if (before(slots[w], k)) k = slots[w];
  return k;
}

constexpr int kManyKeys = 96;  // candidates from which on a sharper bound is looked for (2 groups of 32 beams over 92931 tokens, scores up to 20 apart: 27.4 us, 144 without)
constexpr int kFew = 1024, kFewKeys = 512;  // candidates that are counted out; more (many equal ones, hardly any numbers) are taken one after the other
constexpr int kPieces = 4, kPiece = kBeamThreads * 4 * kPieces;  // 16 logits per thread at a time

__global__ void __launch_bounds__(kBeamThreads) beam_select_kernel(BeamArgs a) {
  union Lds {
    struct { __attribute__((aligned(16))) float logit[kFew]; int at[kFew]; } piece;
    struct { __attribute__((aligned(32))) double score[kFewKeys]; float logit[kFewKeys]; int beam[kFewKeys], token[kFewKeys]; } all;
  };
  __shared__ Lds few;
  __shared__ Key slots[kBeamWaves];
  __shared__ float tops[kBeamWaves], bounds[64];
  __shared__ __attribute__((aligned(16))) float best_logit[2][DTAS_MAX_BEAMS];
  __shared__ int best_at[2][DTAS_MAX_BEAMS];
  __shared__ double sums[kBeamWaves], log_sum[DTAS_MAX_BEAMS], stat_s[kBeamThreads];
  __shared__ float top_of[DTAS_MAX_BEAMS], chosen_score[DTAS_MAX_BEAMS], stat_m[kBeamThreads];
  __shared__ int chosen_beam[DTAS_MAX_BEAMS], chosen_token[DTAS_MAX_BEAMS];
  __shared__ int above[2][kBeamWaves], flag, counts[2];  // (of one piece and of the next: a wavefront may be that far ahead of another)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = blockIdx.x, w = blockIdx.y, W = a.beams;
  const int64_t g = blockIdx.z, from = static_cast<int64_t>(part) * a.per;
  const int here = static_cast<int>(a.V - from < a.per ? a.V - from : a.per), stride = 2 + W;
  const bool plain = finite(a.scores[g * W + w]) && !(a.done && a.done[g * W + w] != 0);
  auto most = [&](const float* of) {
    float v = of[0];
#pragma unroll
    for (int i = 1; i < kBeamWaves; ++i) v = fmaxf(v, of[i]);
    return v;
  };
  // the W-th best of 64 maxima of eight threads each: as many are as good as it
  static_assert(kBeamThreads == 64 * 8 && DTAS_MAX_BEAMS <= 64, "a lane for each");
  auto bound_of = [&](float own) {
    const float eight = max_of_eight(own);
    if ((lane & 7) == 0) bounds[tid >> 3] = eight;
    __syncthreads();
    return nth_in_wave(bounds[lane], W);
  };
  if (plain) {
    const float* row = a.logits + (g * W + w) * a.V + from;
    float x[kPieces][4], y[kPieces][4];
    auto load = [&](float (&to)[kPieces][4], int base) {
#pragma unroll
      for (int u = 0; u < kPieces; ++u) {
        const int i = base + u * kBeamThreads * 4 + tid * 4;
        if (i + 4 <= here) {
          f32x4 v;  // (rows of an odd vocabulary begin off 16 bytes)
          __builtin_memcpy(&v, __builtin_assume_aligned(row + i, 4), 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) to[u][j] = v[j];
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) to[u][j] = i + j < here ? row[i + j] : -INFINITY;
        }
      }
    };
    load(x, 0);
    if (tid < 2) counts[tid] = 0;
    int have = 0, side = 0;  // (of the best so far, in best_logit[side])
    float limit = -INFINITY, m = -INFINITY;
    double s = 0.0;
    for (int base = 0, turn = 0; base < here; base += kPiece, turn ^= 1) {
      if (base + kPiece < here) load(y, base + kPiece);
      float own = -INFINITY;
#pragma unroll
      for (int u = 0; u < kPieces; ++u) own = fmaxf(own, fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3])));
      if (have < W) {
        limit = bound_of(own);
      }
      const float wave_top = wave_max(own);
      if (wave_top > m) {
        s = m == -INFINITY ? s : s * exp(static_cast<double>(m) - static_cast<double>(wave_top));  // (before the first number: nought, or NaN where one was among them, which stays)
        m = wave_top;
      }
      float terms[kPieces];
      const float at = m == -INFINITY ? 0.f : m, c = at * kLog2e;
      if (__builtin_amdgcn_readfirstlane(fabsf(at) < 0x1p20f)) {  // (of what is no number the sum is none)
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
          float e[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) e[j] = __builtin_amdgcn_exp2f(fmaf(x[u][j], kLog2e, -c));
          terms[u] = (e[0] + e[1]) + (e[2] + e[3]);
        }
        s += static_cast<double>((terms[0] + terms[1]) + (terms[2] + terms[3])) * __builtin_amdgcn_exp2f(-fmaf(at, kLog2e, -c));
      } else {
        bool strange = false;
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
          terms[u] = (exp_below(x[u][0], m) + exp_below(x[u][1], m)) + (exp_below(x[u][2], m) + exp_below(x[u][3], m));
#pragma unroll
          for (int j = 0; j < 4; ++j) strange = strange || x[u][j] != x[u][j];
        }
        s += strange ? __builtin_nan("") : static_cast<double>((terms[0] + terms[1]) + (terms[2] + terms[3]));
      }
      // (an equal one behind the best so far is no better)
      const float above = have == W ? limit : below_of(limit);
      if (own > above) {
#pragma unroll
        for (int u = 0; u < kPieces; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (x[u][j] > above) {
              const int n = atomicAdd(&counts[turn], 1);
              if (n < kFew) {
                few.piece.logit[n] = x[u][j];
                few.piece.at[n] = base + u * kBeamThreads * 4 + tid * 4 + j;
              }
            }
      }
      __syncthreads();
      const int n = counts[turn];
      if (n > 0) {
        const int old = have;
        const float* old_logit = best_logit[side];
        const int* old_at = best_at[side];
        side ^= 1;
        if (n <= kFew) {
          have = old + n < W ? old + n : W;
          for (int i = tid; i < n + old; i += kBeamThreads) {
            const float mine = i < n ? few.piece.logit[i] : old_logit[i - n];
            const int at = i < n ? few.piece.at[i] : old_at[i - n];
            int rank = 0, level = 0;
            auto count = [&](const float* of, int many) {
              for (int k = 0; k < many; k += 4) {
                const f32x4 some = *reinterpret_cast<const f32x4*>(of + k);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const bool in = k + j < many;
                  rank += in && some[j] > mine ? 1 : 0;
                  level += in && some[j] == mine ? 1 : 0;
                }
              }
            };
            count(few.piece.logit, n);
            count(old_logit, old);
            if (level > 1) {  // (equal ones, but for itself, go by their places)
              for (int k = 0; k < n; ++k) rank += few.piece.logit[k] == mine && few.piece.at[k] < at ? 1 : 0;
              for (int k = 0; k < old; ++k) rank += old_logit[k] == mine && old_at[k] < at ? 1 : 0;
            }
            if (rank < W) {
              best_logit[side][rank] = mine;
              best_at[side][rank] = at;
            }
          }
        } else {
          float last = INFINITY;
          int last_at = -1;
          for (have = 0; have < W; ++have) {
            Key best = no_key();
            auto offer = [&](float logit, int at) {
              const Key k{0.0, logit, 0, at};
              if (finite(logit) && (logit < last || (logit == last && at > last_at)) && before(k, best)) best = k;
            };
#pragma unroll
            for (int u = 0; u < kPieces; ++u)
#pragma unroll
              for (int j = 0; j < 4; ++j) offer(x[u][j], base + u * kBeamThreads * 4 + tid * 4 + j);
            if (tid < old) offer(old_logit[tid], old_at[tid]);
            best = first_in_block(best, slots);
            if (best.token == INT32_MAX) break;
            last = best.logit;
            last_at = best.token;
            if (tid == 0) {
              best_logit[side][have] = last;
              best_at[side][have] = last_at;
            }
          }
        }
        __syncthreads();
        if (tid == 0) counts[turn] = 0;  // (a barrier stands before it is used again, and before the list is)
        if (have == W) limit = best_logit[side][W - 1];
      }
#pragma unroll
      for (int u = 0; u < kPieces; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[u][j] = y[u][j];
    }
    if (lane == 0) tops[wave] = m;
    __syncthreads();
    const float top = most(tops);
    s = sum_in_last(s);
    if (m != -INFINITY) s *= exp(static_cast<double>(m) - static_cast<double>(top));
    if (lane == 63) sums[wave] = s;
    __syncthreads();
    uint64_t* room = a.room + ((g * W + w) * a.parts + part) * stride;
    if (tid < have) put(room + 2 + tid, pair_of(best_logit[side][tid], static_cast<unsigned>(from + best_at[side][tid])));
    if (tid == 0) {
      double all = sums[0];
      for (int i = 1; i < kBeamWaves; ++i) all += sums[i];
      put(room, pair_of(top, static_cast<unsigned>(have)));
      put(room + 1, __builtin_bit_cast(uint64_t, all));
    }
  }
  // ---- whoever is last among the group's workgroups.  What they left passes the L2 (the XCDs' are not coherent); an arrival is counted once its own has drained
  const int lists = W * a.parts;
  if (lists > 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
      const unsigned arrived = __hip_atomic_fetch_add(a.arrivals + g, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      flag = arrived == static_cast<unsigned>(lists) - 1;
      if (flag) put(a.arrivals + g, 0u);  // re-armed for the next launch
    }
  } else if (tid == 0) {
    flag = 1;
  }
  if (tid == 0) counts[0] = 0;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (!flag) return;
  const uint64_t* room = a.room + g * W * a.parts * stride;
  const float* scores = a.scores + g * W;
  const int* done = a.done ? a.done + g * W : nullptr;
  auto is_done = [&](int i) { return done && done[i] != 0; };
  auto goes_on = [&](int i) { return finite(scores[i]) && is_done(i) && a.eos >= 0 && a.eos < a.V; };
  // A list is a part of a beam, a thread's (there are no more than threads: beam_parts).  Of fewer than a wavefront has lanes, though, the W-th best of their first candidates would be no bound: `depth` threads go through a list
  // there, thread (list, sub) through its candidates sub, sub + depth, ..., so that a wavefront's are the first ones of all (18 groups of 32 beams over 9143 tokens 54 us, 269 without).
  // What the parts left, and a thread's first candidates, in one trip to memory (further ones, if there are more, are read when they are needed).
  constexpr int kAhead = 4;
  struct List {
    uint64_t head, sum, one[kAhead];
  };
  const int wanted = lists >= 64 ? (W + kAhead - 1) / kAhead : W, depth = kBeamThreads / lists < wanted ? kBeamThreads / lists : wanted;
  const int sub_of = depth == 1 ? 0 : tid / lists, list_of = tid - sub_of * lists, beam_of = list_of / a.parts;
  const bool listed = list_of < lists && sub_of < depth, sole = listed && sub_of == 0;
  const uint64_t* from_list = room + static_cast<int64_t>(listed ? list_of : 0) * stride;
  List mine{};
  if (listed && finite(scores[beam_of]) && !is_done(beam_of)) {
    mine.head = get(from_list);
    mine.sum = get(from_list + 1);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) mine.one[u] = get(from_list + 2 + (sub_of + u * depth < W ? sub_of + u * depth : W - 1));
  }
  if (sole) {
    stat_m[tid] = first_of(mine.head);
    stat_s[tid] = __builtin_bit_cast(double, mine.sum);
  }
  __syncthreads();
  // the beams' sums, several beams to a wavefront where there are few parts
  int width = 1;
  while (width < a.parts && width < 64) width *= 2;
  const int each = 64 / width, sub = lane / width, first = lane - sub * width;
  for (int i0 = wave * each; i0 < W; i0 += kBeamWaves * each) {
    const int i = i0 + sub;
    const bool plain_row = i < W && finite(scores[i]) && !is_done(i);
    float m = -INFINITY;
    double s = 0.0;
    for (int p = first; plain_row && p < a.parts; p += 64) {  // (one lane's parts: one sum on the larger maximum)
      const int t = i * a.parts + p;
      const float o = stat_m[t], both = fmaxf(m, o);
      const double more = stat_s[t];
      s = (m == -INFINITY ? s : s * exp(static_cast<double>(m) - static_cast<double>(both))) + (o == -INFINITY ? more : more * exp(static_cast<double>(o) - static_cast<double>(both)));
      m = both;
    }
    const float top = max_over(m, width);
    const double sum = sum_over(m == -INFINITY ? s : s * exp(static_cast<double>(m) - static_cast<double>(top)), width);  // (a part of -inf has a sum of nought)
    if (plain_row && first == 0) {
      top_of[i] = top;
      log_sum[i] = log(sum);
    }
  }
  __syncthreads();
  auto normal = [&](int i) { return finite(scores[i]) && !is_done(i) && finite(top_of[i]) && fabs(log_sum[i]) < INFINITY; };
  auto key_of = [&](int i, uint64_t one) {
    const float x = first_of(one);
    return Key{static_cast<double>(scores[i]) + ((static_cast<double>(x) - static_cast<double>(top_of[i])) - log_sum[i]), x, i, static_cast<int>(one >> 32)};
  };
  auto ended_key = [&](int i) { return Key{static_cast<double>(scores[i]), 0.f, i, static_cast<int>(a.eos)}; };
  const int size = static_cast<int>(mine.head >> 32);
  const bool goes = listed && normal(beam_of), ended = sole && !goes && list_of == beam_of * a.parts && goes_on(beam_of);
  // the bound that the threads' first candidates give, rounded to 32 bits like what is held against it (a beam that is done has one candidate, in its first part's place)
  float own = -INFINITY;
  if (goes && size > sub_of) own = static_cast<float>(key_of(beam_of, mine.one[0]).score);
  if (ended) own = static_cast<float>(ended_key(beam_of).score);
  float least;
  if (lists >= 8 * W) {  // (fewer: there are no W maxima of eight threads)
    least = bound_of(own);
  } else {
    const float bound = nth_in_wave(own, W);
    if (lane == 0) bounds[wave] = bound;
    __syncthreads();
    least = most(bounds);
  }
  auto keep = [&](const Key& k) {
    const int n = atomicAdd(&counts[0], 1);
    if (n >= kFewKeys) return;
    few.all.score[n] = k.score;
    few.all.logit[n] = k.logit;
    few.all.beam[n] = k.beam;
    few.all.token[n] = k.token;
  };
  auto collect = [&] {
    bool more = goes;
    for (int k0 = sub_of; more && k0 < size; k0 += kAhead * depth) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const uint64_t one = k0 == sub_of ? mine.one[u] : get(from_list + 2 + (k0 + u * depth < size ? k0 + u * depth : size - 1));
        const Key k = key_of(beam_of, one);
        more = more && k0 + u * depth < size && static_cast<float>(k.score) >= least;
        if (more) keep(k);
      }
    }
    if (ended) keep(ended_key(beam_of));
    __syncthreads();
    return counts[0];
  };
  int n = collect();
  if (n > kManyKeys) {
    // some beams lead the others by far, and the bound is what these have: the W-th best of all that the threads hold, bit by bit
    unsigned keys[kAhead], best = 0;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) keys[u] = goes && sub_of + u * depth < size ? key_bits(static_cast<float>(key_of(beam_of, mine.one[u]).score)) : 0u;
    if (ended) keys[0] = key_bits(static_cast<float>(ended_key(beam_of).score));
    for (int i = 31; i >= kLastBit; --i) {
      const unsigned next = best | 1u << i;
      int some = 0;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) some += __builtin_popcountll(__builtin_amdgcn_ballot_w64(keys[u] >= next));
      if (lane == 0) above[i & 1][wave] = some;
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int k = 0; k < kBeamWaves; ++k) all += above[i & 1][k];
      best = all >= W ? next : best;
    }
    least = fmaxf(least, of_key_bits(best));
    if (tid == 0) counts[0] = 0;
    __syncthreads();
    n = collect();
  }
  int found = n < W ? n : W;
  if (n <= kFewKeys) {
    for (int i = tid; i < n; i += kBeamThreads) {
      const Key key{few.all.score[i], few.all.logit[i], few.all.beam[i], few.all.token[i]};
      int rank = 0, level = 0;
      for (int k = 0; k < n; k += 4) {
        const f64x4 some = *reinterpret_cast<const f64x4*>(few.all.score + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool in = k + j < n;
          rank += in && some[j] > key.score ? 1 : 0;
          level += in && some[j] == key.score ? 1 : 0;
        }
      }
      if (level > 1)
        for (int k = 0; k < n; ++k)
          if (few.all.score[k] == key.score) rank += before(Key{key.score, few.all.logit[k], few.all.beam[k], few.all.token[k]}, key) ? 1 : 0;
      if (rank < W) {
        chosen_beam[rank] = key.beam;
        chosen_token[rank] = key.token;
        chosen_score[rank] = static_cast<float>(key.score);
      }
    }
  } else {
    Key last = no_key();
    for (found = 0; found < W; ++found) {
      Key best = no_key();
      auto offer = [&](const Key& k) {
        if ((found == 0 || before(last, k)) && before(k, best)) best = k;
      };
      for (int k = 0; sole && goes && k < size; ++k) offer(key_of(beam_of, get(from_list + 2 + k)));
      if (ended) offer(ended_key(beam_of));
      best = first_in_block(best, slots);
      if (best.token == INT32_MAX) break;
      last = best;
      if (tid == 0) {
        chosen_beam[found] = best.beam;
        chosen_token[found] = best.token;
        chosen_score[found] = static_cast<float>(best.score);
      }
    }
  }
  __syncthreads();
  if (found < W && tid == 0) {  // fewer candidates with a number than beams: the first of the others
    for (int i = 0, v = 0, k = found; k < W; ++v) {
      if (v == a.V) ++i, v = 0;
      bool taken = false;
      for (int c = 0; c < found; ++c) taken = taken || (chosen_beam[c] == i && chosen_token[c] == v);
      if (taken) continue;
      chosen_beam[k] = i;
      chosen_token[k] = v;
      chosen_score[k++] = -INFINITY;
    }
  }
  __syncthreads();
  const bool one_of = tid < W;
  const int parent = one_of ? chosen_beam[tid] : 0, token = one_of ? chosen_token[tid] : 0;
  const bool over = (done && done[parent] != 0) || token == a.eos;
  __syncthreads();  // (scores and done may be the outputs: they have been read)
  if (!one_of) return;
  a.parents[g * W + tid] = parent;
  a.tokens[g * W + tid] = token;
  a.new_scores[g * W + tid] = chosen_score[tid];
  if (a.new_done) a.new_done[g * W + tid] = over ? 1 : 0;
}

constexpr int64_t kBeamWords = int64_t{1} << 25, kLeastPart = 2048;  // 64-bit words of a launch's lists; logits of a part
// Parts of a row: two workgroups per CU (and so a group's never more than a workgroup has threads), of 2048 logits at least (4096: 13.6 us instead of 14.1 for one group of 4 beams, 44.0 instead of 38.6 for one of 32, even for the others).
inline int64_t beam_parts(int64_t rows, int64_t V) {
  static_assert(kBeamThreads >= 512 && kBeamThreads >= DTAS_MAX_BEAMS, "a thread for each part of a group");
  int64_t parts = rows < 512 ? 512 / rows : 1;
  if (parts > ceil_div(V, kLeastPart)) parts = ceil_div(V, kLeastPart);
  const int64_t per = ceil_div(ceil_div(V, parts), 4) * 4;
  return ceil_div(V, per);
}

int launch_beam(BeamArgs a, int64_t groups, hipStream_t s) {
  a.parts = static_cast<int>(beam_parts(groups * a.beams, a.V));
  a.per = static_cast<int>(ceil_div(ceil_div(a.V, a.parts), 4) * 4);
  const int64_t words = static_cast<int64_t>(a.beams) * a.parts * (2 + a.beams);
  // as many groups at a time as 256 MiB of the workspace, and a grid, hold
  int64_t some = kBeamWords / words;
  if (some > 65535) some = 65535;
  for (int64_t g = 0; g < groups; g += some) {
    const int64_t now = groups - g < some ? groups - g : some;
    float* room = nullptr;
    std::unique_lock<std::recursive_mutex> lock;
    if (split_scratch(s, static_cast<size_t>(now * words) * 8, static_cast<size_t>(now), a.parts, &room, &a.arrivals, &lock) != 0) return -1;
    a.room = reinterpret_cast<uint64_t*>(room);
    hipLaunchKernelGGL(beam_select_kernel, dim3(static_cast<unsigned>(a.parts), static_cast<unsigned>(a.beams), static_cast<unsigned>(now)), dim3(kBeamThreads), 0, s, a);
    if (check_launch("beam_select") != 0) return -1;
    const int64_t rows = now * a.beams;
    a.logits += rows * a.V;
    a.scores += rows;
    if (a.done) a.done += rows;
    a.tokens += rows;
    a.parents += rows;
    a.new_scores += rows;
    if (a.new_done) a.new_done += rows;
  }
  return 0;
}

}  // namespace
}  // namespace dtas

extern "C" int dtas_beam_select_f32(const void* logits, const void* scores, const void* done, void* tokens, void* parents, void* new_scores, void* new_done,
                                    int64_t groups, int64_t beams, int64_t V, int64_t eos, void* stream) {
  using namespace dtas;
  clear_error();
  if (groups < 0 || beams < 0 || V < 0) return fail("beam_select: negative extent groups=%lld beams=%lld V=%lld", (long long)groups, (long long)beams, (long long)V);
  if (beams > DTAS_MAX_BEAMS) return fail("beam_select: up to %d beams, got %lld", DTAS_MAX_BEAMS, (long long)beams);
  if ((done == nullptr) != (new_done == nullptr)) return fail("beam_select: done and new_done go together");
  if (groups == 0 || beams == 0) return 0;
  if (V == 0) return fail("beam_select: no token to choose from");
  if (V > (int64_t{1} << 30) || groups > INT32_MAX || V > (int64_t{1} << 60) / beams / groups) return fail("beam_select: the extents overflow");
  if (!logits || !scores || !tokens || !parents || !new_scores) return fail("beam_select: NULL buffer");
  const int64_t rows = groups * beams;
  struct Span { const void* at; int64_t bytes; };
  const Span in[] = {{logits, rows * V * 4}, {scores, rows * 4}, {done, done ? rows * 4 : 0}}, out[] = {{tokens, rows * 4}, {parents, rows * 4}, {new_scores, rows * 4}, {new_done, new_done ? rows * 4 : 0}};
  const void* const same[] = {nullptr, nullptr, scores, done};
  for (int i = 0; i < 4; ++i) {
    if (!out[i].at) continue;
    for (const Span& o : in)
      if (o.at && !(o.at == same[i] && out[i].at == o.at) && overlaps(out[i].at, out[i].bytes, o.at, o.bytes)) return fail("beam_select: output overlaps an input");
    for (int j = 0; j < i; ++j)
      if (out[j].at && overlaps(out[i].at, out[i].bytes, out[j].at, out[j].bytes)) return fail("beam_select: the outputs overlap");
  }
  BeamArgs a{static_cast<const float*>(logits), static_cast<const float*>(scores), static_cast<const int*>(done), static_cast<int*>(tokens), static_cast<int*>(parents),
             static_cast<float*>(new_scores), static_cast<int*>(new_done), static_cast<int>(beams), 0, 0, V, eos, nullptr, nullptr};
  return launch_beam(a, groups, static_cast<hipStream_t>(stream));
}
