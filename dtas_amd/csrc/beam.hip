// Beam search's selection over beams and vocabulary, for gfx950.
//
//   candidate (w, v) of a group: scores[w] + logits[w][v] - log sum_u exp(logits[w][u]); of a beam that is done: (w, eos) with scores[w]
//   the `beams` best, by (score descending, w, v ascending); what is no finite number counts as -inf
//
// Within a beam the order is that of the logits, so one pass over them is enough: a workgroup has a piece of one beam's logits in registers, and leaves
// its maximum, its sum of exponentials (terms in 32 bits, each product with log2 e kept to twice that; the sum in 64) and its best candidates in their order; whoever is
// last among a group's workgroups has the sums of all and compares what is left, in 64 bits.
// Both times the best W of many are found without sorting them: every lane has the best of its own, the W-th best of these in a wavefront is as good as W of all at least, so only
// what is not below that (the best of the wavefronts') can be among the W; these few are counted out against each other.
#include "gemm_common.h"

namespace dtas {
namespace {

struct BeamArgs {
  const float *logits, *scores;
  const int* done;
  int *tokens, *parents;
  float* new_scores;
  int* new_done;
  int beams, parts;
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

constexpr int kBeamThreads = 256, kBeamWaves = kBeamThreads / 64;

// exp(x - m) for x <= m: the exponent as the rounded product with log2 e and what that rounding left
__device__ __forceinline__ float exp_below(float x, float m) {
  constexpr float kHigh = 1.44269502f, kLow = 1.92596299e-8f, kLn2 = 0.693147182f;
  const float d = x - m, t = d * kHigh;
  if (!(t > -200.f)) return x == x ? 0.f : x;  // (that is nothing next to the maximum's 1; what is no number stays none)
  const float e = __builtin_amdgcn_exp2f(t), r = fmaf(d, kHigh, -t) + d * kLow;
  return fmaf(e, r * kLn2, e);
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
// The W-th largest of the lanes' values
__device__ __forceinline__ float nth_in_wave(float v, int W, int lane) {
  int above = 0;
#pragma unroll 16
  for (int i = 0; i < 64; ++i) {
    const float o = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i));
    above += o > v || (o == v && i < lane) ? 1 : 0;
  }
  const uint64_t at = __builtin_amdgcn_ballot_w64(above == W - 1);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), at ? __builtin_ctzll(at) : 0));
}
__device__ __forceinline__ double nth_in_wave(double v, int W, int lane) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const int low = static_cast<int>(bits), high = static_cast<int>(bits >> 32);
  auto lane_of = [&](int i) {
    const unsigned l = __builtin_amdgcn_readlane(low, i), h = __builtin_amdgcn_readlane(high, i);
    return __builtin_bit_cast(double, static_cast<uint64_t>(h) << 32 | l);
  };
  int above = 0;
#pragma unroll 8
  for (int i = 0; i < 64; ++i) {
    const double o = lane_of(i);
    above += o > v || (o == v && i < lane) ? 1 : 0;
  }
  const uint64_t at = __builtin_amdgcn_ballot_w64(above == W - 1);
  return lane_of(at ? __builtin_ctzll(at) : 0);
}

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

constexpr int kFew = 1024, kFewKeys = 512;  // candidates that are counted out; more (many equal ones, hardly any numbers) are taken one after the other

template <int U>  // 16-byte pieces per thread
__global__ void __launch_bounds__(kBeamThreads) beam_select_kernel(BeamArgs a) {
  union Lds {
    struct { float logit[kFew]; int at[kFew]; } piece;
    struct { double score[kFewKeys]; float logit[kFewKeys]; int beam[kFewKeys], token[kFewKeys]; } all;
  };
  __shared__ Lds few;
  __shared__ Key slots[kBeamWaves];
  __shared__ float tops[kBeamWaves], bounds[kBeamWaves];
  __shared__ double sums[kBeamWaves], key_bounds[kBeamWaves];
  __shared__ double log_sum[DTAS_MAX_BEAMS];
  __shared__ float top_of[DTAS_MAX_BEAMS], chosen_score[DTAS_MAX_BEAMS];
  __shared__ int chosen_beam[DTAS_MAX_BEAMS], chosen_token[DTAS_MAX_BEAMS];
  __shared__ int flag, count;
  constexpr int kPiece = kBeamThreads * 4 * U;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = blockIdx.x, w = blockIdx.y, W = a.beams;
  const int64_t g = blockIdx.z, from = static_cast<int64_t>(part) * kPiece;
  const int here = static_cast<int>(a.V - from < kPiece ? a.V - from : kPiece), stride = 2 + W;
  const bool plain = finite(a.scores[g * W + w]) && !(a.done && a.done[g * W + w] != 0);
  if (plain) {
    const float* row = a.logits + (g * W + w) * a.V + from;
    float x[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = u * kBeamThreads * 4 + tid * 4;
      if (i + 4 <= here) {
        f32x4 v;  // (rows of an odd vocabulary begin off 16 bytes)
        __builtin_memcpy(&v, __builtin_assume_aligned(row + i, 4), 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[u][j] = v[j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[u][j] = i + j < here ? row[i + j] : -INFINITY;
      }
    }
    if (tid == 0) count = 0;
    float own = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) own = fmaxf(own, fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3])));
    const float wave_top = wave_max(own), bound = nth_in_wave(own, W, lane);
    if (lane == 0) {
      tops[wave] = wave_top;
      bounds[wave] = bound;
    }
    __syncthreads();
    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), least = fmaxf(fmaxf(bounds[0], bounds[1]), fmaxf(bounds[2], bounds[3]));
    double sum = 0.0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (x[u][j] >= least && finite(x[u][j])) {
          const int n = atomicAdd(&count, 1);
          if (n < kFew) {
            few.piece.logit[n] = x[u][j];
            few.piece.at[n] = u * kBeamThreads * 4 + tid * 4 + j;
          }
        }
        sum += x[u][j] == -INFINITY ? 0.f : exp_below(x[u][j], top);
      }
    sum = sum_over(sum, 64);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    uint64_t* room = a.room + ((g * W + w) * a.parts + part) * stride;
    const int n = count;
    int found = n < W ? n : W;
    if (n <= kFew) {
      for (int i = tid; i < n; i += kBeamThreads) {
        const float mine = few.piece.logit[i];
        const int at = few.piece.at[i];
        int rank = 0;
        for (int k = 0; k < n; ++k) rank += few.piece.logit[k] > mine || (few.piece.logit[k] == mine && few.piece.at[k] < at) ? 1 : 0;
        if (rank < W) put(room + 2 + rank, pair_of(mine, static_cast<unsigned>(from + at)));
      }
    } else {
      float last = INFINITY;
      int last_at = -1;
      for (found = 0; found < W; ++found) {
        Key best = no_key();
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const Key k{0.0, x[u][j], 0, u * kBeamThreads * 4 + tid * 4 + j};
            if (finite(k.logit) && (k.logit < last || (k.logit == last && k.token > last_at)) && before(k, best)) best = k;
          }
        best = first_in_block(best, slots);
        if (best.token == INT32_MAX) break;
        last = best.logit;
        last_at = best.token;
        if (tid == 0) put(room + 2 + found, pair_of(last, static_cast<unsigned>(from + last_at)));
      }
    }
    if (tid == 0) {
      put(room, pair_of(top, static_cast<unsigned>(found)));
      put(room + 1, __builtin_bit_cast(uint64_t, ((sums[0] + sums[1]) + sums[2]) + sums[3]));
    }
  }
  // ---- whoever is last among the group's workgroups.  What they left passes the L2 (the XCDs' are not coherent); an arrival is counted once its own has drained
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const unsigned arrived = __hip_atomic_fetch_add(a.arrivals + g, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    flag = arrived == static_cast<unsigned>(W) * a.parts - 1;
    if (flag) put(a.arrivals + g, 0u);  // re-armed for the next launch
    count = 0;
  }
  __syncthreads();
  if (!flag) return;
  const uint64_t* room = a.room + g * W * a.parts * stride;
  const float* scores = a.scores + g * W;
  const int* done = a.done ? a.done + g * W : nullptr;
  // the beams' sums, several beams to a wavefront where there are few parts
  int width = 1;
  while (width < a.parts && width < 64) width *= 2;
  const int each = 64 / width, sub = lane / width, first = lane - sub * width;
  for (int i0 = wave * each; i0 < W; i0 += kBeamWaves * each) {
    const int i = i0 + sub;
    const bool plain_row = i < W && finite(scores[i]) && !(done && done[i] != 0);
    float m = -INFINITY;
    double s = 0.0;
    if (plain_row && first < a.parts) {
      m = first_of(get(room + (i * a.parts + first) * stride));
      s = __builtin_bit_cast(double, get(room + (i * a.parts + first) * stride + 1));
    }
    for (int p = first + 64; plain_row && p < a.parts; p += 64) {  // (parts of one lane's: one sum on the larger maximum)
      const float o = first_of(get(room + (i * a.parts + p) * stride)), both = fmaxf(m, o);
      const double t = __builtin_bit_cast(double, get(room + (i * a.parts + p) * stride + 1));
      s = (m == -INFINITY ? s : s * exp(static_cast<double>(m) - static_cast<double>(both))) + (o == -INFINITY ? t : t * exp(static_cast<double>(o) - static_cast<double>(both)));
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
  auto is_done = [&](int i) { return done && done[i] != 0; };
  auto normal = [&](int i) { return finite(scores[i]) && !is_done(i) && finite(top_of[i]) && fabs(log_sum[i]) < INFINITY; };
  auto key_of = [&](int i, uint64_t one) {
    const float x = first_of(one);
    return Key{static_cast<double>(scores[i]) + ((static_cast<double>(x) - static_cast<double>(top_of[i])) - log_sum[i]), x, i, static_cast<int>(one >> 32)};
  };
  auto ended_key = [&](int i) { return Key{static_cast<double>(scores[i]), 0.f, i, static_cast<int>(a.eos)}; };
  auto goes_on = [&](int i) { return finite(scores[i]) && is_done(i) && a.eos >= 0 && a.eos < a.V; };
  // the lists' first candidates (a beam that is done has one, in its first part's place), and the bound that they give
  const int lists = W * a.parts;
  double own = -INFINITY;
  for (int t = tid; t < lists; t += kBeamThreads) {
    const int i = t / a.parts;
    if (normal(i)) {
      const uint64_t head = get(room + static_cast<int64_t>(t) * stride), one = get(room + static_cast<int64_t>(t) * stride + 2);
      if (static_cast<int>(head >> 32) > 0) own = fmax(own, key_of(i, one).score);
    } else if (t == i * a.parts && goes_on(i)) {
      own = fmax(own, ended_key(i).score);
    }
  }
  const double bound = nth_in_wave(own, W, lane);
  if (lane == 0) key_bounds[wave] = bound;
  __syncthreads();
  const double least = fmax(fmax(key_bounds[0], key_bounds[1]), fmax(key_bounds[2], key_bounds[3]));
  auto keep = [&](const Key& k) {
    const int n = atomicAdd(&count, 1);
    if (n >= kFewKeys) return;
    few.all.score[n] = k.score;
    few.all.logit[n] = k.logit;
    few.all.beam[n] = k.beam;
    few.all.token[n] = k.token;
  };
  for (int t = tid; t < lists; t += kBeamThreads) {
    const int i = t / a.parts;
    if (normal(i)) {
      const uint64_t* at = room + static_cast<int64_t>(t) * stride;
      const int n = static_cast<int>(get(at) >> 32);
      bool more = n > 0;
      for (int k0 = 0; more; k0 += 4) {
        uint64_t some[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) some[u] = get(at + 2 + (k0 + u < n ? k0 + u : n - 1));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const Key k = key_of(i, some[u]);
          more = more && k0 + u < n && k.score >= least;
          if (more) keep(k);
        }
      }
    } else if (t == i * a.parts && goes_on(i)) {
      keep(ended_key(i));
    }
  }
  __syncthreads();
  const int n = count;
  int found = n < W ? n : W;
  if (n <= kFewKeys) {
    for (int i = tid; i < n; i += kBeamThreads) {
      const Key mine{few.all.score[i], few.all.logit[i], few.all.beam[i], few.all.token[i]};
      int rank = 0;
      for (int k = 0; k < n; ++k) rank += before(Key{few.all.score[k], few.all.logit[k], few.all.beam[k], few.all.token[k]}, mine) ? 1 : 0;
      if (rank < W) {
        chosen_beam[rank] = mine.beam;
        chosen_token[rank] = mine.token;
        chosen_score[rank] = static_cast<float>(mine.score);
      }
    }
  } else {
    Key last = no_key();
    for (found = 0; found < W; ++found) {
      Key best = no_key();
      auto offer = [&](const Key& k) {
        if ((found == 0 || before(last, k)) && before(k, best)) best = k;
      };
      for (int t = tid; t < lists; t += kBeamThreads) {
        const int i = t / a.parts;
        const uint64_t* at = room + static_cast<int64_t>(t) * stride;
        const int many = normal(i) ? static_cast<int>(get(at) >> 32) : 0;
        for (int k = 0; k < many; ++k) offer(key_of(i, get(at + 2 + k)));
        if (t == i * a.parts && goes_on(i)) offer(ended_key(i));
      }
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
  const bool mine = tid < W;
  const int parent = mine ? chosen_beam[tid] : 0, token = mine ? chosen_token[tid] : 0;
  const bool ended = (done && done[parent] != 0) || token == a.eos;
  __syncthreads();  // (scores and done may be the outputs: they have been read)
  if (!mine) return;
  a.parents[g * W + tid] = parent;
  a.tokens[g * W + tid] = token;
  a.new_scores[g * W + tid] = chosen_score[tid];
  if (a.new_done) a.new_done[g * W + tid] = ended ? 1 : 0;
}

constexpr int64_t kBeamWords = int64_t{1} << 25, kBeamPiece = kBeamThreads * 4 * 2;  // (64-bit words of a launch; the smallest piece)
template <int U>
int launch_beam(BeamArgs a, int64_t groups, hipStream_t s) {
  a.parts = static_cast<int>(ceil_div(a.V, kBeamThreads * 4 * U));
  const int64_t per_group = static_cast<int64_t>(a.beams) * a.parts, words = per_group * (2 + a.beams);
  // as many groups at a time as 256 MiB of the workspace, and a grid, hold
  int64_t some = kBeamWords / words;
  if (some > 65535) some = 65535;
  for (int64_t g = 0; g < groups; g += some) {
    const int64_t now = groups - g < some ? groups - g : some;
    float* room = nullptr;
    std::unique_lock<std::recursive_mutex> lock;
    if (split_scratch(s, static_cast<size_t>(now * words) * 8, static_cast<size_t>(now), a.parts, &room, &a.arrivals, &lock) != 0) return -1;
    a.room = reinterpret_cast<uint64_t*>(room);
    hipLaunchKernelGGL(beam_select_kernel<U>, dim3(static_cast<unsigned>(a.parts), static_cast<unsigned>(a.beams), static_cast<unsigned>(now)), dim3(kBeamThreads), 0, s, a);
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
  if (V > INT32_MAX || groups > INT32_MAX || V > (int64_t{1} << 60) / beams / groups) return fail("beam_select: the extents overflow");
  if (beams * ceil_div(V, kBeamPiece) * (2 + beams) > kBeamWords) return fail("beam_select: a vocabulary of %lld is too large", (long long)V);
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
             static_cast<float*>(new_scores), static_cast<int*>(new_done), static_cast<int>(beams), 0, V, eos, nullptr, nullptr};
  hipStream_t s = static_cast<hipStream_t>(stream);
  // pieces of 2048, 4096 or 8192 logits: as many workgroups as two per CU, or as fill the chip while the pieces are the smallest
  if (rows * ceil_div(V, 8192) >= 512) return launch_beam<8>(a, groups, s);
  if (rows * ceil_div(V, 4096) >= 512) return launch_beam<4>(a, groups, s);
  return launch_beam<2>(a, groups, s);
}
