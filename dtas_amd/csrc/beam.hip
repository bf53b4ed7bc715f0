// Beam search's selection over beams and vocabulary, for gfx950.
//
//   candidate (w, v) of a group: scores[w] + logits[w][v] - log sum_u exp(logits[w][u]); of a beam that is done: (w, eos) with scores[w]
//   the `beams` best, by (score descending, w, v ascending); what is no finite number counts as -inf
//
// Within a beam the order is that of the logits, so one pass over them is enough: a workgroup has a piece of one beam's logits in registers, and leaves
// its maximum, its sum of exponentials (terms in 32 bits, each product with log2 e kept to twice that; the sum in 64) and its best candidates; whoever is last
// among a group's workgroups has the sums of all and compares what is left, in 64 bits.
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

__device__ __forceinline__ double sum_in_wave(double v) {
#pragma unroll
  for (int k = 1; k < 64; k *= 2) v += __shfl_xor(v, k);
  return v;
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

template <int U>  // 16-byte pieces per thread
__global__ void __launch_bounds__(kBeamThreads) beam_select_kernel(BeamArgs a) {
  __shared__ Key slots[kBeamWaves];
  __shared__ float tops[kBeamWaves];
  __shared__ double sums[kBeamWaves];
  __shared__ double log_sum[DTAS_MAX_BEAMS];
  __shared__ float top_of[DTAS_MAX_BEAMS];
  __shared__ int chosen_beam[DTAS_MAX_BEAMS], chosen_token[DTAS_MAX_BEAMS];
  __shared__ float chosen_score[DTAS_MAX_BEAMS];
  __shared__ int flag;
  constexpr int kPiece = kBeamThreads * 4 * U;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = blockIdx.x % a.parts, w = static_cast<int>(blockIdx.x / a.parts % a.beams), W = a.beams;
  const int64_t g = blockIdx.x / a.parts / a.beams;
  const int64_t from = static_cast<int64_t>(part) * kPiece;
  const int here = static_cast<int>(a.V - from < kPiece ? a.V - from : kPiece);
  const int stride = 2 + W;
  const bool plain = finite(a.scores[g * W + w]) && !(a.done && a.done[g * W + w] != 0);
  if (plain) {
    const float* row = a.logits + (g * W + w) * a.V + from;
    float x[U][4];
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = u * kBeamThreads * 4 + tid * 4;
      if (i + 4 <= here) {
        f32x4 v;
        __builtin_memcpy(&v, __builtin_assume_aligned(row + i, 4), 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[u][j] = v[j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[u][j] = i + j < here ? row[i + j] : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, x[u][j]);
    }
    top = wave_max(top);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    double sum = 0.0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += x[u][j] == -INFINITY ? 0.f : exp_below(x[u][j], top);
    sum = sum_in_wave(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    uint64_t* room = a.room + ((g * W + w) * a.parts + part) * stride;
    // the best, one after the other
    float last = INFINITY;
    int last_at = -1, found = 0;
    for (; found < W; ++found) {
      Key best = no_key();
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = u * kBeamThreads * 4 + tid * 4 + j;
          const Key k{0.0, x[u][j], 0, at};
          if (finite(x[u][j]) && (x[u][j] < last || (x[u][j] == last && at > last_at)) && before(k, best)) best = k;
        }
      best = first_in_block(best, slots);
      if (best.token == INT32_MAX) break;
      last = best.logit;
      last_at = best.token;
      if (tid == 0) put(room + 2 + found, pair_of(last, static_cast<unsigned>(from + last_at)));
    }
    if (tid == 0) {
      put(room, pair_of(top, static_cast<unsigned>(found)));
      put(room + 1, __builtin_bit_cast(uint64_t, ((sums[0] + sums[1]) + sums[2]) + sums[3]));
    }
  }
  // ---- whoever is last among the group's workgroups.  What they left passes the L2 (the XCDs' are not coherent); an arrival is counted once its own has drained
  if (tid == 0) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const unsigned arrived = __hip_atomic_fetch_add(a.arrivals + g, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    flag = arrived == static_cast<unsigned>(W) * a.parts - 1;
    if (flag) put(a.arrivals + g, 0u);  // re-armed for the next launch
  }
  __syncthreads();
  if (!flag) return;
  const uint64_t* room = a.room + g * W * a.parts * stride;
  const float* scores = a.scores + g * W;
  const int* done = a.done ? a.done + g * W : nullptr;
  for (int i = wave; i < W; i += kBeamWaves) {
    if (!finite(scores[i]) || (done && done[i] != 0)) continue;
    float top = -INFINITY;
    for (int p = lane; p < a.parts; p += 64) top = fmaxf(top, first_of(get(room + (i * a.parts + p) * stride)));
    top = wave_max(top);
    double sum = 0.0;
    for (int p = lane; p < a.parts; p += 64) {
      const float m = first_of(get(room + (i * a.parts + p) * stride));
      const double s = __builtin_bit_cast(double, get(room + (i * a.parts + p) * stride + 1));
      sum += m == -INFINITY ? s : s * exp(static_cast<double>(m) - static_cast<double>(top));  // (a part of -inf has a sum of nought)
    }
    sum = sum_in_wave(sum);
    if (lane == 0) {
      top_of[i] = top;
      log_sum[i] = log(sum);
    }
  }
  __syncthreads();
  auto normal = [&](int i) { return finite(scores[i]) && !(done && done[i] != 0) && finite(top_of[i]) && fabs(log_sum[i]) < INFINITY; };
  Key last = no_key();
  int found = 0;
  for (; found < W; ++found) {
    Key best = no_key();
    auto offer = [&](const Key& k) {
      if ((found == 0 || before(last, k)) && before(k, best)) best = k;
    };
    for (int t = tid; t < W * a.parts; t += kBeamThreads) {
      const int i = t / a.parts;
      if (!normal(i)) continue;
      const uint64_t* at = room + static_cast<int64_t>(t) * stride;
      const int n = static_cast<int>(get(at) >> 32);
      for (int k = 0; k < n; ++k) {
        const uint64_t one = get(at + 2 + k);
        const float x = first_of(one);
        offer(Key{static_cast<double>(scores[i]) + ((static_cast<double>(x) - static_cast<double>(top_of[i])) - log_sum[i]), x, i, static_cast<int>(one >> 32)});
      }
    }
    for (int i = tid; i < W; i += kBeamThreads)
      if (done && done[i] != 0 && finite(scores[i]) && a.eos >= 0 && a.eos < a.V) offer(Key{static_cast<double>(scores[i]), 0.f, i, static_cast<int>(a.eos)});
    best = first_in_block(best, slots);
    if (best.token == INT32_MAX) break;
    last = best;
    if (tid == 0) {
      chosen_beam[found] = best.beam;
      chosen_token[found] = best.token;
      chosen_score[found] = static_cast<float>(best.score);
    }
  }
  if (tid == 0) {  // fewer candidates with a number than beams: the first of the others
    for (int i = 0, v = 0, n = found; n < W; ++v) {
      if (v == a.V) ++i, v = 0;
      bool taken = false;
      for (int k = 0; k < found; ++k) taken = taken || (chosen_beam[k] == i && chosen_token[k] == v);
      if (taken) continue;
      chosen_beam[n] = i;
      chosen_token[n] = v;
      chosen_score[n++] = -INFINITY;
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

constexpr int64_t kBeamWords = int64_t{1} << 25, kBeamPiece = kBeamThreads * 4 * 4;  // (64-bit words of a launch; the smallest piece)
template <int U>
int launch_beam(BeamArgs a, int64_t groups, hipStream_t s) {
  a.parts = static_cast<int>(ceil_div(a.V, kBeamThreads * 4 * U));
  const int64_t per_group = static_cast<int64_t>(a.beams) * a.parts, words = per_group * (2 + a.beams);
  // as many groups at a time as 256 MiB of the workspace, and a grid, hold
  int64_t some = kBeamWords / words;
  if (some > INT32_MAX / per_group) some = INT32_MAX / per_group;
  for (int64_t g = 0; g < groups; g += some) {
    const int64_t now = groups - g < some ? groups - g : some;
    float* room = nullptr;
    std::unique_lock<std::recursive_mutex> lock;
    if (split_scratch(s, static_cast<size_t>(now * words) * 8, static_cast<size_t>(now), a.parts, &room, &a.arrivals, &lock) != 0) return -1;
    a.room = reinterpret_cast<uint64_t*>(room);
    hipLaunchKernelGGL(beam_select_kernel<U>, dim3(static_cast<unsigned>(now * per_group)), dim3(kBeamThreads), 0, s, a);
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
  return launch_beam<4>(a, groups, static_cast<hipStream_t>(stream));
}
