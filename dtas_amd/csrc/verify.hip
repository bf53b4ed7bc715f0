// Drafted tokens against the target's probabilities, and what is accepted into the key/value cache, for gfx950.
#include "dtas_device.h"
#include "dtas_host.h"

namespace dtas {
namespace {

// ---- verification of a tree of drafted tokens ----------------------------------------------------------------------
// Node 0 is the last token already chosen.  target[b, i, :] is the large model's distribution behind node i, draft[b, i, :] the one
// that the children of i were drawn from, one after the other and independently.  The walk stands at a node with p, q, its rows; it
// offers the children in the order of their index.  With p' = p at first, a child with token x is accepted if accept * q(x) < p'(x); a
// child that is refused leaves p' = norm(max(p' - q, 0)).  The tokens chosen this way are distributed as the target alone would choose
// them.  p' needs no vector: after k refusals it is max(p - c q, 0) / S(c) with S(c) = sum max(p - c q, 0), where c starts at 0
// (S = 1: the rows are distributions) and grows by S with every refusal,
//     max(p - c q, 0) / S - q = max(p - (c + S) q, 0) / S   wherever it is positive,
// so a refusal costs one sum over the rows and an acceptance none.  Where no child is accepted the next token is the first v whose
// prefix sum of max(p - c q, 0) exceeds sample * total.  Sums and comparisons are in 64 bits: the products of two fp32 numbers are
// exact there, and a token is chosen next to a border of the prefix sums.
constexpr int kVerifyThreads = 1024;

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int i = 32; i > 0; i >>= 1) v += __shfl_xor(v, i);
  return v;
}

__device__ __forceinline__ double rest_of(float p, float q, double c) {
  const double w = fma(-c, static_cast<double>(q), static_cast<double>(p));
  return w > 0.0 ? w : 0.0;  // (NaN too)
}

__global__ void __launch_bounds__(kVerifyThreads) verify_tree_kernel(const float* __restrict__ target, const float* __restrict__ draft,
                                                                     const int* __restrict__ tokens, const int* __restrict__ parents,
                                                                     const float* __restrict__ accept, const float* __restrict__ sample,
                                                                     int* __restrict__ path, int* __restrict__ count, int* __restrict__ next,
                                                                     int T, int64_t V) {
  constexpr int kWaves = kVerifyThreads / 64;
  __shared__ float at_p[DTAS_MAX_TREE_NODES], at_q[DTAS_MAX_TREE_NODES], at_u[DTAS_MAX_TREE_NODES];
  __shared__ int at_parent[DTAS_MAX_TREE_NODES];
  __shared__ double part[2][kWaves];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  int phase = 0;
  if (tid < T) {
    const int parent = parents[b * T + tid], token = tokens[b * T + tid];
    const bool offered = tid > 0 && parent >= 0 && parent < tid && token >= 0 && token < V;
    at_parent[tid] = offered ? parent : -1;
    at_u[tid] = accept[b * T + tid];
    at_p[tid] = offered ? target[(b * T + parent) * V + token] : 0.f;
    at_q[tid] = offered ? draft[(b * T + parent) * V + token] : 0.f;
    path[b * T + tid] = tid == 0 ? 0 : -1;
  }
  __syncthreads();
  // the sum of max(p - c q, 0) over [lo, hi), one contiguous piece per wavefront; every thread returns with the pieces in `part`
  auto sums = [&](const float* p, const float* q, double c, int64_t lo, int64_t piece, int64_t hi) -> const double* {
    double s = 0.0;
    const int64_t from = lo + wave * piece, to = from + piece < hi ? from + piece : hi;
    for (int64_t v = from + lane; v < to; v += 64) s += rest_of(p[v], q[v], c);
    s = wave_sum64(s);
    double* bank = part[phase++ & 1];
    if (lane == 0) bank[wave] = s;
    __syncthreads();
    return bank;
  };
  int at = 0, accepted = 1;
  double c = 0.0, left = 1.0;
  for (int i = 1; i < T; ++i) {
    if (at_parent[i] != at) continue;
    const double q = static_cast<double>(at_q[i]), rest = rest_of(at_p[i], at_q[i], c);
    if (static_cast<double>(at_u[i]) * q * left < rest) {
      if (tid == 0) path[b * T + accepted] = i;
      ++accepted;
      at = i;
      c = 0.0;
      left = 1.0;
    } else {
      c += left;
      const double* bank = sums(target + (b * T + at) * V, draft + (b * T + at) * V, c, 0, (V + kWaves - 1) / kWaves, V);
      left = 0.0;
      for (int w = 0; w < kWaves; ++w) left += bank[w];
    }
  }
  const float* p = target + (b * T + at) * V;
  const float* q = draft + (b * T + at) * V;
  int64_t lo = 0, hi = V;
  double goal = 0.0, base = 0.0;
  bool first = true;
  int chosen = -1;
  while (hi > lo) {
    const int64_t piece = (hi - lo + kWaves - 1) / kWaves;
    const double* bank = sums(p, q, c, lo, piece, hi);
    if (first) {
      double total = 0.0;
      for (int w = 0; w < kWaves; ++w) total += bank[w];
      if (!(total > 0.0)) {
        if (c == 0.0) break;  // a row of zeros: there is no token
        c = 0.0;              // nothing is left of the target (its rows equal the draft's): the target itself
        continue;
      }
      const double r = static_cast<double>(sample[b]);
      goal = (r > 0.0 ? r < 1.0 ? r : 1.0 : 0.0) * total;
      first = false;
    }
    int w_at = -1;
    double before = base;
    for (int w = 0; w < kWaves; ++w) {
      if (bank[w] > 0.0) {
        w_at = w;  // (the last one with a positive sum, where rounding leaves the goal behind all of them)
        base = before;
        if (before + bank[w] > goal) break;
      }
      before += bank[w];
    }
    lo += w_at * piece;
    hi = lo + piece < hi ? lo + piece : hi;
    if (piece == 1) {
      chosen = static_cast<int>(lo);
      break;
    }
  }
  if (tid == 0) {
    count[b] = accepted;
    next[b] = chosen;
  }
}

// ---- the accepted rows into the cache -------------------------------------------------------------------------------
// cache[l, b, h, lens[b] + j, :] = new[l, b, path[b, j], h, :] for j < count[b]; no path: all rows in their order.  Rows that would
// fall outside [0, capacity), and path entries outside [0, T), are left out.  One thread per 16 bytes (or per element), of K
// (blockIdx.y = 0) and V (1).
template <typename U>
__global__ void __launch_bounds__(256) cache_append_kernel(const U* __restrict__ K, const U* __restrict__ V, const int* __restrict__ path,
                                                           const int* __restrict__ count, U* __restrict__ Kc, U* __restrict__ Vc,
                                                           const int* __restrict__ lens, int B, int T, int slots, int H, int per_row, int64_t capacity,
                                                           int64_t total) {
  const U* from = blockIdx.y ? V : K;
  U* to = blockIdx.y ? Vc : Kc;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
    // i = (((l B + b) slots + j) H + h) per_row + e
    const int e = static_cast<int>(i % per_row);
    int64_t r = i / per_row;
    const int h = static_cast<int>(r % H);
    r /= H;
    const int j = static_cast<int>(r % slots);
    r /= slots;
    const int b = static_cast<int>(r % B);
    const int64_t lb = r;
    if (count && j >= count[b]) continue;
    const int node = path ? path[static_cast<int64_t>(b) * slots + j] : j;
    const int64_t row = static_cast<int64_t>(lens[b]) + j;
    if (node < 0 || node >= T || row < 0 || row >= capacity) continue;
    to[((lb * H + h) * capacity + row) * per_row + e] = from[((lb * T + node) * H + h) * per_row + e];
  }
}

}  // namespace
}  // namespace dtas

extern "C" int dtas_verify_tree_f32(const void* target, const void* draft, const void* tokens, const void* parents, const void* accept,
                                    const void* sample, void* path, void* count, void* next, int64_t batch, int64_t nodes, int64_t V,
                                    void* stream) {
  using namespace dtas;
  clear_error();
  if (batch < 0 || nodes < 0 || V < 0) return fail("verify_tree: negative extent batch=%lld nodes=%lld V=%lld", (long long)batch, (long long)nodes, (long long)V);
  if (nodes > DTAS_MAX_TREE_NODES) return fail("verify_tree: a tree holds up to %d nodes, got %lld", DTAS_MAX_TREE_NODES, (long long)nodes);
  if (batch == 0) return 0;
  if (nodes == 0 || V == 0) return fail("verify_tree: no node, or no token, to choose from");
  if (V > INT32_MAX || batch > INT32_MAX) return fail("verify_tree: the extents overflow");
  if (!target || !draft || !tokens || !parents || !accept || !sample || !path || !count || !next) return fail("verify_tree: NULL buffer");
  const int64_t all = batch * nodes;
  struct Span { const void* at; int64_t bytes; };
  const Span in[] = {{target, all * V * 4}, {draft, all * V * 4}, {tokens, all * 4}, {parents, all * 4}, {accept, all * 4}, {sample, batch * 4}};
  const Span out[] = {{path, all * 4}, {count, batch * 4}, {next, batch * 4}};
  for (int i = 0; i < 3; ++i) {
    for (const Span& o : in)
      if (overlaps(out[i].at, out[i].bytes, o.at, o.bytes)) return fail("verify_tree: output overlaps an input");
    for (int j = 0; j < i; ++j)
      if (overlaps(out[i].at, out[i].bytes, out[j].at, out[j].bytes)) return fail("verify_tree: the outputs overlap");
  }
  hipLaunchKernelGGL(verify_tree_kernel, dim3(static_cast<unsigned>(batch)), dim3(kVerifyThreads), 0, static_cast<hipStream_t>(stream),
                     static_cast<const float*>(target), static_cast<const float*>(draft), static_cast<const int*>(tokens),
                     static_cast<const int*>(parents), static_cast<const float*>(accept), static_cast<const float*>(sample), static_cast<int*>(path),
                     static_cast<int*>(count), static_cast<int*>(next), static_cast<int>(nodes), V);
  return check_launch("verify_tree");
}

extern "C" int dtas_cache_append_f16(const void* K, const void* V, const void* path, const void* count, void* K_cache, void* V_cache,
                                     const void* lens, int64_t layers, int64_t batch, int64_t nodes, int64_t slots, int64_t kv_heads, int64_t d,
                                     int64_t capacity, void* stream) {
  using namespace dtas;
  clear_error();
  if (layers < 0 || batch < 0 || nodes < 0 || slots < 0 || kv_heads < 0 || d < 0 || capacity < 0)
    return fail("cache_append: negative extent layers=%lld batch=%lld nodes=%lld slots=%lld kv_heads=%lld d=%lld capacity=%lld", (long long)layers,
                (long long)batch, (long long)nodes, (long long)slots, (long long)kv_heads, (long long)d, (long long)capacity);
  if ((path == nullptr) != (count == nullptr)) return fail("cache_append: path and count go together");
  if (!path && slots != nodes) return fail("cache_append: without a path every row has its slot (%lld rows, %lld slots)", (long long)nodes, (long long)slots);
  if (layers == 0 || batch == 0 || nodes == 0 || slots == 0 || kv_heads == 0 || d == 0 || capacity == 0) return 0;
  constexpr int64_t kMost = int64_t{1} << 60;
  if (batch > INT32_MAX || nodes > INT32_MAX || slots > INT32_MAX || kv_heads > INT32_MAX || d > INT32_MAX || capacity > INT32_MAX ||
      batch > kMost / layers / kv_heads / d / capacity || batch > kMost / layers / kv_heads / d / nodes || batch > kMost / layers / kv_heads / d / slots)
    return fail("cache_append: the extents overflow");
  if (!K || !V || !K_cache || !V_cache || !lens) return fail("cache_append: NULL buffer");
  const int64_t new_bytes = layers * batch * nodes * kv_heads * d * 2, cache_bytes = layers * batch * kv_heads * capacity * d * 2;
  struct Span { const void* at; int64_t bytes; };
  const Span in[] = {{K, new_bytes}, {V, new_bytes}, {path, path ? batch * slots * 4 : 0}, {count, count ? batch * 4 : 0}, {lens, batch * 4}};
  for (const Span& o : in)
    if (o.at && (overlaps(K_cache, cache_bytes, o.at, o.bytes) || overlaps(V_cache, cache_bytes, o.at, o.bytes)))
      return fail("cache_append: a cache overlaps an input");
  if (overlaps(K_cache, cache_bytes, V_cache, cache_bytes)) return fail("cache_append: the caches overlap");
  const bool wide = d % 8 == 0 && aligned(K, 16) && aligned(V, 16) && aligned(K_cache, 16) && aligned(V_cache, 16);
  const int64_t per_row = wide ? d / 8 : d, total = layers * batch * slots * kv_heads * per_row;
  const int64_t grid = ceil_div(total, 256) < (int64_t{1} << 22) ? ceil_div(total, 256) : int64_t{1} << 22;
  auto go = [&](auto* tag) {
    using U = std::remove_pointer_t<decltype(tag)>;
    hipLaunchKernelGGL(cache_append_kernel<U>, dim3(static_cast<unsigned>(grid), 2), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const U*>(K), static_cast<const U*>(V), static_cast<const int*>(path), static_cast<const int*>(count),
                       static_cast<U*>(K_cache), static_cast<U*>(V_cache), static_cast<const int*>(lens), static_cast<int>(batch),
                       static_cast<int>(nodes), static_cast<int>(slots), static_cast<int>(kv_heads), static_cast<int>(per_row), capacity, total);
  };
  if (wide) go(static_cast<u32x4*>(nullptr));
  else go(static_cast<half_t*>(nullptr));
  return check_launch("cache_append");
}
