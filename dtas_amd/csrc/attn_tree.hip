// Attention of a tree of drafted tokens over a key/value cache, for gfx950.
//
//   row (b, t, h): query t of sequence b, query head h, which shares key head h / (heads / kv_heads)
//   sees the keys [0, lens[b]) of the cache, the nodes on the path from its own node up to a root, and its own node
//   out[b, t, h, :] = sum_j softmax_j(scale * Q[b, t, h, :] . k_j) v_j                   fp32 scores, statistics and sums
//
// The nodes' own keys and values lie beside the cache (only what is accepted later joins it).  A node's parent is parents[b][node]
// if that lies in [0, node), and none otherwise: whatever the buffer holds, it describes a forest.  Nothing is read of the cache
// behind lens[b], and what the other nodes of the tree hold, infinities and NaN included, does not reach a row that does not see them.
#include "dtas_device.h"
#include "dtas_host.h"

namespace dtas {
namespace {

struct TreeArgs {
  const half_t *Q, *K, *V, *Kc, *Vc;
  const int *lens, *parents;
  half_t* out;
  int T, Tq, heads, kv_heads, d;
  int64_t capacity;
  float scale_log2;  // scale * log2(e): the softmax is taken in powers of two
};

__device__ __forceinline__ int64_t clamp_len(int len, int64_t capacity) {
  return len < 0 ? 0 : len > capacity ? capacity : static_cast<int64_t>(len);
}

// any head dimension up to 256 and any alignment: one wavefront per row, one pass with the running maximum and sum
__global__ void __launch_bounds__(64) attn_tree_scalar_kernel(TreeArgs a, int64_t rows) {
  const int lane = threadIdx.x;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int h = static_cast<int>(r % a.heads), hk = h / (a.heads / a.kv_heads);
    const int64_t bt = r / a.heads;
    const int t = static_cast<int>(bt % a.Tq);
    const int64_t b = bt / a.Tq;
    const half_t* q = a.Q + r * a.d;
    float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) qv[i] = lane + 64 * i < a.d ? static_cast<float>(q[lane + 64 * i]) : 0.f;
    float top = -INFINITY, sum = 0.f;
    auto visit = [&](const half_t* k, const half_t* v) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < a.d) s = fmaf(qv[i], static_cast<float>(k[lane + 64 * i]), s);
      s = wave_sum(s) * a.scale_log2;
      const float next = fmaxf(top, s);
      const float keep = next == -INFINITY ? 1.f : exp2f(top - next), p = next == -INFINITY ? 0.f : exp2f(s - next);
      top = next;
      sum = fmaf(sum, keep, p);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < a.d) o[i] = fmaf(o[i], keep, p * static_cast<float>(v[lane + 64 * i]));
    };
    const int64_t len = clamp_len(a.lens[b], a.capacity), cached = (b * a.kv_heads + hk) * a.capacity;
    for (int64_t j = 0; j < len; ++j) visit(a.Kc + (cached + j) * a.d, a.Vc + (cached + j) * a.d);
    for (int node = a.T - a.Tq + t;;) {
      const int64_t at = ((b * a.T + node) * a.kv_heads + hk) * a.d;
      visit(a.K + at, a.V + at);
      const int up = a.parents[b * a.T + node];
      if (up < 0 || up >= node) break;
      node = up;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < a.d) a.out[r * a.d + lane + 64 * i] = static_cast<half_t>(o[i] / sum);
  }
}

}  // namespace
}  // namespace dtas

extern "C" int dtas_attn_tree_f16(const void* Q, const void* K, const void* V, const void* K_cache, const void* V_cache, const void* lens,
                                  const void* parents, void* out, int64_t batch, int64_t nodes, int64_t rows, int64_t heads,
                                  int64_t kv_heads, int64_t d, int64_t capacity, float scale, void* stream) {
  using namespace dtas;
  clear_error();
  if (batch < 0 || nodes < 0 || rows < 0 || heads < 0 || kv_heads < 0 || d < 0 || capacity < 0)
    return fail("attn_tree: negative extent batch=%lld nodes=%lld rows=%lld heads=%lld kv_heads=%lld d=%lld capacity=%lld", (long long)batch,
                (long long)nodes, (long long)rows, (long long)heads, (long long)kv_heads, (long long)d, (long long)capacity);
  if (nodes > DTAS_MAX_TREE_NODES) return fail("attn_tree: a tree holds up to %d nodes, got %lld", DTAS_MAX_TREE_NODES, (long long)nodes);
  if (rows > nodes) return fail("attn_tree: %lld query rows of a tree of %lld nodes", (long long)rows, (long long)nodes);
  if (batch == 0 || rows == 0 || heads == 0 || d == 0) return 0;
  if (kv_heads == 0 || heads % kv_heads != 0)
    return fail("attn_tree: %lld query heads do not share %lld key heads evenly", (long long)heads, (long long)kv_heads);
  if (d > 256) return fail("attn_tree: head dimensions up to 256, got %lld", (long long)d);
  constexpr int64_t kMost = int64_t{1} << 60;
  if (heads > 65535 || batch > (int64_t{1} << 31) || capacity > INT32_MAX || capacity > kMost / d / kv_heads / batch)
    return fail("attn_tree: the extents overflow");
  if (!(scale >= -3.0e38f && scale <= 3.0e38f)) return fail("attn_tree: the scale is not a finite number");
  if (!Q || !K || !V || !lens || !parents || !out || (capacity > 0 && (!K_cache || !V_cache))) return fail("attn_tree: NULL buffer");
  const int64_t out_bytes = batch * rows * heads * d * 2, new_bytes = batch * nodes * kv_heads * d * 2, cache_bytes = batch * kv_heads * capacity * d * 2;
  if (overlaps(out, out_bytes, Q, out_bytes) || overlaps(out, out_bytes, K, new_bytes) || overlaps(out, out_bytes, V, new_bytes) ||
      overlaps(out, out_bytes, K_cache, cache_bytes) || overlaps(out, out_bytes, V_cache, cache_bytes) || overlaps(out, out_bytes, lens, batch * 4) ||
      overlaps(out, out_bytes, parents, batch * nodes * 4))
    return fail("attn_tree: output overlaps an input");
  TreeArgs a{static_cast<const half_t*>(Q), static_cast<const half_t*>(K), static_cast<const half_t*>(V), static_cast<const half_t*>(K_cache),
             static_cast<const half_t*>(V_cache), static_cast<const int*>(lens), static_cast<const int*>(parents), static_cast<half_t*>(out),
             static_cast<int>(nodes), static_cast<int>(rows), static_cast<int>(heads), static_cast<int>(kv_heads), static_cast<int>(d), capacity,
             scale * 1.4426950408889634f};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t total = batch * rows * heads;
  const int64_t grid = total < (int64_t{1} << 22) ? total : int64_t{1} << 22;
  hipLaunchKernelGGL(attn_tree_scalar_kernel, dim3(static_cast<unsigned>(grid)), dim3(64), 0, s, a, total);
  return check_launch("attn_tree");
}
