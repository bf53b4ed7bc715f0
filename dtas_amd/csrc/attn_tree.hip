// Attention of a tree of drafted tokens over a key/value cache, for gfx950.
//
//   row (b, t, h): query t of sequence b, query head h, which shares key head h / (heads / kv_heads)
//   sees the keys [0, lens[b]) of the cache, the nodes on the path from its own node up to a root, and its own node
//   out[b, t, h, :] = sum_j softmax_j(scale * Q[b, t, h, :] . k_j) v_j                   fp32 scores, statistics and sums
//
// The nodes' own keys and values lie beside the cache (only what is accepted later joins it).  A node's parent is parents[b][node]
// if that lies in [0, node), and none otherwise: whatever the buffer holds, it describes a forest.  Nothing is read of the cache
// behind lens[b], and what the other nodes of the tree hold, infinities and NaN included, does not reach a row that does not see them.
#include "gemm_common.h"

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

// ---- head dimensions that are multiples of 8, data on 16-byte boundaries: the matrix cores -----------------------------------
// A workgroup serves up to 16 RT rows of one key head (its query heads' rows of all nodes: they read the same keys) and a run of
// the keys; its four wavefronts take blocks of 32 keys in turn, each for all the rows and without a barrier until the end.
//   S^T = K Q^T   A = 16 keys: a lane's 8 channels of one key are 16 contiguous bytes, loaded from memory straight into the operand's
//                 registers; B = 16 rows.  Lane l holds keys 4 (l >> 4) .. + 3 of row l & 15.
//   O^T = V^T P^T B = P^T as the scores' lanes hold it, its 8 keys per lane being 4 (l >> 4) .. + 3 of the block's two halves: the order of
//                 the keys inside an MFMA is free, so P never moves.  A = V^T in the same order: 4 keys of one channel per
//                 transposing LDS read, from the block's V rows (32 bytes longer than a row: eight rows fall on different banks).
// A wavefront holds one block of K and one of V on their way in registers while it works on the block before.
constexpr int kBlockKeys = 32;
constexpr int v_row_bytes(int DP) { return 2 * DP + 32; }
constexpr int wave_bytes(int DP) { return kBlockKeys * v_row_bytes(DP); }

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

// the nodes on the path of node `lane` up to a root, its own included, by doubling the reach six times
__device__ __forceinline__ uint64_t ancestors(const int* parents, int T, int lane) {
  int up = lane < T ? parents[lane] : -1;
  if (up < 0 || up >= lane) up = -1;
  uint64_t line = uint64_t{1} << lane;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    const int from = up < 0 ? lane : up;
    const uint64_t more = __shfl(static_cast<unsigned long long>(line), from);
    const int further = __shfl(up, from);
    if (up >= 0) line |= more;
    up = up >= 0 ? further : -1;
  }
  return line;
}

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

template <int DP, int RT, int W>
__global__ void __launch_bounds__(64 * W) attn_tree_kernel(TreeArgs a, int row_groups, int nsplit, float* __restrict__ ws,
                                                        unsigned* __restrict__ arrivals) {
  constexpr int KS = DP / 32, DT = DP / 16, VL = DP / 16;  // k steps, channel tiles, 16-byte pieces of V per lane and block
  constexpr int kRows = 16 * RT, kChunks = DP / 8;
  constexpr int kPartial = kRows * (DP + 2);               // floats of a split's share: sums, then maxima, then weights
  __shared__ __attribute__((aligned(16))) char lds[W * wave_bytes(DP)];
  __shared__ float stat_m[W][kRows], stat_l[W][kRows];
  __shared__ int last_flag;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quarter = lane >> 4, i16 = lane & 15;
  const int g = a.heads / a.kv_heads, R = a.Tq * g;
  const unsigned units = gridDim.x / row_groups;           // (key head, split) pairs; the row groups of one meet on one XCD
  const int rg = static_cast<int>(blockIdx.x / units), unit = static_cast<int>(blockIdx.x % units);
  const int bh = unit / nsplit, z = unit % nsplit, b = bh / a.kv_heads, hk = bh % a.kv_heads;
  const int64_t len = clamp_len(a.lens[b], a.capacity);
  const int cached_blocks = static_cast<int>((len + kBlockKeys - 1) / kBlockKeys), blocks = cached_blocks + (a.T + kBlockKeys - 1) / kBlockKeys;
  // a split takes at least a block per wavefront; splits beyond what that leaves have nothing to do
  int splits = (blocks + W - 1) / W;
  splits = splits < nsplit ? splits : nsplit;
  if (z >= splits) return;
  const int first = static_cast<int>(static_cast<int64_t>(blocks) * z / splits), end = static_cast<int>(static_cast<int64_t>(blocks) * (z + 1) / splits);

  // ---- the rows: operands of Q, and which nodes each sees
  f16x8 q[RT][KS];
  uint64_t sees[RT];
  const uint64_t line = end > cached_blocks ? ancestors(a.parents + static_cast<int64_t>(b) * a.T, a.T, lane) : 0;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    int r = rg * kRows + rt * 16 + i16;
    r = r < R ? r : R - 1;
    const int t = r / g;
    const half_t* row = a.Q + ((static_cast<int64_t>(b) * a.Tq + t) * a.heads + hk * g + r % g) * a.d;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int at = ks * 32 + quarter * 8;
      q[rt][ks] = at < a.d ? *reinterpret_cast<const f16x8*>(row + at) : f16x8{};
    }
    sees[rt] = __shfl(static_cast<unsigned long long>(line), a.T - a.Tq + t);
  }

  f32x4 o[RT][DT];
  float top[RT], sum[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    top[rt] = -INFINITY;
    sum[rt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  char* mine = lds + wave * wave_bytes(DP);
  const unsigned tr_at = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)mine)) +
                         (4 * quarter + (i16 >> 2)) * v_row_bytes(DP) + (i16 & 3) * 8;
  f16x8 kf[2][KS];
  u32x4 vf[VL];
  // block `blk`: of the cache, or of the nodes' own keys; rows behind its last valid key repeat that one.  A block's rows lie within 4 GiB
  struct Block {
    const char *k, *v;
    unsigned stride;  // bytes between keys
    int valid;
  };
  auto source = [&](int blk) -> Block {
    if (blk < cached_blocks) {
      const int64_t at = (static_cast<int64_t>(bh) * a.capacity + static_cast<int64_t>(blk) * kBlockKeys) * a.d;
      return {reinterpret_cast<const char*>(a.Kc + at), reinterpret_cast<const char*>(a.Vc + at), 2u * a.d, static_cast<int>(len - static_cast<int64_t>(blk) * kBlockKeys)};
    }
    const int node = (blk - cached_blocks) * kBlockKeys;
    const int64_t at = ((static_cast<int64_t>(b) * a.T + node) * a.kv_heads + hk) * a.d;
    return {reinterpret_cast<const char*>(a.K + at), reinterpret_cast<const char*>(a.V + at), 2u * a.kv_heads * a.d, a.T - node};
  };
  auto load_k = [&](const Block& s) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int row = kt * 16 + i16;
      const unsigned at = static_cast<unsigned>(row < s.valid ? row : s.valid - 1) * s.stride + quarter * 16;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kf[kt][ks] = ks * 32 + quarter * 8 < a.d ? *reinterpret_cast<const f16x8*>(s.k + (at + ks * 64)) : f16x8{};
    }
  };
  auto load_v = [&](const Block& s) {
#pragma unroll
    for (int n = 0; n < VL; ++n) {
      const int id = n * 64 + lane, row = id / kChunks, c = id % kChunks;
      const unsigned at = static_cast<unsigned>(row < s.valid ? row : s.valid - 1) * s.stride + c * 16;
      vf[n] = c * 8 < a.d ? *reinterpret_cast<const u32x4*>(s.v + at) : u32x4{0u, 0u, 0u, 0u};
    }
  };
  // one block: the scores from kf, the next block on its way (if there is one), V by way of the LDS
  auto visit = [&](auto tree_tag, int valid, int base, bool more, int next) {
    constexpr bool TREE = decltype(tree_tag)::value;
    f32x4 s[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        s[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s[rt][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[kt][ks], q[rt][ks], s[rt][kt], 0, 0, 0);
      }
    Block coming{};
    if (!TREE && more) {
      coming = source(next);
      load_k(coming);
    }
    // A value of a node that is no number must not meet the zero weights of the rows that do not see it: such a block (rare) is
    // multiplied out key by key instead
    bool odd = false;
    if (TREE) {
#pragma unroll
      for (int n = 0; n < VL; ++n)
#pragma unroll
        for (int w = 0; w < 4; ++w) odd = odd || (vf[n][w] & 0x7c00u) == 0x7c00u || (vf[n][w] & 0x7c000000u) == 0x7c000000u;
      odd = __builtin_amdgcn_ballot_w64(odd) != 0;
    }
    if (!odd) {
#pragma unroll
      for (int n = 0; n < VL; ++n) {
        const int id = n * 64 + lane, row = id / kChunks, c = id % kChunks;
        *reinterpret_cast<u32x4*>(mine + row * v_row_bytes(DP) + c * 16) = vf[n];
      }
    }
    if (!TREE && more) load_v(coming);

    f16x8 p[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float x[8], best = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = s[rt][e >> 2][e & 3] * a.scale_log2;
        const int key = (e >> 2) * 16 + 4 * quarter + (e & 3);
        if (TREE) x[e] = (sees[rt] >> (base + key)) & 1 ? x[e] : -INFINITY;
        else if (valid < kBlockKeys) x[e] = key < valid ? x[e] : -INFINITY;
        best = fmaxf(best, x[e]);
      }
      best = fmaxf(max_of_row(best), top[rt]);
      if (__builtin_amdgcn_ballot_w64(best > top[rt]) != 0) {
        const float keep = best == -INFINITY ? 1.f : exp2_fast(top[rt] - best);
        sum[rt] *= keep;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[rt][dt][j] *= keep;
        top[rt] = best;
      }
      const float from = best == -INFINITY ? 0.f : best;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = exp2_fast(x[e] - from);
        sum[rt] += x[e];
        p[rt][e] = static_cast<half_t>(x[e]);
      }
      if (TREE && odd) {
        // P by way of the LDS; a row adds up the values that it sees
        float* at_p = reinterpret_cast<float*>(mine);
#pragma unroll
        for (int e = 0; e < 8; ++e) at_p[((e >> 2) * 16 + 4 * quarter + (e & 3)) * 16 + i16] = x[e];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        for (int key = 0; key < kBlockKeys && base + key < a.T; ++key) {
          const float weight = at_p[key * 16 + i16];
          const half_t* v = a.V + ((static_cast<int64_t>(b) * a.T + base + key) * a.kv_heads + hk) * a.d;
          if ((sees[rt] >> (base + key)) & 1) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (dt * 16 + 4 * quarter < a.d) o[rt][dt][j] = fmaf(weight, static_cast<float>(v[dt * 16 + 4 * quarter + j]), o[rt][dt][j]);
          }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
    }
    if (odd) return;
    auto add = [&](int dt, const f16x4& lo, const f16x4& hi) {
      const f16x8 vt = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, p[rt], o[rt][dt], 0, 0, 0);
    };
#pragma unroll
    for (int dt = 0; dt + 4 <= DT; dt += 4) {
      f16x4 lo[4], hi[4];
      read_v<DP>(tr_at + dt * 32, lo, hi);
#pragma unroll
      for (int u = 0; u < 4; ++u) add(dt + u, lo[u], hi[u]);
    }
    if constexpr (DT % 4 == 2) {
      f16x4 lo[2], hi[2];
      read_v<DP>(tr_at + (DT - 2) * 32, lo, hi);
      add(DT - 2, lo[0], hi[0]);
      add(DT - 1, lo[1], hi[1]);
    }
  };

  // The tree's blocks, two at most, are the last ones: a wavefront has one of them at most, as its last
  int blk = first + wave;
  if (blk < end) {
    const Block s = source(blk);
    load_k(s);
    load_v(s);
  }
  for (; blk < end && blk < cached_blocks; blk += W)
    visit(std::false_type{}, static_cast<int>(len - static_cast<int64_t>(blk) * kBlockKeys), 0, blk + W < end, blk + W);
  if (blk < end) visit(std::true_type{}, 0, (blk - cached_blocks) * kBlockKeys, false, 0);

  // ---- the wavefronts' shares, joined in their order
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    sum[rt] = sum_of_row(sum[rt]);
    if (quarter == 0) {
      stat_m[wave][rt * 16 + i16] = top[rt];
      stat_l[wave][rt * 16 + i16] = sum[rt];
    }
  }
  __syncthreads();
  auto weight_of = [](float m, float best) { return best == -INFINITY ? 0.f : exp2_fast(m - best); };
  auto best_of = [&](int r) {
    float best = stat_m[0][r];
#pragma unroll
    for (int w = 1; w < W; ++w) best = fmaxf(best, stat_m[w][r]);
    return best;
  };
  const int tile = bh * row_groups + rg, my_rows = R - rg * kRows < kRows ? R - rg * kRows : kRows;
  float* share = ws + (static_cast<int64_t>(tile) * nsplit + z) * kPartial;
  auto out_row = [&](int r) -> half_t* {
    return a.out + ((static_cast<int64_t>(b) * a.Tq + r / g) * a.heads + hk * g + r % g) * a.d;
  };
  constexpr int kPitch = DP + 4;  // floats: the sixteen rows of a store start 16 bytes apart in the banks
  static_assert(16 * kPitch * 4 <= wave_bytes(DP), "a wavefront's sums of sixteen rows fit its piece of the LDS");
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row0 = rt * 16;
    if (row0 >= my_rows) break;
    {
      const float w = weight_of(top[rt], best_of(row0 + i16));
      float* to = reinterpret_cast<float*>(mine) + i16 * kPitch + 4 * quarter;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(to + dt * 16) = f32x4{o[rt][dt][0] * w, o[rt][dt][1] * w, o[rt][dt][2] * w, o[rt][dt][3] * w};
    }
    __syncthreads();
    for (int at = tid; at < 16 * (DP / 4); at += 64 * W) {
      const int i = at / (DP / 4), c = 4 * (at % (DP / 4)), r = row0 + i;
      if (r >= my_rows || c >= a.d) continue;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      float l = 0.f;
      const float best = best_of(r);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const f32x4 part = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + w * wave_bytes(DP)) + i * kPitch + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += part[j];
        l += stat_l[w][r] * weight_of(stat_m[w][r], best);
      }
      if (splits > 1) {
        store_out(v, reinterpret_cast<f32x4*>(share + r * DP + c), true);
        if (c == 0)
          __hip_atomic_store(reinterpret_cast<uint64_t*>(share + kRows * DP) + r,
                             static_cast<uint64_t>(__builtin_bit_cast(unsigned, best)) | static_cast<uint64_t>(__builtin_bit_cast(unsigned, l)) << 32,
                             __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      } else {
        const float inv = 1.f / l;
        *reinterpret_cast<f16x4*>(out_row(rg * kRows + r) + c) = f16x4{static_cast<half_t>(v[0] * inv), static_cast<half_t>(v[1] * inv),
                                                                       static_cast<half_t>(v[2] * inv), static_cast<half_t>(v[3] * inv)};
      }
    }
    __syncthreads();
  }
  if (splits == 1) return;

  // ---- the splits' shares, joined in their order by whoever arrives last.  The shares pass the L2 (the XCDs' are not coherent): once the
  // stores have drained they are visible everywhere, and only then is the arrival counted
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const unsigned before = __hip_atomic_fetch_add(arrivals + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last_flag = before == static_cast<unsigned>(splits) - 1;
    if (last_flag) __hip_atomic_store(arrivals + tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // re-armed for the next launch
  }
  __syncthreads();
  if (!last_flag) return;
  const float* shares = ws + static_cast<int64_t>(tile) * nsplit * kPartial;
  uint64_t* stats = reinterpret_cast<uint64_t*>(lds);  // [split][row]: maximum and sum; the sum turns into the split's weight
  for (int at = tid; at < splits * kRows; at += 64 * W)
    if (at % kRows < my_rows)
      stats[at] = __hip_atomic_load(reinterpret_cast<const uint64_t*>(shares + static_cast<int64_t>(at / kRows) * kPartial + kRows * DP) + at % kRows,
                                    __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  for (int at = tid; at < my_rows * (DP / 4); at += 64 * W) {
    const int i = at / (DP / 4), c = 4 * (at % (DP / 4));
    if (c >= a.d) continue;
    float best = -INFINITY, l = 0.f;
    for (int y = 0; y < splits; ++y) best = fmaxf(best, __builtin_bit_cast(float, static_cast<unsigned>(stats[y * kRows + i])));
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    constexpr int kAtOnce = 8;  // shares requested before the first is used: a trip to memory per eight splits
    for (int y0 = 0; y0 < splits; y0 += kAtOnce) {
      uint64_t one[kAtOnce], other[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int y = y0 + u < splits ? y0 + u : splits - 1;
        const uint64_t* from = reinterpret_cast<const uint64_t*>(shares + static_cast<int64_t>(y) * kPartial + i * DP + c);
        one[u] = __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        other[u] = __hip_atomic_load(from + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (y0 + u >= splits) break;
        const uint64_t two = stats[(y0 + u) * kRows + i];
        const float w = weight_of(__builtin_bit_cast(float, static_cast<unsigned>(two)), best);
        l = fmaf(w, __builtin_bit_cast(float, static_cast<unsigned>(two >> 32)), l);
        v[0] = fmaf(w, __builtin_bit_cast(float, static_cast<unsigned>(one[u])), v[0]);
        v[1] = fmaf(w, __builtin_bit_cast(float, static_cast<unsigned>(one[u] >> 32)), v[1]);
        v[2] = fmaf(w, __builtin_bit_cast(float, static_cast<unsigned>(other[u])), v[2]);
        v[3] = fmaf(w, __builtin_bit_cast(float, static_cast<unsigned>(other[u] >> 32)), v[3]);
      }
    }
    const float inv = 1.f / l;
    *reinterpret_cast<f16x4*>(out_row(rg * kRows + i) + c) = f16x4{static_cast<half_t>(v[0] * inv), static_cast<half_t>(v[1] * inv),
                                                                   static_cast<half_t>(v[2] * inv), static_cast<half_t>(v[3] * inv)};
  }
}

template <int DP, int RT, int W>
int launch_tree(const TreeArgs& a, int64_t batch, hipStream_t s) {
  constexpr int kRows = 16 * RT;
  const int64_t groups = ceil_div(static_cast<int64_t>(a.Tq) * (a.heads / a.kv_heads), kRows), tiles = batch * a.kv_heads * groups;
  // a workgroup for each CU, while a split keeps a block of keys per wavefront and the statistics of all splits fit the LDS
  constexpr int kMostSplits = 64 / RT;
  int64_t nsplit = kNumCU / tiles;
  const int64_t blocks = ceil_div(a.capacity, kBlockKeys) + ceil_div(a.T, kBlockKeys), useful = ceil_div(blocks, W);
  nsplit = nsplit > useful ? useful : nsplit;
  nsplit = nsplit > kMostSplits ? kMostSplits : nsplit;
  nsplit = nsplit < 1 ? 1 : nsplit;
  if (tiles * nsplit > INT32_MAX) return fail("attn_tree: the launch has too many workgroups");
  static_assert(kMostSplits * kRows * 8 <= W * wave_bytes(DP), "the splits' statistics fit the LDS");
  float* partials = nullptr;
  unsigned* arrivals = nullptr;
  std::unique_lock<std::recursive_mutex> lock;
  if (nsplit > 1 && split_scratch(s, static_cast<size_t>(tiles * nsplit) * kRows * (DP + 2) * sizeof(float), static_cast<size_t>(tiles),
                                  static_cast<int>(nsplit), &partials, &arrivals, &lock) != 0)
    return -1;
  hipLaunchKernelGGL((attn_tree_kernel<DP, RT, W>), dim3(static_cast<unsigned>(tiles * nsplit)), dim3(64 * W), 0, s, a, static_cast<int>(groups),
                     static_cast<int>(nsplit), partials, arrivals);
  return check_launch("attn_tree");
}

template <int DP>
int launch_tree_rows(const TreeArgs& a, int64_t batch, hipStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.Tq) * (a.heads / a.kv_heads);
  if (rows <= 16) return launch_tree<DP, 1, (DP <= 128 ? 8 : 4)>(a, batch, s);
  if (rows <= 32 || DP > 128) return launch_tree<DP, 2, (DP <= 128 ? 8 : 4)>(a, batch, s);  // (more sums than 512 registers hold, beyond 128 channels)
  if constexpr (DP <= 128) return launch_tree<DP, 4, 4>(a, batch, s);
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
  if (d % 8 == 0 && aligned(Q, 16) && aligned(K, 16) && aligned(V, 16) && aligned(K_cache, 16) && aligned(V_cache, 16) && aligned(out, 16)) {
    if (d <= 64) return launch_tree_rows<64>(a, batch, s);
    if (d <= 96) return launch_tree_rows<96>(a, batch, s);
    if (d <= 128) return launch_tree_rows<128>(a, batch, s);
    if (d <= 192) return launch_tree_rows<192>(a, batch, s);
    return launch_tree_rows<256>(a, batch, s);
  }
  const int64_t total = batch * rows * heads;
  const int64_t grid = total < (int64_t{1} << 22) ? total : int64_t{1} << 22;
  hipLaunchKernelGGL(attn_tree_scalar_kernel, dim3(static_cast<unsigned>(grid)), dim3(64), 0, s, a, total);
  return check_launch("attn_tree");
}
