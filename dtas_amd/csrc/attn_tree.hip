// Attention of a tree of drafted tokens over a key/value cache, for gfx950.
//
//   row (b, t, h): query t of sequence b, query head h, which shares key head h / (heads / kv_heads)
//   sees the keys [0, lens[b]) of the cache, the nodes on the path from its own node up to a root, and its own node
//   out[b, t, h, :] = sum_j softmax_j(scale * Q[b, t, h, :] . k_j) v_j                   fp32 scores, statistics and sums
//
// The nodes' own keys and values lie beside the cache (only what is accepted later joins it).  A node's parent is parents[b][node]
// if that lies in [0, node), and none otherwise: whatever the buffer holds, it describes a forest.  Nothing is read of the cache
// behind lens[b], and what the other nodes of the tree hold, infinities and NaN included, does not reach a row that does not see them.
#include "attn_rows.h"

namespace dtas {
namespace {

struct TreeArgs {
  const half_t *Q, *K, *V, *Kc, *Vc;
  const int *lens, *parents;
  half_t* out;
  int T, Tq, heads, kv_heads, d;
  int64_t capacity;
  float scale_log2;  // |scale| * log2(e): the softmax is taken in powers of two
  half_t sign;       // the scale's: 1, -1, or 0 (scale_log2 is 1 then)
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
      s = wave_sum(s) * static_cast<float>(a.sign);  // (the maximum is that of the products: their differences are scaled, no product overflows by the scale)
      const float next = fmaxf(top, s);
      const float keep = next == -INFINITY ? 1.f : exp2f((top - next) * a.scale_log2), p = s == -INFINITY ? 0.f : exp2f((s - next) * a.scale_log2);  // (a score that is no number has no weight that is one)
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
// The query heads' rows of one key head (of all nodes) read the same keys and form one problem of R = Tq * heads / kv_heads rows.
//   S^T = K Q^T   A = 16 keys, B = 16 rows: lane l holds keys 4 (l >> 4) .. + 3 of row l & 15, so a row's maximum and sum take
//                 the four lanes l, l ^ 16, l ^ 32, l ^ 48.
//   O^T = V^T P^T B = P^T as the scores' lanes hold it, its 8 keys per lane being 4 (l >> 4) .. + 3 of two key tiles: the order of
//                 the keys inside an MFMA is free, so P never moves.  A = V^T in the same order: 4 keys of one channel per
//                 transposing LDS read, from V's rows (32 bytes longer than a row: eight rows fall on different banks).
// P is rounded to fp16 for its product, the type that the matrix cores take at this rate (in two halves, its products would take twice the MFMAs): 2^-11 of a weight down to
// 2^-25 of the largest, 2^-36 of that below (see kRoom).  On random inputs results are 2.5 .. 2.9e-4 off the exact ones (root mean square, relative) where rounding to fp16 at the end
// alone makes 2.1e-4.  Scores, maxima, sums and O stay in fp32.
// Two kernels: of few rows (`launch_tree_rows` says which) the wavefronts of a workgroup share the keys and load K's operands straight from memory; with more rows
// they share the rows and every key passes through the LDS once.
constexpr int k_row_bytes(int DP) { return 2 * DP + 16; }  // (the same 16 bytes of sixteen keys fall on different banks)

// the nodes on the path of node `lane`, with parent `up`, to a root, its own included, by doubling the reach six times
__device__ __forceinline__ uint64_t ancestors(int up, int lane) {
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

// the nodes that the row tiles see, from every lane's node
template <int RT>
__device__ __forceinline__ void see(uint64_t (&sees)[RT], int up, int lane, int row0, int R, int g, int T, int Tq) {
  const uint64_t line = ancestors(up, lane);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + rt * 16 + (lane & 15);
    sees[rt] = __shfl(static_cast<unsigned long long>(line), T - Tq + (r < R ? r : R - 1) / g);
  }
}

// ---- Which part of which sequence a workgroup has.  A sequence's units of keys (the blocks of its cache, those of the nodes behind) are cut into runs of
// `per` units at most, the smallest `per` with which all sequences together make no more than `budget` parts, and a sequence no more than
// `most`; its parts take consecutive slots.  A part costs what its sums take to be written and read again, all workgroups together the more the more there are:
// with a unit's time t, K parts of U units in all and w for the sums of a part of every problem it is t U / K + w K, least at
// per = U / K = `spread` sqrt(U), spread = sqrt(w / t).  Where the longest sequence in one piece, t longest, takes no more than that and the hand-over (`whole` units
// of time), nothing is cut.
struct Cut {
  int least, most, whole;
  float spread;
};
struct Part {
  int b, z, parts, first;  // sequence, which of its parts, of how many, the sequence's first slot; b < 0: nothing to do
};
__device__ __forceinline__ int units_of(int len, int64_t capacity, int unit, int T) {
  return static_cast<int>((clamp_len(len, capacity) + unit - 1) / unit) + (T + unit - 1) / unit;
}
// (the lanes hold the units of the first 64 sequences: lengths are read once unless there are more)
struct Sequences {
  const int* lens;
  int batch, unit, T;
  int64_t capacity;
  int units0;
  __device__ __forceinline__ Sequences(const TreeArgs& a, int batch_, int unit_, int lane)
      : lens(a.lens), batch(batch_), unit(unit_), T(a.T), capacity(a.capacity), units0(lane < batch_ ? units_of(a.lens[lane], a.capacity, unit_, a.T) : 0) {}
  __device__ __forceinline__ int units(int c, int lane) const { return c == 0 ? units0 : c + lane < batch ? units_of(lens[c + lane], capacity, unit, T) : 0; }
};
__device__ __forceinline__ int least_of(const Cut& cut, int total, int longest) {
  const float run = cut.spread * __builtin_amdgcn_sqrtf(static_cast<float>(total));
  if (static_cast<float>(longest) <= static_cast<float>(cut.whole) + 2.f * run) return longest;
  return run > static_cast<float>(cut.least) ? static_cast<int>(run + 0.5f) : cut.least;
}
__device__ __forceinline__ int deal(const Sequences& s, int budget, const Cut& cut, int lane) {
  int total = 0, longest = 0;
  for (int c = 0; c < s.batch; c += 64) {
    const int units = s.units(c, lane);
    total += wave_total(units);
    const int top = wave_most(units);
    longest = longest > top ? longest : top;
  }
  int per = (total + budget - 1) / budget;
  const int least = least_of(cut, total, longest);
  per = per > least ? per : least;
  per = per > (longest + cut.most - 1) / cut.most ? per : (longest + cut.most - 1) / cut.most;
  for (;;) {  // (per grows until the parts fit; with per = longest every sequence is one part, and budget >= batch)
    int parts = 0;
    for (int c = 0; c < s.batch; c += 64) parts += wave_total((s.units(c, lane) + per - 1) / per);
    if (parts <= budget || per >= longest) return per > longest ? longest : per;
    const int more = static_cast<int>(static_cast<float>(per) * parts / budget);
    per = more > per ? more : per + 1;
  }
}
__device__ __forceinline__ Part find_part(const TreeArgs& a, int batch, int unit, int slot, int budget, const Cut& cut, int lane) {
  if (budget == 0) return Part{slot, 0, 1, slot};
  if (batch == 1) {
    const int units = units_of(a.lens[0], a.capacity, unit, a.T);
    const int least = least_of(cut, units, units);
    int per = (units + budget - 1) / budget;
    per = per > least ? per : least;
    const int parts = (units + per - 1) / per;
    return Part{slot < parts ? 0 : -1, slot, parts, 0};
  }
  const Sequences s(a, batch, unit, lane);
  const int per = deal(s, budget, cut, lane);
  int base = 0;
  for (int c = 0; c < batch; c += 64) {
    const int parts = (s.units(c, lane) + per - 1) / per;
    const int upto = sum_upto(parts);
    const uint64_t here = __builtin_amdgcn_ballot_w64(slot >= base + upto - parts && slot < base + upto);
    if (here) {
      const int l = __builtin_ctzll(here);
      const int n = __builtin_amdgcn_readlane(parts, l), first = base + __builtin_amdgcn_readlane(upto, l) - n;
      return Part{c + l, slot - first, n, first};
    }
    base += __builtin_amdgcn_readlane(upto, 63);
  }
  return Part{-1, 0, 0, 0};
}

// Where a unit of keys lies: in the cache, or among the nodes' own.  Rows behind the last valid key are read as that one again: hidden, and their values
// cleared where the weight zero is multiplied with them (a node's own: where one is no number, see no_number).
struct Keys {
  const char *k, *v;
  unsigned stride;  // bytes between keys (a unit's rows lie within 4 GiB)
  int valid;
};
template <int UNIT>
__device__ __forceinline__ Keys keys_of(const TreeArgs& a, int b, int hk, int64_t len, int cached, int at) {
  if (at < cached) {
    const int64_t from = ((static_cast<int64_t>(b) * a.kv_heads + hk) * a.capacity + static_cast<int64_t>(at) * UNIT) * a.d;
    return {reinterpret_cast<const char*>(a.Kc + from), reinterpret_cast<const char*>(a.Vc + from), 2u * a.d, static_cast<int>(len - static_cast<int64_t>(at) * UNIT)};
  }
  const int node = (at - cached) * UNIT;
  const int64_t from = ((static_cast<int64_t>(b) * a.T + node) * a.kv_heads + hk) * a.d;
  return {reinterpret_cast<const char*>(a.K + from), reinterpret_cast<const char*>(a.V + from), 2u * a.kv_heads * a.d, a.T - node};
}

// Values of a node that are no numbers must not meet the zero weights of the rows that do not see it: such nodes (rare) are multiplied out
// key by key, a row adding up what it sees.  32 nodes from `base` on; s: their weights; `room`: 2 KiB of the LDS, the wavefront's own.
template <int DT>
__device__ __forceinline__ void add_key_by_key(const TreeArgs& a, int b, int hk, int base, const f32x4& s0, const f32x4& s1, uint64_t sees, float* room,
                                               int lane, f32x4 (&o)[DT]) {
  const int quarter = lane >> 4, i16 = lane & 15;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    room[(4 * quarter + j) * 16 + i16] = s0[j];
    room[(16 + 4 * quarter + j) * 16 + i16] = s1[j];
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  for (int key = 0; key < 32 && base + key < a.T; ++key) {
    const float weight = room[key * 16 + i16];
    const half_t* v = a.V + ((static_cast<int64_t>(b) * a.T + base + key) * a.kv_heads + hk) * a.d;
    if ((sees >> (base + key)) & 1) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (dt * 16 + 4 * quarter < a.d) o[dt][j] = fmaf(weight, static_cast<float>(v[dt * 16 + 4 * quarter + j]), o[dt][j]);
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// A value may be infinite where its weight is too small for fp16 (below 2^-36 of the largest): zero times infinity, though the weight is a number in fp32 and the channel
// infinite.  Such a channel shows in O, as NaN where the sum of the weights is a number (rare).  What it is instead depends on the keys alone whose values are no
// numbers: they are looked for in the units first, first + step .. that the wavefront had, and summed with their weights in fp32.  The four lanes of a row hold a quarter of
// its channels each.  (16 rows of 32 heads of 80 with such a key of 3001: 12 -> 16 us, 64 nodes after 65533 104 -> 370.)
template <int DP, int UNIT, int DT>
__device__ __forceinline__ void sum_again(const TreeArgs& a, int b, int hk, int64_t len, int cached, int first, int end, int step, int r, uint64_t sees, float top, float sum,
                                          int lane, f32x4 (&o)[DT]) {
  constexpr int KS = DP / 32;
  f32x4 all = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (dt * 16 + 16 <= below(DP) || dt * 16 + 4 * (lane >> 4) < a.d) all[j] += o[dt][j];
  const float any = (all[0] + all[1]) + (all[2] + all[3]);
  const bool mine = any != any && sum == sum;
  if (__builtin_amdgcn_ballot_w64(mine) == 0) return;
  asm volatile("" : "+v"(lane), "+v"(r));  // (nothing of what follows is computed ahead)
  const int quarter = lane >> 4, g = a.heads / a.kv_heads, R = a.Tq * g, have = r < R ? r : R - 1;
  const half_t* row = a.Q + ((static_cast<int64_t>(b) * a.Tq + have / g) * a.heads + hk * g + have % g) * a.d;
  f16x8 q[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) q[ks] = load_query<DP>(row, ks, quarter, a.d, a.sign);
  f32x4 fresh[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) fresh[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  bool open = mine;  // (a lane whose channels have all become NaN has its answer)
  for (int at = first; at < end && __builtin_amdgcn_ballot_w64(open) != 0; at += step) {
    const Keys s = keys_of<UNIT>(a, b, hk, len, cached, at);
    bool odd = false;
    if (lane < UNIT && lane < s.valid)
      for (int c = 0; c < a.d; c += 8) odd = odd || no_number(*reinterpret_cast<const u32x4*>(s.v + static_cast<unsigned>(lane) * s.stride + 2 * c));
    for (uint64_t keys = __builtin_amdgcn_ballot_w64(odd); keys != 0 && __builtin_amdgcn_ballot_w64(open) != 0; keys &= keys - 1) {
      const int key = __builtin_ctzll(keys);
      float t = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const f16x8 k = load_channels<DP>(s.k + static_cast<unsigned>(key) * s.stride, ks, quarter, a.d);
#pragma unroll
        for (int e = 0; e < 8; ++e) t = fmaf(static_cast<float>(k[e]), static_cast<float>(q[ks][e]), t);
      }
      t = sum_of_row(t);
      const float weight = t == -INFINITY ? 0.f : exp2_fast(fmaf(t - top, a.scale_log2, kRoom));
      const bool shown = at < cached || ((sees >> ((at - cached) * UNIT + key)) & 1);
      const half_t* v = reinterpret_cast<const half_t*>(s.v + static_cast<unsigned>(key) * s.stride);
      float most = __builtin_nanf("");
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        if (dt * 16 + 16 <= below(DP) || dt * 16 + 4 * quarter < a.d) {
          const f16x4 some = *reinterpret_cast<const f16x4*>(v + dt * 16 + 4 * quarter);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            fresh[dt][j] = shown ? fmaf(weight, static_cast<float>(some[j]), fresh[dt][j]) : fresh[dt][j];
            most = fmaxf(most, fresh[dt][j]);
          }
        }
      open = mine && most == most;
    }
  }
  if (mine) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[dt][j] = o[dt][j] != o[dt][j] ? fresh[dt][j] : o[dt][j];
  }
}

__device__ __forceinline__ half_t* out_row(const TreeArgs& a, int b, int hk, int g, int r) {
  return a.out + ((static_cast<int64_t>(b) * a.Tq + r / g) * a.heads + hk * g + r % g) * a.d;
}
template <int DP, int ROWS, int THREADS>
__device__ __forceinline__ void join_parts(const TreeArgs& a, int b, int hk, int g, int row0, int my_rows, const float* shares, int parts, uint64_t* stats) {
  constexpr int kShare = ROWS * (DP + 2), kAtOnce = 8;  // parts requested before the first is used: a trip to memory per eight
  const int tid = threadIdx.x;
  uint64_t one[kAtOnce], other[kAtOnce];
  auto request = [&](int at, int y0) {
    const int i = at / (DP / 4), c = 4 * (at % (DP / 4));
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int y = y0 + u < parts ? y0 + u : parts - 1;
      const uint64_t* from = reinterpret_cast<const uint64_t*>(shares + static_cast<int64_t>(y) * kShare + i * DP + c);
      one[u] = __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      other[u] = __hip_atomic_load(from + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  };
  // (the thread's first sums are on their way while the statistics come)
  const int last = my_rows * (DP / 4);
  if (tid < last) request(tid, 0);
  for (int at = tid; at < parts * ROWS; at += THREADS)
    if (at % ROWS < my_rows)
      stats[at] = __hip_atomic_load(reinterpret_cast<const uint64_t*>(shares + static_cast<int64_t>(at / ROWS) * kShare + ROWS * DP) + at % ROWS, __ATOMIC_RELAXED,
                                    __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  for (int at = tid; at < last; at += THREADS) {
    const int i = at / (DP / 4), c = 4 * (at % (DP / 4));
    if (at != tid) request(at, 0);
    float best = -INFINITY, l = 0.f;
    for (int y = 0; y < parts; ++y) best = fmaxf(best, __builtin_bit_cast(float, static_cast<unsigned>(stats[y * ROWS + i])));
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int y0 = 0; y0 < parts; y0 += kAtOnce) {
      if (y0 > 0) request(at, y0);
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (y0 + u >= parts) break;
        const uint64_t two = stats[(y0 + u) * ROWS + i];
        const float w = weight_of(__builtin_bit_cast(float, static_cast<unsigned>(two)), best, a.scale_log2);
        l = fmaf(w, __builtin_bit_cast(float, static_cast<unsigned>(two >> 32)), l);
        v[0] = fmaf(w, __builtin_bit_cast(float, static_cast<unsigned>(one[u])), v[0]);
        v[1] = fmaf(w, __builtin_bit_cast(float, static_cast<unsigned>(one[u] >> 32)), v[1]);
        v[2] = fmaf(w, __builtin_bit_cast(float, static_cast<unsigned>(other[u])), v[2]);
        v[3] = fmaf(w, __builtin_bit_cast(float, static_cast<unsigned>(other[u] >> 32)), v[3]);
      }
    }
    if (c < a.d) store_row4(out_row(a, b, hk, g, row0 + i) + c, v, 1.f / l);
  }
}

// What a launch is made of: workgroup u has slot u % slots of key head (u / slots) % kv_heads and rows from (u / slots / kv_heads) on.
struct TreeGrid {
  int batch, slots, budget, row_groups;
  Cut cut;
  float* ws;
  unsigned* arrivals;
  int* dealt;  // [batch][2], for the launch that joins many rows: a sequence's parts and its first slot
};

// ---- few rows: the W wavefronts take blocks of 32 keys in turn, each for all 16 RT rows and without a barrier until the end.  A lane's 8 channels
// of one key are 16 contiguous bytes, K's operand as it lies in memory; V passes through a piece of the LDS that is the wavefront's
// own.  One block of K and one of V are on their way in registers while the block before is worked on.
// 4 keys of one channel, from 8 bytes of the LDS that each lane names
__device__ __forceinline__ f16x4 read_transposed(const char* at) {
  typedef __attribute__((__vector_size__(4 * sizeof(__fp16)))) __fp16 fp16x4;
  return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4*)at));
}

template <int DP, int RT, int W>
__global__ void __launch_bounds__(64 * W) attn_tree_kernel(TreeArgs a, TreeGrid grid) {
  constexpr int KS = DP / 32, DT = DP / 16, VL = DP / 16, kBlock = 32;  // k steps, channel tiles, 16-byte pieces of V per lane, keys
  constexpr int kRows = 16 * RT, kChunks = DP / 8, kWave = kBlock * v_row_bytes(DP);
  __shared__ __attribute__((aligned(16))) char lds[W * kWave];
  __shared__ float stat_m[W][kRows], stat_l[W][kRows];
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quarter = lane >> 4, i16 = lane & 15;
  const int g = a.heads / a.kv_heads, R = a.Tq * g;
  const int slot = static_cast<int>(blockIdx.x % grid.slots), hk = static_cast<int>(blockIdx.x / grid.slots % a.kv_heads), rg = static_cast<int>(blockIdx.x / grid.slots / a.kv_heads);
  const Part part = find_part(a, grid.batch, kBlock, slot, grid.budget, grid.cut, lane);
  if (part.b < 0) return;
  const int b = part.b;
  const int64_t len = clamp_len(a.lens[b], a.capacity);
  const int cached = static_cast<int>((len + kBlock - 1) / kBlock), blocks = cached + (a.T + kBlock - 1) / kBlock;
  const int first = static_cast<int>(static_cast<int64_t>(blocks) * part.z / part.parts), end = static_cast<int>(static_cast<int64_t>(blocks) * (part.z + 1) / part.parts);
  const int up = lane < a.T ? a.parents[static_cast<int64_t>(b) * a.T + lane] : -1;

  f16x8 kf[2][KS];
  u32x4 vf[VL];
  auto load_k = [&](const Keys& s) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int row = kt * 16 + i16;
      const unsigned at = static_cast<unsigned>(row < s.valid ? row : s.valid - 1) * s.stride;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kf[kt][ks] = load_channels<DP>(s.k + at, ks, quarter, a.d);
    }
  };
  auto load_v = [&](const Keys& s) {
#pragma unroll
    for (int n = 0; n < VL; ++n) {
      const int id = n * 64 + lane, row = id / kChunks, c = id % kChunks;
      const unsigned at = static_cast<unsigned>(row < s.valid ? row : s.valid - 1) * s.stride + (c * 8 < a.d ? c : a.d / 8 - 1) * 16;
      vf[n] = *reinterpret_cast<const u32x4*>(s.v + at);
    }
  };
  // the tree's blocks, two at most, are the last ones: a wavefront has one of them at most, as its last
  int blk = first + wave;
  if (blk < end) {
    const Keys s = keys_of<kBlock>(a, b, hk, len, cached, blk);
    load_k(s);
    load_v(s);
  }
  f16x8 q[RT][KS];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = rg * kRows + rt * 16 + i16, have = r < R ? r : R - 1;
    const half_t* row = a.Q + ((static_cast<int64_t>(b) * a.Tq + have / g) * a.heads + hk * g + have % g) * a.d;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[rt][ks] = load_query<DP>(row, ks, quarter, a.d, a.sign);
  }
  uint64_t sees[RT] = {};
  if (end > cached) see(sees, up, lane, rg * kRows, R, g, a.T, a.Tq);

  f32x4 o[RT][DT];
  float top[RT], sum[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    top[rt] = -INFINITY;
    sum[rt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  char* mine = lds + wave * kWave;
  const unsigned tr_at = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)mine)) +
                         (4 * quarter + (i16 >> 2)) * v_row_bytes(DP) + (i16 & 3) * 8;

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
    Keys coming{};
    if (!TREE && more) {
      coming = keys_of<kBlock>(a, b, hk, len, cached, next);
      load_k(coming);
    }
    bool odd = false;
    if (TREE) {
#pragma unroll
      for (int n = 0; n < VL; ++n) odd = odd || no_number(vf[n]);
      odd = __builtin_amdgcn_ballot_w64(odd) != 0;
    }
    if (!TREE && valid < kBlock) {  // (the weight of what lies behind the last key is zero, its value has to be as well: that key's own may be no number)
#pragma unroll
      for (int n = 0; n < VL; ++n)
        if ((n * 64 + lane) / kChunks >= valid) vf[n] = u32x4{0u, 0u, 0u, 0u};
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
      if (TREE) weigh<2, DT>(s[rt], false, sees[rt] >> base, quarter, a.scale_log2, top[rt], sum[rt], o[rt]);
      else weigh<2, DT>(s[rt], valid >= kBlock, first_bits(valid), quarter, a.scale_log2, top[rt], sum[rt], o[rt]);
      p[rt] = weights_f16(s[rt][0], s[rt][1]);
      if (TREE && odd) add_key_by_key<DT>(a, b, hk, base, s[rt][0], s[rt][1], sees[rt], reinterpret_cast<float*>(mine), lane, o[rt]);
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
  for (; blk < end && blk < cached; blk += W)
    visit(std::false_type{}, static_cast<int>(len - static_cast<int64_t>(blk) * kBlock < kBlock ? len - static_cast<int64_t>(blk) * kBlock : kBlock), 0, blk + W < end, blk + W);
  if (blk < end) visit(std::true_type{}, 0, (blk - cached) * kBlock, false, 0);

  // ---- the wavefronts' shares, joined in their order
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    sum[rt] = sum_of_row(sum[rt]);
    sum_again<DP, kBlock>(a, b, hk, len, cached, first + wave, end, W, rg * kRows + rt * 16 + i16, sees[rt], top[rt], sum[rt], lane, o[rt]);
    if (quarter == 0) {
      stat_m[wave][rt * 16 + i16] = top[rt];
      stat_l[wave][rt * 16 + i16] = sum[rt];
    }
  }
  __syncthreads();
  auto best_of = [&](int r) {
    float best = stat_m[0][r];
#pragma unroll
    for (int w = 1; w < W; ++w) best = fmaxf(best, stat_m[w][r]);
    return best;
  };
  const int my_rows = R - rg * kRows < kRows ? R - rg * kRows : kRows, problem = hk * grid.row_groups + rg;
  float* shares = grid.ws + (static_cast<int64_t>(problem) * grid.slots + part.first) * (kRows * (DP + 2));
  float* share = shares + static_cast<int64_t>(part.z) * (kRows * (DP + 2));
  constexpr int kPitch = DP + 4;  // floats: the sixteen rows of a store start 16 bytes apart in the banks
  static_assert(16 * kPitch * 4 <= kWave, "a wavefront's sums of sixteen rows fit its piece of the LDS");
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row0 = rt * 16;
    if (row0 >= my_rows) break;
    {
      const float w = weight_of(top[rt], best_of(row0 + i16), a.scale_log2);
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
        const f32x4 some = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + w * kWave) + i * kPitch + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += some[j];
        l += stat_l[w][r] * weight_of(stat_m[w][r], best, a.scale_log2);
      }
      if (part.parts > 1) {
        store_out(v, reinterpret_cast<f32x4*>(share + r * DP + c), true);
        if (c == 0) store_stat(share, kRows, DP, r, best, l);
      } else {
        store_row4(out_row(a, b, hk, g, rg * kRows + r) + c, v, 1.f / l);
      }
    }
    __syncthreads();
  }
  if (part.parts == 1 || !last_to_arrive(grid.arrivals + static_cast<int64_t>(problem) * grid.batch + b, part.parts, &flag)) return;
  static_assert(64 / RT * kRows * 8 <= W * kWave, "the parts' statistics fit the LDS");
  join_parts<DP, kRows, 64 * W>(a, b, hk, g, rg * kRows, my_rows, shares, part.parts, reinterpret_cast<uint64_t*>(lds));
}

// ---- many rows: each of the W wavefronts has 16 RT rows of its own and sees all the part's keys, 64 at a time, through the LDS (two stages of K, two
// of V): K and V are read once for up to 16 RT W rows, and no sum crosses wavefronts.  A tile is two steps: V(t) turns its scores into weights
// (vector instructions), M(t) multiplies them with its values and the next tile's keys with Q (the matrix cores).  With eight wavefronts the second four
// run one step behind the first, so that each SIMD has one wavefront in either step; left to themselves the two do the same at the same
// time (256 rows of 128 against 65533 keys, 8 key heads: 118 us, with the turns 101 .. 110).  Without any loads it takes 84 us, with
// nothing but them 69.  Stages that the loads write themselves, four of each, are up to 5 % shorter; but the compiler has every transposing read wait for
// such loads, so they would have to be outstanding behind its back.
//   tile t's keys are read in M(t - 1), its values in M(t): steps 2 t - 1 and 2 t + 1 of the first four, one later of the others.  What a wavefront
//   loaded of K it stores in V(t) for tile t + 1 (the others: t + 2), of V for tile t (t + 1): behind the last reads of the tile that had the
//   stage before, and a barrier ahead of the first of its own.
template <int DP, int RT, int W>
__global__ void __launch_bounds__(64 * W, DP <= 128 ? 2 : W / 4) attn_tree_rows_kernel(TreeArgs a, TreeGrid grid) {
  constexpr int KS = DP / 32, DT = DP / 16, kTile = 64, kChunks = DP / 8, kRows = 16 * RT * W;
  constexpr int kPieces = (kTile * kChunks + 64 * W - 1) / (64 * W);  // 16-byte pieces of K (and of V) per thread and tile
  constexpr bool kEven = kTile * kChunks % (64 * W) == 0, kTurns = W == 8;
  constexpr int kK = kTile * k_row_bytes(DP), kV = kTile * v_row_bytes(DP);
  __shared__ __attribute__((aligned(16))) char lds_k[2 * kK], lds_v[2 * kV];
  __shared__ int odd_values;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quarter = lane >> 4, i16 = lane & 15;
  const int g = a.heads / a.kv_heads, R = a.Tq * g;
  const int slot = static_cast<int>(blockIdx.x % grid.slots), hk = static_cast<int>(blockIdx.x / grid.slots % a.kv_heads), rg = static_cast<int>(blockIdx.x / grid.slots / a.kv_heads);
  const Part part = find_part(a, grid.batch, kTile, slot, grid.budget, grid.cut, lane);
  if (part.b < 0) return;
  const int b = part.b;
  if (grid.budget > 0 && part.z == 0 && hk == 0 && rg == 0 && tid == 0) {
    grid.dealt[2 * b] = part.parts;
    grid.dealt[2 * b + 1] = part.first;
  }
  const int64_t len = clamp_len(a.lens[b], a.capacity);
  const int cached = static_cast<int>((len + kTile - 1) / kTile), tiles = cached + 1;  // (the tree is one tile, the last)
  const int first = static_cast<int>(static_cast<int64_t>(tiles) * part.z / part.parts), end = static_cast<int>(static_cast<int64_t>(tiles) * (part.z + 1) / part.parts);
  const int up = lane < a.T ? a.parents[static_cast<int64_t>(b) * a.T + lane] : -1;

  // A thread's pieces of a tile: the same rows and channels of every tile.  Whole tiles of the cache follow each other at one distance; channels behind the
  // head's last repeat its last ones and are not stored (K's are cleared once, V's reach no sum that is stored).
  u32x4 kf[kPieces], vf[kPieces];
  unsigned from_at[kPieces];
  const char* cache_k = reinterpret_cast<const char*>(a.Kc + (static_cast<int64_t>(b) * a.kv_heads + hk) * a.capacity * a.d);
  const char* cache_v = reinterpret_cast<const char*>(a.Vc + (static_cast<int64_t>(b) * a.kv_heads + hk) * a.capacity * a.d);
#pragma unroll
  for (int n = 0; n < kPieces; ++n) {
    const int id = n * 64 * W + tid, row = id / kChunks, c = id % kChunks;
    from_at[n] = static_cast<unsigned>(row < kTile ? row : kTile - 1) * 2u * a.d + (c * 8 < a.d ? c : a.d / 8 - 1) * 16;
  }
  auto load = [&](u32x4 (&into)[kPieces], bool values, int at) {
    if (static_cast<int64_t>(at + 1) * kTile <= len) {
      const char* from = (values ? cache_v : cache_k) + static_cast<int64_t>(at) * (kTile * 2 * a.d);
#pragma unroll
      for (int n = 0; n < kPieces; ++n) into[n] = *reinterpret_cast<const u32x4*>(from + from_at[n]);
      return;
    }
    const Keys s = keys_of<kTile>(a, b, hk, len, cached, at);
    const char* from = values ? s.v : s.k;
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
      const int id = n * 64 * W + tid, row = id / kChunks, c = id % kChunks;
      into[n] = *reinterpret_cast<const u32x4*>(from + (static_cast<unsigned>(row < s.valid ? row : s.valid - 1) * s.stride + (c * 8 < a.d ? c : a.d / 8 - 1) * 16));
    }
  };
  auto keep = [&](char* stage, int row_bytes, const u32x4 (&what)[kPieces]) {
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
      const int id = n * 64 * W + tid, row = id / kChunks, c = id % kChunks;
      if (!kEven && row >= kTile) break;
      if (c * 8 < a.d) *reinterpret_cast<u32x4*>(stage + row * row_bytes + c * 16) = what[n];
    }
  };
  auto keep_k = [&](int at) { keep(lds_k + (at & 1) * kK, k_row_bytes(DP), kf); };
  auto keep_v = [&](int at) {
    if (at < cached && static_cast<int64_t>(at + 1) * kTile > len) {  // (the weight of what lies behind the last key is zero, its value has to be as well)
      int valid = static_cast<int>(len - static_cast<int64_t>(at) * kTile);
      asm("" : "+s"(valid));  // (compared here, not once ahead of the loop)
#pragma unroll
      for (int n = 0; n < kPieces; ++n)
        if ((n * 64 * W + tid) / kChunks >= valid) vf[n] = u32x4{0u, 0u, 0u, 0u};
    }
    keep(lds_v + (at & 1) * kV, v_row_bytes(DP), vf);
    if (at >= cached) {
      bool odd = false;
#pragma unroll
      for (int n = 0; n < kPieces; ++n) odd = odd || no_number(vf[n]);
      if (odd) odd_values = 1;
    }
  };
  const int behind = kTurns ? wave / (W / 2) : 0;  // 1: one step behind
  load(kf, false, first);
  load(vf, true, first);
  const int row0 = rg * kRows + wave * 16 * RT;  // the wavefront's first row
  f16x8 q[RT][KS];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + rt * 16 + i16, have = r < R ? r : R - 1;
    const half_t* row = a.Q + ((static_cast<int64_t>(b) * a.Tq + have / g) * a.heads + hk * g + have % g) * a.d;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[rt][ks] = load_query<DP>(row, ks, quarter, a.d, a.sign);
  }
  if (tid == 0) odd_values = 0;
  if (a.d < DP)
    for (int at = tid; at < 2 * kK / 16; at += 64 * W) reinterpret_cast<u32x4*>(lds_k)[at] = u32x4{0u, 0u, 0u, 0u};
  uint64_t sees[RT] = {};
  if (end > cached) see(sees, up, lane, row0, R, g, a.T, a.Tq);
  f32x4 o[RT][DT];
  float top[RT], sum[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    top[rt] = -INFINITY;
    sum[rt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // the LDS is written, and read again, behind this; loads of the next tiles stay on their way
  auto meet = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  meet();
  keep_k(first);
  if (first + 1 < end) load(kf, false, first + 1);
  if (behind) {
    keep_v(first);
    if (first + 1 < end) {
      load(vf, true, first + 1);
      keep_k(first + 1);
      if (first + 2 < end) load(kf, false, first + 2);
    }
  }
  meet();
  const bool has_rows = row0 < R;
  const char* k_at = lds_k + i16 * k_row_bytes(DP) + quarter * 16;
  const char* v_at = lds_v + (4 * quarter + (i16 >> 2)) * v_row_bytes(DP) + (i16 & 3) * 8;
  f32x4 s[RT][4];
  f16x8 p[RT][2];
  // Step M's two halves as one chain: each batch of operands (channel tiles of V^T, a key tile of K) is read ahead of the MFMAs of the batch before it,
  // and waited for behind them; the barriers to the scheduler keep it so.
  constexpr int kBatch = DT % 4 == 0 ? 4 : 2, kBatches = 2 * DT / kBatch;  // channel tiles per batch, batches of both halves
  f16x4 vt[2][kBatch][2];
  f16x8 kt[2][KS];
  auto read_v_batch = [&](int at, int n) {
    const char* from = v_at + (at & 1) * kV + (n / (DT / kBatch)) * 32 * v_row_bytes(DP) + (n % (DT / kBatch)) * kBatch * 32;
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) vt[n & 1][u][h] = read_transposed(from + u * 32 + h * 16 * v_row_bytes(DP));
  };
  auto read_k_tile = [&](int at, int n) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kt[n & 1][ks] = *reinterpret_cast<const f16x8*>(k_at + (at & 1) * kK + n * 16 * k_row_bytes(DP) + ks * 64);
  };
  auto landed = [] {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  auto score = [&](int at) {  // (the first key tile of it is there)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (n < 3) read_k_tile(at, n + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kt[n & 1][ks], q[rt][ks], s[rt][n], 0, 0, 0);
      if (n < 3) landed();
    }
  };
  auto values = [&](int at, bool more) {
    read_v_batch(at, 0);
    landed();
#pragma unroll
    for (int n = 0; n < kBatches; ++n) {
      if (n + 1 < kBatches) read_v_batch(at, n + 1);
      else if (more) read_k_tile(at + 1, 0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int dt = (n % (DT / kBatch)) * kBatch + u;
        const f16x4 lo = vt[n & 1][u][0], hi = vt[n & 1][u][1];
        const f16x8 both = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(both, p[rt][n / (DT / kBatch)], o[rt][dt], 0, 0, 0);
      }
      landed();
    }
  };
  auto weights = [&](bool all, int64_t valid) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      weigh<4, DT>(s[rt], all, valid < 0 ? sees[rt] : first_bits(static_cast<int>(valid)), quarter, a.scale_log2, top[rt], sum[rt], o[rt]);
      p[rt][0] = weights_f16(s[rt][0], s[rt][1]);
      p[rt][1] = weights_f16(s[rt][2], s[rt][3]);
    }
  };
  // step V's part in the staging: what was loaded a tile ago into its stages, the next on its way
  auto pass_on = [&](int at) {
    const int tk = at + 1 + behind, tv = at + behind;
#pragma unroll
    for (int n = 0; n < kPieces; ++n) asm volatile("" : "+v"(kf[n]), "+v"(vf[n]));  // (they are there, whichever way the branches go)
    if (tk < end) keep_k(tk);
    if (tv < end) keep_v(tv);
    if (tk + 1 < end) load(kf, false, tk + 1);
    if (tv + 1 < end) load(vf, true, tv + 1);
  };
  if (has_rows) {
    read_k_tile(first, 0);
    landed();
    score(first);
  }
  if (kTurns && behind) meet();
  int at = first;
  for (; at < end && at < cached; ++at) {
    pass_on(at);
    if (has_rows) weights(len - static_cast<int64_t>(at) * kTile >= kTile, len - static_cast<int64_t>(at) * kTile < kTile ? len - static_cast<int64_t>(at) * kTile : kTile);
    meet();
    if (has_rows) {
      values(at, at + 1 < end);
      if (at + 1 < end) score(at + 1);
    }
    if (kTurns) meet();
  }
  if (at < end) {  // the tree's tile
    pass_on(at);
    if (has_rows) weights(false, -1);
    meet();
    if (has_rows && odd_values != 0) {
      // (no keys are read any more: their stages are free)
      float* room = reinterpret_cast<float*>(lds_k) + wave * 512;
      static_assert(W * 2048 <= 2 * kK, "the wavefronts' weights of 32 keys fit the stages of K");
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        add_key_by_key<DT>(a, b, hk, 0, s[rt][0], s[rt][1], sees[rt], room, lane, o[rt]);
        add_key_by_key<DT>(a, b, hk, 32, s[rt][2], s[rt][3], sees[rt], room, lane, o[rt]);
      }
    } else if (has_rows) {
      values(at, false);
    }
    if (kTurns) meet();
  }
  if (kTurns && !behind) meet();

  const int my_rows = R - rg * kRows < kRows ? R - rg * kRows : kRows, problem = hk * grid.row_groups + rg;
  float* shares = grid.ws + (static_cast<int64_t>(problem) * grid.slots + part.first) * (kRows * (DP + 2));
  float* share = shares + static_cast<int64_t>(part.z) * (kRows * (DP + 2));
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = wave * 16 * RT + rt * 16 + i16;
    sum[rt] = sum_of_row(sum[rt]);
    sum_again<DP, kTile>(a, b, hk, len, cached, first, end, 1, rg * kRows + r, sees[rt], top[rt], sum[rt], lane, o[rt]);
    if (r >= my_rows) continue;
    const float inv = 1.f / sum[rt];
    half_t* row = out_row(a, b, hk, g, rg * kRows + r);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int c = dt * 16 + 4 * quarter;
      if (c >= a.d) continue;
      if (part.parts > 1) *reinterpret_cast<f32x4*>(share + r * DP + c) = o[rt][dt];
      else store_row4(row + c, o[rt][dt], inv);
    }
    if (part.parts > 1 && quarter == 0)
      *(reinterpret_cast<uint64_t*>(share + kRows * DP) + r) = static_cast<uint64_t>(__builtin_bit_cast(unsigned, top[rt])) |
                                                               static_cast<uint64_t>(__builtin_bit_cast(unsigned, sum[rt])) << 32;
  }
}

// The parts of many rows joined: four rows of one problem and sequence per workgroup, a wavefront each, DP / 4 lanes to a part's row
template <int DP>
__global__ void __launch_bounds__(256) attn_tree_join_kernel(TreeArgs a, TreeGrid grid, int rows) {
  constexpr int kLanes = DP / 4, kParts = 64 / kLanes;  // (several parts at a time)
  const int lane = threadIdx.x & 63, g = a.heads / a.kv_heads, R = a.Tq * g;
  const int r = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), hk = blockIdx.y, b = blockIdx.z;
  if (r >= R) return;
  const int parts = grid.dealt[2 * b], share_size = rows * (DP + 2), i = r % rows;
  if (parts == 1) return;
  const float* shares = grid.ws + (static_cast<int64_t>(hk * grid.row_groups + r / rows) * grid.slots + grid.dealt[2 * b + 1]) * share_size;
  const int sub = lane / kLanes, c = 4 * (lane % kLanes);
  const float* from = shares + static_cast<int64_t>(i) * DP + c;
  constexpr int kAtOnce = 8;
  f32x4 some[kAtOnce];
  auto request = [&](int y0) {
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int y = y0 + u * kParts + sub;
      some[u] = *reinterpret_cast<const f32x4*>(from + static_cast<int64_t>(y < parts ? y : parts - 1) * share_size);
    }
  };
  request(0);
  // a lane holds a part's maximum and sum (at most 64 parts)
  uint64_t two = 0xff800000u;
  if (lane < parts) two = *(reinterpret_cast<const uint64_t*>(shares + static_cast<int64_t>(lane) * share_size + rows * DP) + i);
  const float top = __builtin_bit_cast(float, static_cast<unsigned>(two)), w = weight_of(top, wave_max(top), a.scale_log2);
  const float total = wave_sum(w * __builtin_bit_cast(float, static_cast<unsigned>(two >> 32)));
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int y0 = 0; y0 < parts; y0 += kAtOnce * kParts) {
    if (y0 > 0) request(y0);
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int y = y0 + u * kParts + sub;
      if (y0 + u * kParts >= parts) break;
      const float wy = __shfl(w, y & 63);
      if (y < parts) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = fmaf(wy, some[u][j], v[j]);
      }
    }
  }
  const f32x4 own = v;
#pragma unroll
  for (int k = 1; k < kParts; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += __shfl(own[j], (lane % kLanes + k * kLanes) & 63);  // (those of the first lanes, which store)
  if (lane < kLanes && c < a.d) store_row4(out_row(a, b, hk, g, r) + c, v, 1.f / total);
}

// The launch of a kernel for `rows` rows and `threads` threads per workgroup and units of `unit` keys, parts of them as `cut` says: one workgroup
// per CU.  The lengths lie on the device: what is chosen here, and below, is chosen by the capacity (what the kernels cut, by the lengths).  `handed`: what a part's sums cost, in units of time (0: those of few rows are little)
struct TreeShape {
  int rows, threads, unit;
  Cut cut;
  float handed;
};
template <typename Kernel>
int launch_tree(Kernel kernel, const TreeArgs& a, int64_t batch, int DP, const TreeShape& shape, bool counts, hipStream_t s, TreeGrid* grid, std::unique_lock<std::recursive_mutex>* lock) {
  const int64_t groups = ceil_div(static_cast<int64_t>(a.Tq) * (a.heads / a.kv_heads), shape.rows), problems = a.kv_heads * groups;
  int64_t budget = kNumCU / problems;
  Cut cut = shape.cut;
  cut.spread = sqrtf(shape.handed * static_cast<float>(problems));
  if (shape.handed == 0.f && problems * batch < 16) cut.whole = 0;  // (few workgroups, each slower than its hand-over)
  const int64_t units = ceil_div(a.capacity, shape.unit) + ceil_div(a.T, shape.unit), useful = static_cast<float>(units) <= static_cast<float>(cut.whole) + 2.f * cut.spread * sqrtf(static_cast<float>(units + batch - 1)) ? 0 : batch * ceil_div(units, cut.least), limit = batch * cut.most;
  budget = budget > useful ? useful : budget;
  budget = budget > limit ? limit : budget;
  // Every sequence in one piece: no workgroup is left for a second one.  (Also where one is far longer than the others: 8 sequences on 32 key heads of 128, one after 32000 keys
  // and seven after 100, take 398 us, the long one alone 91.)
  if (budget <= batch) budget = 0;
  const int64_t slots = budget == 0 ? batch : budget;
  if (batch > INT32_MAX || problems * slots > INT32_MAX) return fail("attn_tree: the launch has too many workgroups");
  *grid = TreeGrid{static_cast<int>(batch), static_cast<int>(slots), static_cast<int>(budget), static_cast<int>(groups), cut, nullptr, nullptr, nullptr};
  const size_t sums = static_cast<size_t>(problems * slots) * shape.rows * (DP + 2);
  if (budget > 0 && split_scratch(s, (sums + 2 * static_cast<size_t>(batch)) * sizeof(float), counts ? static_cast<size_t>(problems * batch) : 1, static_cast<int>(budget), &grid->ws,
                                  &grid->arrivals, lock) != 0)
    return -1;
  if (budget > 0) grid->dealt = reinterpret_cast<int*>(grid->ws + sums);
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(problems * slots)), dim3(shape.threads), 0, s, a, *grid);
  return check_launch("attn_tree");
}
template <int DP, int RT, int W>
int launch_few(const TreeArgs& a, int64_t batch, hipStream_t s) {
  // Parts of W / 2 blocks at least, W of 32 rows (1 node, 32 heads on 8, after 500 keys 9.1 -> 8.3 us; 26 rows after 1000 would take 13.7 instead of 12.9), and none
  // where a wavefront has two or three blocks of the whole (16 nodes, 32 heads of 80, after 500 9.1 -> 7.5; 2 x 8 nodes, 32 heads on 8, after 600 15.6 -> 14.0).
  TreeGrid grid;
  std::unique_lock<std::recursive_mutex> lock;
  return launch_tree(attn_tree_kernel<DP, RT, W>, a, batch, DP, TreeShape{16 * RT, 64 * W, 32, Cut{RT == 1 ? W / 2 : W, 64 / RT, 5 * W / 2, 0.f}, 0.f}, true, s, &grid, &lock);
}
// us that a workgroup of `rows` rows takes for a tile of 64 keys
inline float tile_us(int rows, int DP) { return 0.6f + static_cast<float>(rows * DP) / 16384.f; }
// us of all tiles with `rows` rows per workgroup and full caches: one piece per sequence, or one workgroup per CU, whose sums are handed over (see launch_rows)
inline float blocks_us(const TreeArgs& a, int64_t batch, int rows, int DP) {
  const int64_t all = static_cast<int64_t>(a.Tq) * (a.heads / a.kv_heads), problems = a.kv_heads * ceil_div(all, rows);
  const float units = static_cast<float>(ceil_div(a.capacity, 64) + 1), tile = tile_us(rows, DP), whole = static_cast<float>(batch * problems) / kNumCU;
  const float uncut = (whole > 1.f ? whole : 1.f) * units * tile;
  if (kNumCU / problems <= batch) return uncut;
  const float share = units * whole > 2.f ? units * whole : 2.f, parts = static_cast<float>(batch * problems) * units / share;
  const float cut = share * tile + 4.f + parts * static_cast<float>(all < rows ? all : rows) * (DP + 2) * 8 / 4e6f;
  return cut < uncut ? cut : uncut;
}
template <int DP, int RT, int W>
int launch_rows(const TreeArgs& a, int64_t batch, hipStream_t s) {
  TreeGrid grid;
  std::unique_lock<std::recursive_mutex> lock;  // (held until the kernel that joins the parts is enqueued as well)
  // Times in us: a tile of 64 keys; the second launch and what it waits for, 4; a part's sums, written and read at 4 TB/s.  8 sequences of 128 rows, 8 key heads,
  // after 250 keys 20.0 -> 17.5.
  const int64_t all = static_cast<int64_t>(a.Tq) * (a.heads / a.kv_heads);
  const float tile = tile_us(16 * RT * W, DP), sums = static_cast<float>(all < 16 * RT * W ? all : 16 * RT * W) * (DP + 2) * 4;
  const TreeShape shape{16 * RT * W, 64 * W, 64, Cut{2, 64, static_cast<int>(4.f / tile), 0.f}, 2.f * sums / (4e6f * tile)};
  if (launch_tree(attn_tree_rows_kernel<DP, RT, W>, a, batch, DP, shape, false, s, &grid, &lock) != 0) return -1;
  if (grid.budget == 0) return 0;
  hipLaunchKernelGGL(attn_tree_join_kernel<DP>, dim3(static_cast<unsigned>(ceil_div(all, 4)), static_cast<unsigned>(a.kv_heads), static_cast<unsigned>(batch)),
                     dim3(256), 0, s, a, grid, shape.rows);
  return check_launch("attn_tree");
}

template <int DP>
int launch_tree_rows(const TreeArgs& a, int64_t batch, hipStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.Tq) * (a.heads / a.kv_heads);
  // Beyond 16 rows, or 8 of heads of more than 128, sharing the keys pays only where they are few: 32 rows of 64 heads on 8 after 300 keys 8.1 us, sharing the rows 10.3,
  // 20 rows of 32 on 8 after 500 12.8 / 11.6, 32 rows after 1000 16.7 / 13.2, after 16000 29.5 / 20.2; 16 rows of 256 after 1569 19.2 / 15.5.  16 rows of 80
  // after 3001 12.6 / 15.6, one row of 256 on 8 heads after 4000 16.5 / 21.6.
  // (heads of 64, two sequences; 32 rows of 128 on 8 heads after 300 keys of one sequence take 14.7 sharing the keys and 11.3 sharing the rows)
  const bool few = a.capacity <= 384;
  if (rows <= (DP <= 128 ? 16 : 8) || (rows <= 16 && few)) return launch_few<DP, 1, (DP <= 128 ? 8 : 4)>(a, batch, s);
  if (rows <= 32 && few) return launch_few<DP, 2, (DP <= 128 ? 8 : 4)>(a, batch, s);
  // Blocks of 64, 128 or 256 rows: larger ones read K and V less often, smaller ones hand fewer sums over.  256 rows on 8 heads of 128 after 1000 / 4000 / 16000 / 65533
  // keys: 15.0, 21.7, 48.3, 163 us in blocks of 64, 19.1, 23.2, 37.8, 118 of 128, 23.7, 27.8, 39.2, 102 of 256.  (The caches full: after 1000 keys in a cache of 32768 rows blocks of
  // 256 are taken, and 24.1 us.)
  if (rows <= 64) return launch_rows<DP, 1, 4>(a, batch, s);
  const float by64 = blocks_us(a, batch, 64, DP), by128 = blocks_us(a, batch, 128, DP);
  if constexpr (DP <= 128) {
    const float by256 = rows > 128 ? blocks_us(a, batch, 256, DP) : INFINITY;
    if (by256 < by64 && by256 < by128) return launch_rows<DP, 2, 8>(a, batch, s);
  }
  return by64 < by128 ? launch_rows<DP, 1, 4>(a, batch, s) : launch_rows<DP, 1, 8>(a, batch, s);
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
  if (!(scale >= -2.0e38f && scale <= 2.0e38f)) return fail("attn_tree: the scale is not a finite number up to 2e38");
  if (!Q || !K || !V || !lens || !parents || !out || (capacity > 0 && (!K_cache || !V_cache))) return fail("attn_tree: NULL buffer");
  const int64_t out_bytes = batch * rows * heads * d * 2, new_bytes = batch * nodes * kv_heads * d * 2, cache_bytes = batch * kv_heads * capacity * d * 2;
  if (overlaps(out, out_bytes, Q, out_bytes) || overlaps(out, out_bytes, K, new_bytes) || overlaps(out, out_bytes, V, new_bytes) ||
      overlaps(out, out_bytes, K_cache, cache_bytes) || overlaps(out, out_bytes, V_cache, cache_bytes) || overlaps(out, out_bytes, lens, batch * 4) ||
      overlaps(out, out_bytes, parents, batch * nodes * 4))
    return fail("attn_tree: output overlaps an input");
  TreeArgs a{static_cast<const half_t*>(Q), static_cast<const half_t*>(K), static_cast<const half_t*>(V), static_cast<const half_t*>(K_cache),
             static_cast<const half_t*>(V_cache), static_cast<const int*>(lens), static_cast<const int*>(parents), static_cast<half_t*>(out),
             static_cast<int>(nodes), static_cast<int>(rows), static_cast<int>(heads), static_cast<int>(kv_heads), static_cast<int>(d), capacity,
             scale == 0.f ? 1.f : fabsf(scale) * 1.4426950408889634f, static_cast<half_t>(scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f)};
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
