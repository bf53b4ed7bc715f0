// Attention of one new token per sequence over keys and values in pages, for gfx950.
//
//   row (b, h): query head h of sequence b, which shares key head h / (heads / kv_heads), sees the positions j < lens[b];
//   position j lies in page table[b][j / page], row j % page
//   out[b, h, :] = sum_j softmax_j(scale * Q[b, h, :] . k_j) v_j                         fp32 scores, statistics and sums
//
// Positions in pages outside [0, pages) are not seen; a row that sees nothing is zeros.
#include "attn_rows.h"

namespace dtas {
namespace {

struct PagedArgs {
  const half_t *Q, *K, *V;
  const int *table, *lens;
  half_t* out;
  int heads, kv_heads, d, pages;
  unsigned page, room;  // positions that a table holds at most
  int64_t columns;
  float scale_log2;  // |scale| * log2(e): the softmax is taken in powers of two
  half_t sign;       // the scale's: 1, -1, or 0 (scale_log2 is 1 then)
};

// positions of a sequence (its table holds no more)
__device__ __forceinline__ unsigned length_of(const PagedArgs& a, int64_t b) {
  const int len = a.lens[b];
  return len < 0 ? 0u : static_cast<unsigned>(len) > a.room ? a.room : static_cast<unsigned>(len);
}

// any head dimension up to 256, any page and any alignment: one wavefront per row, one pass with the running maximum and sum
__global__ void __launch_bounds__(64) attn_paged_scalar_kernel(PagedArgs a, int64_t rows) {
  const int lane = threadIdx.x;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int h = static_cast<int>(r % a.heads), hk = h / (a.heads / a.kv_heads);
    const int64_t b = r / a.heads;
    const half_t* q = a.Q + r * a.d;
    float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) qv[i] = lane + 64 * i < a.d ? static_cast<float>(q[lane + 64 * i]) : 0.f;
    float top = -INFINITY, sum = 0.f;
    bool any = false;
    const unsigned len = length_of(a, b);
    for (unsigned j0 = 0, c = 0; j0 < len; j0 += a.page, ++c) {
      const int p = a.table[b * a.columns + c];
      if (p < 0 || p >= a.pages) continue;
      any = true;
      const unsigned some = len - j0 < a.page ? len - j0 : a.page;
      const int64_t at = (static_cast<int64_t>(p) * a.kv_heads + hk) * a.page * a.d;
      const half_t *k = a.K + at, *v = a.V + at;
      for (unsigned j = 0; j < some; ++j, k += a.d, v += a.d) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (lane + 64 * i < a.d) s = fmaf(qv[i], static_cast<float>(k[lane + 64 * i]), s);
        s = wave_sum(s) * static_cast<float>(a.sign);  // (the maximum is that of the products: their differences are scaled, no product overflows by the scale)
        const float next = fmaxf(top, s);
        const float keep = next == -INFINITY ? 1.f : exp2f((top - next) * a.scale_log2), w = s == -INFINITY ? 0.f : exp2f((s - next) * a.scale_log2);  // (a score that is no number has no weight that is one)
        top = next;
        sum = fmaf(sum, keep, w);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (lane + 64 * i < a.d) o[i] = fmaf(o[i], keep, w * static_cast<float>(v[lane + 64 * i]));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < a.d) a.out[r * a.d + lane + 64 * i] = any ? static_cast<half_t>(o[i] / sum) : half_t{0};
  }
}

// ---- head dimensions that are multiples of 8, pages of a multiple of 16, data on 16-byte boundaries: the matrix cores -----------------------
// The query heads that share a key head, of all sequences of a group, form one problem of R rows: S^T = K Q^T and O^T = V^T P^T, 16 keys or channels by 16 rows to an
// instruction, as the tree's attention has them (attn_rows.h).  A wavefront takes a visit at a time: two halves of 16 keys, each from one page, so that
// all its addresses are a scalar and a lane's constant.  K comes as the matrix cores take it, straight from memory; V passes through a piece of the LDS that is the
// wavefront's own and is read from there transposed.  The next visit's K and V are on their way in registers, and the table's entries a block further ahead.
// In a group a block is visited once for every page that its sequences name there; rows that do not name it have their scores masked.
// Sequences are cut into parts by their lengths, on the device: see find_part.
struct PagedGrid {
  int problems, slots, beams, sub, subs;  // a problem: `sub` sequences at most of a group of `beams`, `subs` of which make up the group
  int row_groups, extra, least, most;     // extra: parts that all problems together may have beyond one each (0: nothing is cut)
  float whole;
  float* ws;
  unsigned* arrivals;
};
struct Part {
  int p, z, parts, first;  // problem, which of its parts, of how many, where the first one's sums lie; p < 0: nothing to do
};
__device__ __forceinline__ int first_sequence(const PagedGrid& grid, int p, int* count) {
  const int group = p / grid.subs, s = p - group * grid.subs, left = grid.beams - s * grid.sub;
  *count = left < grid.sub ? left : grid.sub;
  return group * grid.beams + s * grid.sub;
}
// blocks of 32 keys of a problem: those of its longest sequence
__device__ __forceinline__ int blocks_of(const PagedArgs& a, const PagedGrid& grid, int p) {
  int count;
  const int b = first_sequence(grid, p, &count);
  unsigned longest = 0;
  for (int i = 0; i < count; ++i) {
    const unsigned len = length_of(a, b + i);
    longest = longest > len ? longest : len;
  }
  return static_cast<int>((longest + 31) / 32);
}
// Parts of at most `per` blocks: a workgroup's even share of all blocks, `least` at least, and no more than `most` parts of one problem; nothing is cut where the longest problem is
// not much more than that.  Every problem has a part; all have problems + blocks / per <= problems + extra.
__device__ __forceinline__ int blocks_per_part(const PagedGrid& grid, float total, int longest) {
  const float even = total * 1.0001f / static_cast<float>(grid.extra);
  if (static_cast<float>(longest) <= grid.whole * even + static_cast<float>(grid.least)) return longest > 0 ? longest : 1;
  int per = static_cast<int>(even) + 1;
  per = per > grid.least ? per : grid.least;
  const int few = (longest + grid.most - 1) / grid.most;
  return per > few ? per : few;
}
__device__ __forceinline__ int parts_of(int blocks, int per) { return blocks > per ? (blocks + per - 1) / per : 1; }
__device__ __forceinline__ Part found_at(int slot, int p0, int parts, int upto, int cut_upto, int lane_base, int cut_base) {
  const uint64_t here = __builtin_amdgcn_ballot_w64(slot >= lane_base + upto - parts && slot < lane_base + upto);
  if (here == 0) return Part{-1, 0, 0, 0};
  const int l = __builtin_ctzll(here), n = __builtin_amdgcn_readlane(parts, l);
  return Part{p0 + l, slot - (lane_base + __builtin_amdgcn_readlane(upto, l) - n), n, cut_base + __builtin_amdgcn_readlane(cut_upto, l) - n};
}
template <int W>
__device__ __forceinline__ Part find_part(const PagedArgs& a, const PagedGrid& grid, int slot, int lane, int wave) {
  if (grid.extra == 0) return Part{slot, 0, 1, 0};
  if (grid.problems <= 64) {
    const int blocks = lane < grid.problems ? blocks_of(a, grid, lane) : 0;
    const int per = blocks_per_part(grid, wave_sum(static_cast<float>(blocks)), wave_most(blocks));
    const int parts = lane < grid.problems ? parts_of(blocks, per) : 0;
    return found_at(slot, 0, parts, sum_upto(parts), sum_upto(parts > 1 ? parts : 0), 0, 0);
  }
  // the wavefronts have a range of the problems each
  __shared__ float totals[W];
  __shared__ int longest[W], counts[W], cuts[W];
  __shared__ Part found;
  const int range = (grid.problems + 64 * W - 1) / (64 * W) * 64, from = wave * range, to = from + range < grid.problems ? from + range : grid.problems;
  float total = 0.f;
  int most = 0;
  for (int c = from; c < to; c += 64) {
    const int blocks = c + lane < to ? blocks_of(a, grid, c + lane) : 0, top = wave_most(blocks);
    total += wave_sum(static_cast<float>(blocks));
    most = most > top ? most : top;
  }
  if (lane == 0) {
    totals[wave] = total;
    longest[wave] = most;
  }
  if (threadIdx.x == 0) found.p = -1;
  __syncthreads();
  total = 0.f;
  most = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    total += totals[w];
    most = most > longest[w] ? most : longest[w];
  }
  const int per = blocks_per_part(grid, total, most);
  int count = 0, cut = 0;
  for (int c = from; c < to; c += 64) {
    const int parts = c + lane < to ? parts_of(blocks_of(a, grid, c + lane), per) : 0;
    count += wave_total(parts);
    cut += wave_total(parts > 1 ? parts : 0);
  }
  if (lane == 0) {
    counts[wave] = count;
    cuts[wave] = cut;
  }
  __syncthreads();
  int base = 0, cut_base = 0;
#pragma unroll
  for (int w = 0; w < W; ++w)
    if (w < wave) {
      base += counts[w];
      cut_base += cuts[w];
    }
  if (slot >= base && slot < base + count) {
    for (int c = from; c < to; c += 64) {
      const int parts = c + lane < to ? parts_of(blocks_of(a, grid, c + lane), per) : 0, upto = sum_upto(parts), cut_upto = sum_upto(parts > 1 ? parts : 0);
      const Part part = found_at(slot, c, parts, upto, cut_upto, base, cut_base);
      if (part.p >= 0) {
        if (lane == 0) found = part;
        break;
      }
      base += __builtin_amdgcn_readlane(upto, 63);
      cut_base += __builtin_amdgcn_readlane(cut_upto, 63);
    }
  }
  __syncthreads();
  const Part part = found;
  return Part{__builtin_amdgcn_readfirstlane(part.p), __builtin_amdgcn_readfirstlane(part.z), __builtin_amdgcn_readfirstlane(part.parts),
              __builtin_amdgcn_readfirstlane(part.first)};
}

// two halves of 16 keys at positions pos and pos + 16, where their K and V lie, and which sequences of the problem (bits) see them
struct Visit {
  const char *k[2], *v[2];
  unsigned pos, seen[2];
};
__device__ __forceinline__ unsigned bits_below(int n) { return n <= 0 ? 0u : n >= 16 ? 0xffffu : (1u << n) - 1u; }
// over the sixteen rows of the lanes
__device__ __forceinline__ unsigned any_row(unsigned v) {
  v |= __builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xB1, 0xf, 0xf, true);   // quad_perm xor 1, xor 2, row_half_mirror, row_mirror
  v |= __builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4E, 0xf, 0xf, true);
  v |= __builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x141, 0xf, 0xf, true);
  v |= __builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x140, 0xf, 0xf, true);
  return static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(v), 0));
}

// A value may be infinite where its weight is too small for fp16 (below 2^-36 of the largest): zero times infinity, though the weight is a number in fp32 and the channel
// infinite.  Such a channel shows in O, as NaN where the sum of the weights is a number (rare).  What it is instead depends on the keys alone whose values are no
// numbers: they are looked for in the wavefront's blocks first, first + step .., and summed with their weights in fp32.  The four lanes of a row hold a quarter of
// its channels each, and follow their own row's table.
template <int DP, int KS, int DT>
__device__ __forceinline__ void sum_again(const PagedArgs& a, const int* names, int beam, int hk, unsigned len, unsigned longest, unsigned first, unsigned step,
                                          const f16x8 (&q)[KS], float top, float sum, int lane, f32x4 (&o)[DT]) {
  f32x4 all = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (dt * 16 + 16 <= below(DP) || dt * 16 + 4 * (lane >> 4) < a.d) all[j] += o[dt][j];
  const float some = (all[0] + all[1]) + (all[2] + all[3]);
  const bool mine = some != some && sum == sum;
  if (__builtin_amdgcn_ballot_w64(mine) == 0) return;
  asm volatile("" : "+v"(lane), "+v"(beam));  // (nothing of what follows is computed ahead)
  const int quarter = lane >> 4;
  f32x4 fresh[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) fresh[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (unsigned at = first; at < (longest + 31) / 32; at += step)
    for (unsigned pos = at * 32; pos < at * 32 + 32 && pos < longest; ++pos) {
      const unsigned column = pos / a.page;
      const int page = pos < len ? names[static_cast<int64_t>(beam) * a.columns + column] : -1;
      const bool shown = static_cast<unsigned>(page) < static_cast<unsigned>(a.pages);
      const int64_t from = ((static_cast<int64_t>(shown ? page : 0) * a.kv_heads + hk) * a.page + (pos - column * a.page)) * a.d;
      const half_t *k = a.K + from, *v = a.V + from;
      bool odd = false;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        if (dt * 16 + 4 * quarter < a.d) {
          const f16x4 four = *reinterpret_cast<const f16x4*>(v + dt * 16 + 4 * quarter);
#pragma unroll
          for (int j = 0; j < 4; ++j) odd = odd || !(fabsf(static_cast<float>(four[j])) < INFINITY);
        }
      if (__builtin_amdgcn_ballot_w64(odd && shown) == 0) continue;
      float t = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const f16x8 some_k = load_channels<DP>(reinterpret_cast<const char*>(k), ks, quarter, a.d);
#pragma unroll
        for (int e = 0; e < 8; ++e) t = fmaf(static_cast<float>(some_k[e]), static_cast<float>(q[ks][e]), t);
      }
      t = sum_of_row(t);
      const float weight = t == -INFINITY ? 0.f : exp2_fast(fmaf(t - top, a.scale_log2, kRoom));
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        if (dt * 16 + 4 * quarter < a.d) {
          const f16x4 four = *reinterpret_cast<const f16x4*>(v + dt * 16 + 4 * quarter);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float value = static_cast<float>(four[j]);
            if (shown && !(fabsf(value) < INFINITY)) fresh[dt][j] = fmaf(weight, value, fresh[dt][j]);
          }
        }
    }
  if (mine) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[dt][j] = o[dt][j] != o[dt][j] ? fresh[dt][j] : o[dt][j];
  }
}

template <int DP, int RT, int W, bool GROUP>
__global__ void __launch_bounds__(64 * W) attn_paged_kernel(PagedArgs a, PagedGrid grid) {
  constexpr int KS = DP / 32, DT = DP / 16, VL = DP / 16, VH = VL / 2;  // k steps, channel tiles, 16-byte pieces of V per lane, of a half
  constexpr int kRows = 16 * RT, kChunks = DP / 8, kWave = 32 * v_row_bytes(DP), kShare = kRows * (DP + 2);
  __shared__ __attribute__((aligned(16))) char lds[W * kWave];
  __shared__ float stat_m[W][kRows], stat_l[W][kRows];
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quarter = lane >> 4, i16 = lane & 15;
  const int g = a.heads / a.kv_heads;
  const int slot = static_cast<int>(blockIdx.x % grid.slots), hk = static_cast<int>(blockIdx.x / grid.slots % a.kv_heads), rg = static_cast<int>(blockIdx.x / grid.slots / a.kv_heads);
  const Part part = find_part<W>(a, grid, slot, lane, wave);
  if (part.p < 0) return;
  int nb = 1;
  const int b0 = GROUP ? first_sequence(grid, part.p, &nb) : part.p, R = nb * g;
  const unsigned row_bytes = 2u * a.d;
  const int64_t head_bytes = static_cast<int64_t>(a.page) * row_bytes, page_bytes = head_bytes * a.kv_heads;
  const char *Kh = reinterpret_cast<const char*>(a.K) + hk * head_bytes, *Vh = reinterpret_cast<const char*>(a.V) + hk * head_bytes;

  // ---- the rows
  f16x8 q[RT][KS];
  unsigned row_len[RT];
  int beam[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = rg * kRows + rt * 16 + i16, have = r < R ? r : R - 1;
    beam[rt] = GROUP ? have / g : 0;
    const half_t* row = a.Q + (static_cast<int64_t>(b0 + beam[rt]) * a.heads + hk * g + (have - beam[rt] * g)) * a.d;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[rt][ks] = load_query<DP>(row, ks, quarter, a.d, a.sign);
    row_len[rt] = length_of(a, b0 + beam[rt]);
  }
  // lengths of the sequences (GROUP: lane i & 31 holds sequence i's), the longest and the shortest
  const unsigned my_len = GROUP ? ((lane & 31) < nb ? length_of(a, b0 + (lane & 31)) : 0u) : length_of(a, b0);
  const unsigned longest = GROUP ? static_cast<unsigned>(wave_most(static_cast<int>(my_len))) : static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(my_len)));
  const unsigned shortest = GROUP ? 0x7fffffffu - static_cast<unsigned>(wave_most((lane & 31) < nb ? static_cast<int>(0x7fffffffu - my_len) : 0)) : longest;
  const unsigned blocks = (longest + 31) / 32, stride = static_cast<unsigned>(part.parts) * W;
  const unsigned everyone = nb >= 32 ? ~0u : (1u << nb) - 1u;

  // ---- where the next visit is
  const int* names = a.table + static_cast<int64_t>(b0) * a.columns;
  auto place = [&](int page, unsigned in_page, const char*& k, const char*& v) {
    const int64_t at = page * page_bytes + static_cast<int64_t>(in_page) * row_bytes;
    k = Kh + at;
    v = Vh + at;
  };
  unsigned blk = static_cast<unsigned>(wave) * part.parts + part.z;  // the block whose entries come next
  // GROUP: a block's entries, lane (half, sequence); else those of 32 of the wavefront's blocks, lane (block, half)
  auto gather = [&](unsigned at, int& entry, unsigned& in_page) {
    const unsigned pos = GROUP ? at * 32 + (lane >> 5) * 16 : (at + (lane >> 1) * stride) * 32 + (lane & 1) * 16;
    const unsigned column = pos / a.page;
    in_page = pos - column * a.page;
    entry = pos < my_len && (!GROUP || (lane & 31) < nb) ? names[(GROUP ? static_cast<int64_t>(lane & 31) * a.columns : 0) + column] : -1;
  };
  int entry, entry_next;
  unsigned in_page, in_page_next, left[2] = {0, 0}, pos_now = 0;
  int taken = 0;  // (of the 32 blocks)
  gather(blk, entry, in_page);
  gather(blk + (GROUP ? stride : 32 * stride), entry_next, in_page_next);
  auto advance = [&](Visit& to) -> bool {
    if constexpr (GROUP) {
      while ((left[0] | left[1]) == 0) {
        if (blk >= blocks) return false;
        if (taken != 0) {  // (the first block's entries are there)
          entry = entry_next;
          in_page = in_page_next;
          gather(blk + stride, entry_next, in_page_next);
        }
        taken = 1;
        pos_now = blk * 32;
        blk += stride;
        const uint64_t some = __builtin_amdgcn_ballot_w64(static_cast<unsigned>(entry) < static_cast<unsigned>(a.pages));
        left[0] = static_cast<unsigned>(some);
        left[1] = static_cast<unsigned>(some >> 32);
      }
      to.pos = pos_now;
      int page[2] = {0, 0};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        to.seen[h] = 0;
        if (left[h] != 0) {
          page[h] = __builtin_amdgcn_readlane(entry, __builtin_ctz(left[h]) + 32 * h);
          to.seen[h] = static_cast<unsigned>(__builtin_amdgcn_ballot_w64(entry == page[h]) >> (32 * h)) & left[h];
          left[h] &= ~to.seen[h];
        }
      }
      // (a half that nobody sees here is read from the other's page)
      if (to.seen[0] == 0) page[0] = page[1];
      if (to.seen[1] == 0) page[1] = page[0];
#pragma unroll
      for (int h = 0; h < 2; ++h) place(page[h], static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(in_page), 32 * h)), to.k[h], to.v[h]);
    } else {
      if (blk >= blocks) return false;
      if (taken == 32) {
        entry = entry_next;
        in_page = in_page_next;
        gather(blk + 32 * stride, entry_next, in_page_next);
        taken = 0;
      }
      to.pos = blk * 32;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int page = __builtin_amdgcn_readlane(entry, 2 * taken + h);
        const bool there = static_cast<unsigned>(page) < static_cast<unsigned>(a.pages);
        to.seen[h] = there ? 1u : 0u;
        place(there ? page : 0, static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(in_page), 2 * taken + h)), to.k[h], to.v[h]);
      }
      ++taken;
      blk += stride;
    }
    return true;
  };

  // ---- a lane's pieces of K and V
  f16x8 kf[2][KS];
  u32x4 vf[VL];
  unsigned k_at[KS], v_at[VH];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int at = ks * 32 + quarter * 8;
    k_at[ks] = i16 * row_bytes + 2u * (at < a.d ? at : a.d - 8);
  }
#pragma unroll
  for (int n = 0; n < VH; ++n) {
    const int id = n * 64 + lane, c = id % kChunks;
    v_at[n] = id / kChunks * row_bytes + 16u * (c * 8 < a.d ? c : a.d / 8 - 1);
  }
  auto load_k = [&](const Visit& from) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kf[kt][ks] = *reinterpret_cast<const f16x8*>(from.k[kt] + k_at[ks]);
  };
  auto load_v = [&](const Visit& from) {
#pragma unroll
    for (int n = 0; n < VL; ++n) vf[n] = *reinterpret_cast<const u32x4*>(from.v[n / VH] + v_at[n % VH]);
  };

  f32x4 o[RT][DT];
  float top[RT], sum[RT];
  bool saw[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    top[rt] = -INFINITY;
    sum[rt] = 0.f;
    saw[rt] = false;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  char* mine = lds + wave * kWave;
  const unsigned tr_at = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)mine)) +
                         (4 * quarter + (i16 >> 2)) * v_row_bytes(DP) + (i16 & 3) * 8;

  auto visit = [&](const Visit& here, bool more, const Visit& next) {
    f32x4 s[RT][2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        if (ks * 32 + 32 > below(DP) && ks * 32 + quarter * 8 >= a.d) kf[kt][ks] = f16x8{};
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        s[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s[rt][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[kt][ks], q[rt][ks], s[rt][kt], 0, 0, 0);
      }
    if (more) load_k(next);
    const bool all = here.seen[0] == everyone && here.seen[1] == everyone && here.pos + 32 <= shortest;
    unsigned shown[RT];
    bool odd = false;
    if (!all) {
      unsigned any = 0;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int have = static_cast<int>(row_len[rt]) - static_cast<int>(here.pos);
        shown[rt] = ((here.seen[0] >> beam[rt]) & 1 ? bits_below(have) : 0u) | ((here.seen[1] >> beam[rt]) & 1 ? bits_below(have - 16) : 0u) << 16;
        saw[rt] = saw[rt] || shown[rt] != 0;
        any |= shown[rt];
      }
      any = any_row(any);
      // values that nobody sees would meet weights of zero, and may be no numbers
#pragma unroll
      for (int n = 0; n < VL; ++n)
        if (!((any >> ((n * 64 + lane) / kChunks)) & 1)) vf[n] = u32x4{0u, 0u, 0u, 0u};
      if constexpr (GROUP) {  // nor must those that only some rows see
#pragma unroll
        for (int n = 0; n < VL; ++n) odd = odd || no_number(vf[n]);
        odd = __builtin_amdgcn_ballot_w64(odd) != 0;
      }
    } else {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        shown[rt] = ~0u;
        saw[rt] = true;
      }
    }
    if (!GROUP || !odd) {
#pragma unroll
      for (int n = 0; n < VL; ++n) {
        const int id = n * 64 + lane, row = id / kChunks, c = id % kChunks;
        *reinterpret_cast<u32x4*>(mine + row * v_row_bytes(DP) + c * 16) = vf[n];
      }
    }
    if (more) load_v(next);
    f16x8 p[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      weigh<2, DT>(s[rt], all, shown[rt], quarter, a.scale_log2, top[rt], sum[rt], o[rt]);
      p[rt] = weights_f16(s[rt][0], s[rt][1]);
      if (GROUP && odd) {  // (rare) key by key, a row adding up what it sees
        float* room = reinterpret_cast<float*>(mine);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          room[(4 * quarter + j) * 16 + i16] = s[rt][0][j];
          room[(16 + 4 * quarter + j) * 16 + i16] = s[rt][1][j];
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        for (int key = 0; key < 32; ++key) {
          const float weight = room[key * 16 + i16];
          const half_t* v = reinterpret_cast<const half_t*>((key < 16 ? here.v[0] : here.v[1]) + (key & 15) * row_bytes);
          if ((shown[rt] >> key) & 1) {
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
    if (GROUP && odd) return;
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
  Visit here{}, next{};
  bool more = advance(here);
  if (more) {
    load_k(here);
    load_v(here);
  }
  while (more) {
    more = advance(next);
    visit(here, more, next);
    here = next;
  }

  // ---- the wavefronts' shares, joined in their order.  A row that saw nothing says so by a sum of -1 (its weight is zero where another's is not)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    sum[rt] = sum_of_row(sum[rt]);
    sum_again<DP>(a, names, beam[rt], hk, row_len[rt], longest, static_cast<unsigned>(wave) * part.parts + part.z, stride, q[rt], top[rt], sum[rt], lane, o[rt]);
    if (quarter == 0) {
      stat_m[wave][rt * 16 + i16] = top[rt];
      stat_l[wave][rt * 16 + i16] = saw[rt] ? sum[rt] : -1.f;
    }
  }
  __syncthreads();
  auto best_of = [&](int r) {
    float best = stat_m[0][r];
#pragma unroll
    for (int w = 1; w < W; ++w) best = fmaxf(best, stat_m[w][r]);
    return best;
  };
  const int my_rows = R - rg * kRows < kRows ? R - rg * kRows : kRows;
  const int64_t problem = static_cast<int64_t>(hk) * grid.row_groups + rg;
  float* shares = grid.ws + (problem * 2 * grid.extra + part.first) * kShare;
  float* share = shares + static_cast<int64_t>(part.z) * kShare;
  auto out_row = [&](int r) {  // (of this workgroup's)
    const int at = rg * kRows + r, beam_of = GROUP ? at / g : 0;
    return a.out + (static_cast<int64_t>(b0 + beam_of) * a.heads + hk * g + (at - beam_of * g)) * a.d;
  };
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
      bool any = false;
      const float best = best_of(r);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const f32x4 some = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + w * kWave) + i * kPitch + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += some[j];
        l += stat_l[w][r] * weight_of(stat_m[w][r], best, a.scale_log2);
        any = any || !(stat_l[w][r] < 0.f);
      }
      if (part.parts > 1) {
        store_out(v, reinterpret_cast<f32x4*>(share + r * DP + c), true);
        if (c == 0) store_stat(share, kRows, DP, r, best, any ? l : -1.f);
      } else {
        store_row4(out_row(r) + c, v, any ? 1.f / l : 0.f);
      }
    }
    __syncthreads();
  }
  if (part.parts == 1 || !last_to_arrive(grid.arrivals + problem * grid.problems + part.p, part.parts, &flag)) return;

  // ---- whoever is last joins the parts in their order
  static_assert(128 / RT * kRows * 8 <= W * kWave, "the parts' statistics fit the LDS");
  uint64_t* stats = reinterpret_cast<uint64_t*>(lds);
  constexpr int kAtOnce = 8;  // parts requested before the first is used: a trip to memory per eight
  uint64_t one[kAtOnce], other[kAtOnce];
  auto request = [&](int at, int y0) {
    const int i = at / (DP / 4), c = 4 * (at % (DP / 4));
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int y = y0 + u < part.parts ? y0 + u : part.parts - 1;
      const uint64_t* from = reinterpret_cast<const uint64_t*>(shares + static_cast<int64_t>(y) * kShare + i * DP + c);
      one[u] = __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      other[u] = __hip_atomic_load(from + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  };
  const int last = my_rows * (DP / 4);
  if (tid < last) request(tid, 0);  // (on their way while the statistics come)
  for (int at = tid; at < part.parts * kRows; at += 64 * W)
    if (at % kRows < my_rows)
      stats[at] = __hip_atomic_load(reinterpret_cast<const uint64_t*>(shares + static_cast<int64_t>(at / kRows) * kShare + kRows * DP) + at % kRows, __ATOMIC_RELAXED,
                                    __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  for (int at = tid; at < last; at += 64 * W) {
    const int i = at / (DP / 4), c = 4 * (at % (DP / 4));
    if (at != tid) request(at, 0);
    float best = -INFINITY, l = 0.f;
    bool any = false;
    for (int y = 0; y < part.parts; ++y) best = fmaxf(best, __builtin_bit_cast(float, static_cast<unsigned>(stats[y * kRows + i])));
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int y0 = 0; y0 < part.parts; y0 += kAtOnce) {
      if (y0 > 0) request(at, y0);
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (y0 + u >= part.parts) break;
        const uint64_t two = stats[(y0 + u) * kRows + i];
        const float w = weight_of(__builtin_bit_cast(float, static_cast<unsigned>(two)), best, a.scale_log2), theirs = __builtin_bit_cast(float, static_cast<unsigned>(two >> 32));
        any = any || !(theirs < 0.f);
        l = fmaf(w, theirs, l);
        v[0] = fmaf(w, __builtin_bit_cast(float, static_cast<unsigned>(one[u])), v[0]);
        v[1] = fmaf(w, __builtin_bit_cast(float, static_cast<unsigned>(one[u] >> 32)), v[1]);
        v[2] = fmaf(w, __builtin_bit_cast(float, static_cast<unsigned>(other[u])), v[2]);
        v[3] = fmaf(w, __builtin_bit_cast(float, static_cast<unsigned>(other[u] >> 32)), v[3]);
      }
    }
    if (c < a.d) store_row4(out_row(i) + c, v, any ? 1.f / l : 0.f);
  }
}

template <int DP, int RT, int W, bool GROUP>
int launch_paged(const PagedArgs& a, int64_t batch, int beams, int sub, hipStream_t s) {
  const int64_t g = a.heads / a.kv_heads;
  PagedGrid grid{};
  grid.beams = GROUP ? beams : 1;
  grid.sub = GROUP ? sub : 1;
  grid.subs = static_cast<int>(ceil_div(grid.beams, grid.sub));
  const int64_t problems = batch / grid.beams * grid.subs;
  grid.row_groups = GROUP ? 1 : static_cast<int>(ceil_div(g, 16 * RT));
  const int64_t kinds = a.kv_heads * static_cast<int64_t>(grid.row_groups), blocks = ceil_div(a.room, 32);
  grid.least = W;
  grid.most = 128 / RT;
  grid.whole = 1.f;
  constexpr int64_t kParts = 512;
  int64_t extra = ceil_div(kParts, kinds);
  if (blocks <= grid.least) extra = 0;  // (nothing that could be cut)
  grid.extra = static_cast<int>(extra);
  const int64_t slots = problems + extra;
  if (slots > INT32_MAX / kinds) return fail("attn_paged: the launch has too many workgroups");
  grid.problems = static_cast<int>(problems);
  grid.slots = static_cast<int>(slots);
  std::unique_lock<std::recursive_mutex> lock;
  if (extra > 0 && split_scratch(s, static_cast<size_t>(kinds * 2 * extra) * 16 * RT * (DP + 2) * sizeof(float), static_cast<size_t>(kinds * problems), static_cast<int>(extra),
                                 &grid.ws, &grid.arrivals, &lock) != 0)
    return -1;
  hipLaunchKernelGGL((attn_paged_kernel<DP, RT, W, GROUP>), dim3(static_cast<unsigned>(kinds * slots)), dim3(64 * W), 0, s, a, grid);
  return check_launch("attn_paged");
}
template <int DP>
int launch_paged_rows(const PagedArgs& a, int64_t batch, int beams, hipStream_t s) {
  constexpr int W = DP <= 128 ? 8 : 4;
  const int g = a.heads / a.kv_heads;
  // a problem holds as many sequences of a group as 32 rows do
  if (beams > 1 && g <= 16) {
    int sub = 32 / g;
    sub = sub > beams ? beams : sub;
    if (sub * g <= 16) return launch_paged<DP, 1, W, true>(a, batch, beams, sub, s);
    return launch_paged<DP, 2, W, true>(a, batch, beams, sub, s);
  }
  if (g <= 16) return launch_paged<DP, 1, W, false>(a, batch, beams, 1, s);
  return launch_paged<DP, 2, W, false>(a, batch, beams, 1, s);
}

}  // namespace
}  // namespace dtas

extern "C" int dtas_attn_paged_f16(const void* Q, const void* K_pages, const void* V_pages, const void* table, const void* lens, void* out, int64_t batch, int64_t heads,
                                   int64_t kv_heads, int64_t d, int64_t page, int64_t pages, int64_t columns, int64_t beams, float scale, void* stream) {
  using namespace dtas;
  clear_error();
  if (batch < 0 || heads < 0 || kv_heads < 0 || d < 0 || pages < 0 || columns < 0)
    return fail("attn_paged: negative extent batch=%lld heads=%lld kv_heads=%lld d=%lld pages=%lld columns=%lld", (long long)batch, (long long)heads, (long long)kv_heads,
                (long long)d, (long long)pages, (long long)columns);
  if (page < 1) return fail("attn_paged: a page holds at least one position, got %lld", (long long)page);
  if (beams < 1 || batch % beams != 0) return fail("attn_paged: %lld sequences do not form groups of %lld", (long long)batch, (long long)beams);
  if (batch == 0 || heads == 0 || d == 0) return 0;
  if (kv_heads == 0 || heads % kv_heads != 0)
    return fail("attn_paged: %lld query heads do not share %lld key heads evenly", (long long)heads, (long long)kv_heads);
  if (d > 256) return fail("attn_paged: head dimensions up to 256, got %lld", (long long)d);
  constexpr int64_t kMost = int64_t{1} << 60;
  if (heads > 65535 || batch > INT32_MAX || pages > INT32_MAX / page || columns > INT32_MAX || page > INT32_MAX || columns > kMost / batch)
    return fail("attn_paged: the extents overflow");
  if (!(scale >= -2.0e38f && scale <= 2.0e38f)) return fail("attn_paged: the scale is not a finite number up to 2e38");
  if (!Q || !lens || !out || (columns > 0 && !table) || (pages > 0 && (!K_pages || !V_pages))) return fail("attn_paged: NULL buffer");
  const int64_t out_bytes = batch * heads * d * 2, page_bytes = pages * kv_heads * page * d * 2;
  if (overlaps(out, out_bytes, Q, out_bytes) || overlaps(out, out_bytes, K_pages, page_bytes) || overlaps(out, out_bytes, V_pages, page_bytes) ||
      overlaps(out, out_bytes, table, batch * columns * 4) || overlaps(out, out_bytes, lens, batch * 4))
    return fail("attn_paged: output overlaps an input");
  PagedArgs a{static_cast<const half_t*>(Q), static_cast<const half_t*>(K_pages), static_cast<const half_t*>(V_pages), static_cast<const int*>(table),
              static_cast<const int*>(lens), static_cast<half_t*>(out), static_cast<int>(heads), static_cast<int>(kv_heads), static_cast<int>(d), static_cast<int>(pages),
              static_cast<unsigned>(page), static_cast<unsigned>(columns * page < INT32_MAX ? columns * page : INT32_MAX), columns, scale == 0.f ? 1.f : fabsf(scale) * 1.4426950408889634f, static_cast<half_t>(scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d % 8 == 0 && page % 16 == 0 && pages > 0 && aligned(Q, 16) && aligned(K_pages, 16) && aligned(V_pages, 16) && aligned(out, 16)) {
    const int group = static_cast<int>(beams < INT32_MAX ? beams : INT32_MAX);
    if (d <= 64) return launch_paged_rows<64>(a, batch, group, s);
    if (d <= 96) return launch_paged_rows<96>(a, batch, group, s);
    if (d <= 128) return launch_paged_rows<128>(a, batch, group, s);
    if (d <= 192) return launch_paged_rows<192>(a, batch, group, s);
    return launch_paged_rows<256>(a, batch, group, s);
  }
  const int64_t total = batch * heads;
  const int64_t grid = total < (int64_t{1} << 22) ? total : int64_t{1} << 22;
  hipLaunchKernelGGL(attn_paged_scalar_kernel, dim3(static_cast<unsigned>(grid)), dim3(64), 0, s, a, total);
  return check_launch("attn_paged");
}
