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
  unsigned page, magic, shift;  // j / page = (j * magic >> 32) >> shift for j < 2^31
  unsigned room;                // positions that a table holds at most
  int64_t columns;
  float scale_log2;  // |scale| * log2(e): the softmax is taken in powers of two
  half_t sign;       // the scale's: 1, -1, or 0 (scale_log2 is 1 then)
};

// positions of a sequence (its table holds no more)
__device__ __forceinline__ unsigned length_of(const PagedArgs& a, int64_t b) {
  const int len = a.lens[b];
  return len < 0 ? 0u : static_cast<unsigned>(len) > a.room ? a.room : static_cast<unsigned>(len);
}

__device__ __forceinline__ unsigned column_of(const PagedArgs& a, unsigned pos) { return __umulhi(pos, a.magic) >> a.shift; }

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
// wavefront's own and is read from there transposed.  A weight goes into the product with V as two fp16 numbers of 11 bits, itself and what its rounding left, so that the answer has
// the bits of weights in fp32, as element by element (with the first alone it was off by up to 2^-12 of the sum of |v|): 1 after 127 keys 5.46 us with one, 5.54 with both, 4 beams after 32749 41.9 / 42.3,
// 61 after up to 2047 47.5 / 47.8, 16 after up to 65533 level, other forms 0.3 to 2 %.  The next visit's K and V are on their way in registers, and the table's entries a block further ahead.
// In a group a block is visited once for every page that its sequences name there; rows that do not name it have their scores masked.
// The blocks of all problems, one behind the other, are dealt out in equal shares, on the device, which knows the lengths: see Share.
// Memory bounds it: 16 sequences after up to 65533 keys (32 heads on 8 of 128, 2.34 GB) 360 us, 6.5 TB/s, where a kernel that only reads pieces of 8 .. 32 KiB in no order reaches 6.7 .. 6.9;
// 61 after up to 2047 (284 MB) 47.8 us, 5.9 TB/s; 4 beams after 32749 (175 MB) 42.3 us, of which handing the pieces' sums over takes 6 .. 8.  One sequence after 127 keys takes 5.5 us: a launch
// and four trips to memory, one behind the other (length, table, keys, the answer).
constexpr int kAgent = 16;    // loads past the L2 of an XCD (sc1), as atomic ones of the device's scope are, but 16 bytes wide: 4 beams after 32749 keys 41.5 us, 43.9 with two of 8
constexpr int kStreamed = 2;  // loads that nobody repeats (nt): 2.3 GB in pieces of 8 KiB 6.0 TB/s without, 6.8 with
constexpr int kNear = 8;
constexpr int kLonger = 32;    // blocks by which a problem may be longer than an even share
constexpr int kLong = 48;
constexpr int kCounted = 512;  // sequences that are looked at for that
constexpr unsigned kSlotsY = 65535;  // a grid's extent in y
constexpr int most_shares(int RT) { return 256 / RT; }
__device__ __forceinline__ uint64_t pair_of(float a, float b) { return static_cast<uint64_t>(__builtin_bit_cast(unsigned, a)) | static_cast<uint64_t>(__builtin_bit_cast(unsigned, b)) << 32; }
struct PagedGrid {
  int problems, beams, sub, subs;  // a problem: `sub` sequences at most of a group of `beams`, `subs` of which make up the group
  int shares, row_groups;          // workgroups per key head and row group that may share
  float one_of;                    // 1 / shares, and a little
  int least, whole;                // a share's blocks, if there are as many; blocks up to which a problem is in one piece
  int batch, worth;                // sequences; blocks of all of them from which on groups are read together (kLong of them in one at least)
  float* ws;
  unsigned* arrivals;
};
__device__ __forceinline__ int first_sequence(const PagedGrid& grid, int p, int* count) {
  const int group = p / grid.subs, s = p - group * grid.subs, left = grid.beams - s * grid.sub;
  *count = left < grid.sub ? left : grid.sub;
  return group * grid.beams + s * grid.sub;
}
// the length of a problem: that of its longest sequence
template <bool GROUP>
__device__ __forceinline__ unsigned problem_length(const PagedArgs& a, const PagedGrid& grid, int p) {
  if (!GROUP) return length_of(a, p);
  int count;
  const int b = first_sequence(grid, p, &count);
  unsigned longest = length_of(a, b);
  for (int i = 1; i < count; ++i) {
    const unsigned len = length_of(a, b + i);
    longest = longest > len ? longest : len;
  }
  return longest;
}
// its blocks of 32 keys (one, to write its noughts, where it is empty)
__device__ __forceinline__ int blocks_of(unsigned len) { return len < 32 ? 1 : static_cast<int>((len + 31) / 32); }
// Whether groups are read together: what that saves, with pages that are all shared, is more than its longer way costs (launch_paged_rows has the figures).  Of more than kCounted
// sequences as many are looked at, evenly over the batch
__device__ __forceinline__ bool together(const PagedArgs& a, const PagedGrid& grid, int lane) {
  const int some = grid.batch < kCounted ? grid.batch : kCounted;
  int total = 0, top = 0;
#pragma unroll 4
  for (int c = lane; c < some; c += 64) {
    const int blocks = blocks_of(length_of(a, some < kCounted ? c : static_cast<int64_t>(c) * grid.batch / kCounted));
    total += blocks;
    top = top > blocks ? top : blocks;
  }
  total = wave_total(total);
  top = wave_most(top);
  return top >= kLong && static_cast<float>(total) * (static_cast<float>(grid.batch) / static_cast<float>(some)) >= static_cast<float>(grid.worth);
}
// Where the longest problem is not much longer than an even share of all blocks (7 sequences on 32 heads of 80 after 6550 .. 26209 keys: cut 176 us, whole 265; 10 after up to 2000 27.6 / 26.3), or
// short, each workgroup has a problem.  Otherwise workgroup s has the blocks from s * per up to
// (s + 1) * per, but for a boundary less than `near` from the end of a problem, which moves there: a problem is cut into pieces only where that is worth handing its sums over.
// Every workgroup finds out for itself which problem its share begins in (p, of length len, whose blocks begin at `at`), and what pieces there are of a problem follows from where
// its blocks begin and end.
struct Share {
  int p, at, from, to, per, near;  // (p < 0: nothing to do)
  unsigned len;
};
template <int W, bool GROUP>
__device__ __forceinline__ Share find_share(const PagedArgs& a, const PagedGrid& grid, int s, int lane, int wave) {
  auto deal = [&](int total, int longest) {
    int per = static_cast<int>(static_cast<float>(total) * grid.one_of) + 1;  // (a little more than an even share: all of them hold everything)
    per = per > grid.least ? per : grid.least;
    if (longest - kLonger <= per || longest <= grid.whole) return Share{s < grid.problems ? s : -1, 0, 0, 0, 1 << 30, 1, 0};
    const int64_t from = static_cast<int64_t>(s) * per;
    return Share{s < grid.shares && from < total ? 0 : -1, 0, static_cast<int>(from), total - from > per ? static_cast<int>(from + per) : total, per, per / kNear + 1, 0};
  };
  if (grid.shares == 1) {
    Share share{s < grid.problems ? s : -1, 0, 0, 0, 1 << 30, 1, 0};
    if (share.p < 0) return share;
    share.len = problem_length<GROUP>(a, grid, share.p);
    share.to = blocks_of(share.len);
    return share;
  }
  if (grid.problems <= 64) {
    const unsigned len = lane < grid.problems ? problem_length<GROUP>(a, grid, lane) : 0;
    const int blocks = lane < grid.problems ? blocks_of(len) : 0, upto = sum_upto(blocks);
    Share share = deal(__builtin_amdgcn_readlane(upto, 63), wave_most(blocks));
    if (share.p < 0) return share;
    if (share.per == 1 << 30) {
      share.len = static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(len), share.p));
      share.to = blocks_of(share.len);
      return share;
    }
    share.p = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > share.from));
    share.len = static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(len), share.p));
    share.at = __builtin_amdgcn_readlane(upto, share.p) - blocks_of(share.len);
    return share;
  }
  // the wavefronts have a range of the problems each
  __shared__ int totals[W], tops[W], found[2];
  const int range = (grid.problems + 64 * W - 1) / (64 * W) * 64, first = wave * range, last = first + range < grid.problems ? first + range : grid.problems;
  int total = 0, top = 0;
#pragma unroll 4
  for (int c = first + lane; c < last; c += 64) {
    const int blocks = blocks_of(problem_length<GROUP>(a, grid, c));
    total += blocks;
    top = top > blocks ? top : blocks;
  }
  total = wave_total(total);
  top = wave_most(top);
  if (lane == 0) {
    totals[wave] = total;
    tops[wave] = top;
  }
  __syncthreads();
  int base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w == wave) base = all;
    all += totals[w];
    top = top > tops[w] ? top : tops[w];
  }
  Share share = deal(__builtin_amdgcn_readfirstlane(all), __builtin_amdgcn_readfirstlane(top));
  if (share.p < 0) return share;
  if (share.per == 1 << 30) {
    share.len = problem_length<GROUP>(a, grid, share.p);
    share.to = blocks_of(share.len);
    return share;
  }
  if (share.from >= base && share.from < base + total) {
    for (int c = first; c < last; c += 64) {
      const int blocks = c + lane < last ? blocks_of(problem_length<GROUP>(a, grid, c + lane)) : 0, upto = base + sum_upto(blocks);
      const uint64_t behind = __builtin_amdgcn_ballot_w64(upto > share.from);
      if (behind != 0) {
        const int l = __builtin_ctzll(behind), at = __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(blocks, l);  // (outside the branch, where all lanes are)
        if (lane == 0) {
          found[0] = c + l;
          found[1] = at;
        }
        break;
      }
      base = __builtin_amdgcn_readlane(upto, 63);
    }
  }
  __syncthreads();
  share.p = __builtin_amdgcn_readfirstlane(found[0]);
  share.at = __builtin_amdgcn_readfirstlane(found[1]);
  share.len = problem_length<GROUP>(a, grid, share.p);
  return share;
}

// The 8 channels of k step ks that a lane of `quarter` holds.  Of two steps that make up a 128-byte line of a row a lane has 32 contiguous bytes; of a single last one 16.
template <int DP>
__device__ __forceinline__ int channels_at(int ks, int quarter) {
  return ks / 2 * 2 + 1 < DP / 32 ? ks / 2 * 64 + quarter * 16 + (ks & 1) * 8 : ks * 32 + quarter * 8;
}
template <int DP>
__device__ __forceinline__ f16x8 channels_of(const half_t* row, int ks, int quarter, int d) {
  const int at = channels_at<DP>(ks, quarter);
  const f16x8 v = *reinterpret_cast<const f16x8*>(row + (at < d ? at : d - 8));
  return at < d ? v : f16x8{};
}

// two halves of 16 keys at positions pos and pos + 16: where their K and V lie (bytes from the head's first), how many bytes of them are read (what is behind comes as nought,
// and costs nothing), and which sequences of the problem (bits) see them
struct Visit {
  int64_t at[2];
  unsigned bytes[2], seen[2], pos;
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

// About how many blocks the sequences of a group have in common: 64 columns are looked at (which of them does not matter to the result)
__device__ __forceinline__ int common_blocks(const PagedArgs& a, const int* names, int nb, unsigned my_len, unsigned longest, int lane) {
  const unsigned columns = (longest + a.page - 1) / a.page, column = static_cast<unsigned>(static_cast<uint64_t>(columns) * lane / 64);
  const int theirs = column < columns ? names[column] : -1;
  bool same = true;
  for (int i = 1; i < nb; i += 4) {
    int some[4];
    unsigned len[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = i + u < nb ? i + u : nb - 1;
      len[u] = __shfl(my_len, j);
      some[u] = column * a.page < len[u] ? names[static_cast<int64_t>(j) * a.columns + column] : -1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) same = same && some[u] == theirs;
  }
  const uint64_t apart = __builtin_amdgcn_ballot_w64(!same);
  const int l = apart == 0 ? 64 : __builtin_ctzll(apart);
  if (l == 64) return static_cast<int>((longest + 31) / 32);
  return l == 0 ? 0 : static_cast<int>(static_cast<unsigned>(static_cast<uint64_t>(columns) * (l - 1) / 64) * a.page / 32);
}

// An infinite value may meet a weight too small for fp16 (below 2^-36 of the largest), or one whose rounding left nothing, or less than nothing: zero times infinity, or infinities
// of both signs, though the weight is a number in fp32 and the channel infinite.  Such a channel shows in the sums, as NaN where the sum of the weights is a number (rare); what visits of a group took out is known as well.  What it is instead depends
// on the keys alone whose values are no numbers: a thread looks for them in four channels of a row, among what its workgroup visited of the row's sequence (items first .. last), and
// sums them with their weights in fp32.
struct Visited {
  const int* names;  // the problem's tables
  int b0, nb, common, first, last, p_blocks, hk;
};
__device__ f32x4 values_no_numbers(const PagedArgs& a, const Visited& v, int beam, const half_t* q, int channel, float best) {
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  const unsigned len = length_of(a, v.b0 + beam);
  const int blocks = static_cast<int>((len + 31) / 32);
  for (int half = 0; half < 2 * blocks; ++half) {
    const unsigned pos = 16u * half, column = column_of(a, pos);
    const int page = pos < len ? v.names[static_cast<int64_t>(beam) * a.columns + column] : -1;
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pages)) continue;
    int item = half / 2;
    if (item >= v.common) {  // (visited with the first sequence that names the page there)
      int one = 0;
      for (; one < beam; ++one)
        if (pos < length_of(a, v.b0 + one) && v.names[static_cast<int64_t>(one) * a.columns + column] == page) break;
      item = v.common + (item - v.common) * v.nb + one;
    }
    if (item < v.first || item >= v.last) continue;
    const int64_t from = ((static_cast<int64_t>(page) * a.kv_heads + v.hk) * a.page + (pos - column * a.page)) * a.d;
    f16x4 some[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) some[r] = *reinterpret_cast<const f16x4*>(a.V + from + static_cast<int64_t>(r) * a.d + channel);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      bool odd = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) odd = odd || !(fabsf(static_cast<float>(some[r][j])) < INFINITY);
      if (!odd || pos + r >= len) continue;
      const half_t* k = a.K + from + static_cast<int64_t>(r) * a.d;
      float t = 0.f;
      for (int c = 0; c < a.d; ++c) t = fmaf(static_cast<float>(k[c]), static_cast<float>(q[c]), t);
      t *= static_cast<float>(a.sign);
      const float weight = t == -INFINITY ? 0.f : exp2_fast(fmaf(t - best, a.scale_log2, kRoom));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float value = static_cast<float>(some[r][j]);
        if (!(fabsf(value) < INFINITY)) sum[j] = fmaf(weight, value, sum[j]);
      }
    }
  }
  return sum;
}

template <int DP, int RT, int W, bool GROUP>
__global__ void __launch_bounds__(64 * W, DP <= 128 ? 2 : 1) attn_paged_kernel(PagedArgs a, PagedGrid grid) {
  if constexpr (GROUP) {
    if (!together(a, grid, threadIdx.x & 63)) {
      grid.problems = grid.batch;
      grid.sub = 1;
      grid.subs = grid.beams;
    }
  }
  constexpr int KS = DP / 32, DT = DP / 16, VL = DP / 16, VH = VL / 2;  // k steps, channel tiles, 16-byte pieces of V per lane, of a half
  constexpr int kRows = 16 * RT, kChunks = DP / 8, kWave = 32 * v_row_bytes(DP), kShare = kRows * (DP + 2);
  __shared__ __attribute__((aligned(16))) char lds[W * kWave];
  __shared__ float stat_m[W][kRows], stat_l[W][kRows];
  __shared__ int flag, took_out[W];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = a.heads / a.kv_heads;
  // (the key heads of a share next to each other: their pages are)
  int hk = static_cast<int>(blockIdx.x), rg = 0;
  const int s_mine = static_cast<int>(blockIdx.z * kSlotsY + blockIdx.y);
  if (grid.row_groups > 1) {
    rg = hk / a.kv_heads;
    hk -= rg * a.kv_heads;
  }
  const Share share = find_share<W, GROUP>(a, grid, s_mine, threadIdx.x & 63, wave);
  if (share.p < 0) return;
  const unsigned row_bytes = 2u * a.d;
  const int64_t head_bytes = static_cast<int64_t>(a.page) * row_bytes, page_bytes = head_bytes * a.kv_heads;
  const char *Kh = reinterpret_cast<const char*>(a.K) + hk * head_bytes, *Vh = reinterpret_cast<const char*>(a.V) + hk * head_bytes;
  const int64_t kind = static_cast<int64_t>(hk) * grid.row_groups + rg;
  char* mine = lds + wave * kWave;

  for (int p = share.p, begin = share.at, end; begin < share.to; ++p, begin = end) {
    const unsigned longest = static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(p == share.p ? share.len : problem_length<GROUP>(a, grid, p))));
    const int p_blocks = blocks_of(longest);
    end = begin + p_blocks;
    // this problem's cuts: boundaries s from first_cut to last_cut; the blocks that are this workgroup's, and which piece they are
    int first_cut = 1, cuts = 0;
    if (share.per != 1 << 30) {
      first_cut = (begin + share.near + share.per - 1) / share.per;
      const int last_cut = (end - share.near) / share.per;
      cuts = last_cut >= first_cut ? last_cut - first_cut + 1 : 0;
    }
    int lo = 0, hi = p_blocks, z = 0;
    if (begin < share.from) {
      if (share.from - begin < share.near) lo = 0;
      else if (end - share.from < share.near) continue;
      else lo = share.from - begin, z = s_mine - first_cut + 1;
    }
    if (end > share.to) {
      if (share.to - begin < share.near) break;
      if (end - share.to >= share.near) hi = share.to - begin;
    }
    const int parts = cuts + 1;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // (what depends on it is computed for each problem anew: kept from one to the next it would take half the registers)
    const int lane = tid & 63, quarter = lane >> 4, i16 = lane & 15;
    const unsigned tr_at = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)mine)) +
                           (4 * quarter + (i16 >> 2)) * v_row_bytes(DP) + (i16 & 3) * 8;
    int nb = 1;
    const int b0 = GROUP ? first_sequence(grid, p, &nb) : p, R = nb * g;

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
      for (int ks = 0; ks < KS; ++ks) q[rt][ks] = channels_of<DP>(row, ks, quarter, a.d) * a.sign;
      row_len[rt] = GROUP ? length_of(a, b0 + beam[rt]) : longest;
    }
    // lengths of the sequences (GROUP: lane i & 31 holds sequence i's), and the shortest
    const unsigned my_len = GROUP ? ((lane & 31) < nb ? length_of(a, b0 + (lane & 31)) : 0u) : longest;
    const unsigned shortest = GROUP ? 0x7fffffffu - static_cast<unsigned>(wave_most((lane & 31) < nb ? static_cast<int>(0x7fffffffu - my_len) : 0)) : longest;
    const unsigned everyone = nb >= 32 ? ~0u : (1u << nb) - 1u;

    // ---- where the next visit is
    const int* names = a.table + static_cast<int64_t>(b0) * a.columns;
    auto place = [&](Visit& to, int h, int page, unsigned in_page, bool there) {
      const unsigned pos = to.pos + 16 * h, rows = pos < longest ? longest - pos : 0u;
      to.at[h] = page * page_bytes + static_cast<int64_t>(in_page) * row_bytes;
      to.bytes[h] = there ? (rows < 16 ? rows : 16u) * row_bytes : 0u;
    };
    // What the wavefronts take in turn: blocks; in a group a block that all share, and of the others (from about `common` on) a block for each sequence, which visits what that
    // one names first.  So pieces of a group that has grown apart are as long as others.
    int common = p_blocks, first = lo, last = hi;
    if constexpr (GROUP) {
      common = common_blocks(a, names, nb, my_len, longest, lane);
      const int items = common + (p_blocks - common) * nb;
      const float ratio = static_cast<float>(items) / static_cast<float>(p_blocks);
      auto item_of = [&](int at) {
        const int it = static_cast<int>(static_cast<float>(at) * ratio);
        return at >= p_blocks || it > items ? items : it;
      };
      first = item_of(lo);
      last = item_of(hi);
    }
    auto block_of = [&](int it, int& one) {
      one = -1;
      if (!GROUP || it < common) return it;
      const unsigned q = static_cast<unsigned>(it - common), b = q / static_cast<unsigned>(nb);
      one = static_cast<int>(q - b * nb);
      return common + static_cast<int>(b);
    };
    int item = first + wave;  // the one whose entries come next
    // GROUP: a block's entries, lane (half, sequence); else those of 32 of the wavefront's blocks, lane (block, half)
    auto gather = [&](int at, int& entry, unsigned& in_page) {
      int one;
      const unsigned pos = GROUP ? static_cast<unsigned>(block_of(at, one)) * 32 + (lane >> 5) * 16 : static_cast<unsigned>(at + (lane >> 1) * W) * 32 + (lane & 1) * 16;
      const unsigned column = column_of(a, pos);
      in_page = pos - column * a.page;
      entry = pos < my_len && (!GROUP || (lane & 31) < nb) ? names[(GROUP ? static_cast<int64_t>(lane & 31) * a.columns : 0) + column] : -1;
    };
    int entry, entry_next;
    unsigned in_page, in_page_next, left[2] = {0, 0}, pos_now = 0;
    int taken = 0;  // (of the 32 blocks)
    gather(item, entry, in_page);
    entry_next = -1;
    in_page_next = 0;
    if (GROUP || item + 32 * W < last) gather(item + (GROUP ? W : 32 * W), entry_next, in_page_next);
    auto advance = [&](Visit& to) -> bool {
      if constexpr (GROUP) {
        while ((left[0] | left[1]) == 0) {
          if (item >= last) {
            to.bytes[0] = to.bytes[1] = 0;
            return false;
          }
          if (taken != 0) {  // (the first one's entries are there)
            entry = entry_next;
            in_page = in_page_next;
            gather(item + W, entry_next, in_page_next);
          }
          taken = 1;
          int one;
          pos_now = static_cast<unsigned>(block_of(item, one)) * 32;
          item += W;
          const uint64_t some = __builtin_amdgcn_ballot_w64(static_cast<unsigned>(entry) < static_cast<unsigned>(a.pages));
          left[0] = static_cast<unsigned>(some);
          left[1] = static_cast<unsigned>(some >> 32);
          if (one >= 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int page = __builtin_amdgcn_readlane(entry, one + 32 * h);
              const unsigned same = static_cast<unsigned>(__builtin_amdgcn_ballot_w64(entry == page) >> (32 * h)) & left[h];
              left[h] = ((same >> one) & 1) != 0 && __builtin_ctz(same) == one ? same : 0u;
            }
          }
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
#pragma unroll
        for (int h = 0; h < 2; ++h) place(to, h, page[h], static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(in_page), 32 * h)), to.seen[h] != 0);
      } else {
        if (item >= last) {
          to.bytes[0] = to.bytes[1] = 0;
          return false;
        }
        if (taken == 32) {
          entry = entry_next;
          in_page = in_page_next;
          gather(item + 32 * W, entry_next, in_page_next);
          taken = 0;
        }
        to.pos = static_cast<unsigned>(item) * 32;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int page = __builtin_amdgcn_readlane(entry, 2 * taken + h);
          const bool there = static_cast<unsigned>(page) < static_cast<unsigned>(a.pages);
          to.seen[h] = there ? 1u : 0u;
          place(to, h, there ? page : 0, static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(in_page), 2 * taken + h)), there);
        }
        ++taken;
        item += W;
      }
      return true;
    };

    // ---- a lane's pieces of K and V.  As the matrix cores take K, a load would touch 64 bytes of each of sixteen keys; two loads that make up a line fetch it whole for
    // eight keys each instead, and a rotation within sixteen lanes puts the pieces where they belong
    f16x8 kf[2][KS];
    u32x4 vf[VL];
    unsigned k_at[KS], v_at[VH];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const bool pair = ks / 2 * 2 + 1 < KS;
      const int row = pair ? (lane & 7) + 8 * (ks & 1) : i16, at = pair ? ks / 2 * 64 + (lane >> 3) * 8 : channels_at<DP>(ks, quarter);
      k_at[ks] = at < a.d ? row * row_bytes + 2u * at : kOob;
    }
#pragma unroll
    for (int n = 0; n < VH; ++n) {
      const int id = n * 64 + lane, c = id % kChunks;
      v_at[n] = c * 8 < a.d ? id / kChunks * row_bytes + 16u * c : kOob;
    }
    auto load_k = [&](const Visit& from) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const __amdgpu_buffer_rsrc_t r = make_rsrc(Kh + from.at[kt], from.bytes[kt]);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kf[kt][ks] = __builtin_bit_cast(f16x8, __builtin_amdgcn_raw_buffer_load_b128(r, k_at[ks], 0, kStreamed));
      }
    };
    auto settle_k = [&] {  // piece (load n, bit 3 of the lane = x) -> (step x, bit 3 = n)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int ks = 0; ks + 1 < KS; ks += 2) {
          u32x4 even = __builtin_bit_cast(u32x4, kf[kt][ks]), odd = __builtin_bit_cast(u32x4, kf[kt][ks + 1]);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int x = static_cast<int>(even[w]), y = static_cast<int>(odd[w]);
            even[w] = static_cast<unsigned>(__builtin_amdgcn_update_dpp(x, y, 0x128, 0xf, 0xc, false));  // row_ror:8 into lanes 8 .. 15 of a row
            odd[w] = static_cast<unsigned>(__builtin_amdgcn_update_dpp(y, x, 0x128, 0xf, 0x3, false));   // ... 0 .. 7
          }
          kf[kt][ks] = __builtin_bit_cast(f16x8, even);
          kf[kt][ks + 1] = __builtin_bit_cast(f16x8, odd);
        }
      }
    };
    auto load_v = [&](const Visit& from) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const __amdgpu_buffer_rsrc_t r = make_rsrc(Vh + from.at[h], from.bytes[h]);
#pragma unroll
        for (int n = 0; n < VH; ++n) vf[h * VH + n] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, v_at[n], 0, kStreamed));
      }
    };

    f32x4 o[RT][DT];
    float top[RT], sum[RT];
    bool saw[RT];
    unsigned taken_out = 0;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      top[rt] = -INFINITY;
      sum[rt] = 0.f;
      saw[rt] = false;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // (the next one's loads are not behind a branch, behind which the compiler would wait for them whenever it waits for an earlier one: the last visit's next has no bytes)
    auto visit = [&](const Visit& here, const Visit& next) {
      f32x4 s[RT][2];
      settle_k();
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          s[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) s[rt][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[kt][ks], q[rt][ks], s[rt][kt], 0, 0, 0);
        }
      load_k(next);
      const bool all = here.seen[0] == everyone && here.seen[1] == everyone && here.pos + 32 <= shortest;
      unsigned shown[RT];
      if (!all) {
        unsigned any = 0;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const int have = static_cast<int>(row_len[rt]) - static_cast<int>(here.pos);
          shown[rt] = ((here.seen[0] >> beam[rt]) & 1 ? bits_below(have) : 0u) | ((here.seen[1] >> beam[rt]) & 1 ? bits_below(have - 16) : 0u) << 16;
          saw[rt] = saw[rt] || shown[rt] != 0;
          any |= shown[rt];
        }
        if constexpr (GROUP) {
          // values that nobody sees, or only some rows, would meet weights of zero: the former go, and of the latter what is no number (rare), which is added at the end
          any = any_row(any);
#pragma unroll
          for (int n = 0; n < VL; ++n) {
            const bool there = ((any >> ((n * 64 + lane) / kChunks)) & 1) != 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const unsigned low = vf[n][w] & 0x7c00u, high = vf[n][w] & 0x7c000000u, gone = (low == 0x7c00u ? 0xffffu : 0u) | (high == 0x7c000000u ? 0xffff0000u : 0u);
              taken_out |= there ? gone : 0u;
              vf[n][w] = there ? vf[n][w] & ~gone : 0u;
            }
          }
        }
      } else {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          shown[rt] = ~0u;
          saw[rt] = true;
        }
      }
#pragma unroll
      for (int n = 0; n < VL; ++n) {
        const int id = n * 64 + lane, row = id / kChunks, c = id % kChunks;
        *reinterpret_cast<u32x4*>(mine + row * v_row_bytes(DP) + c * 16) = vf[n];
      }
      load_v(next);
      f16x8 p[RT], rest[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        weigh<2, DT>(s[rt], all, shown[rt], quarter, a.scale_log2, top[rt], sum[rt], o[rt]);
        p[rt] = weights_f16(s[rt][0], s[rt][1]);
        rest[rt] = weights_rest(s[rt][0], s[rt][1], p[rt]);
      }
      auto add = [&](int dt0, auto& lo, auto& hi) {
        constexpr int N = sizeof(lo) / sizeof(lo[0]);
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int u = 0; u < N; ++u) {
            const f16x8 vt = {lo[u][0], lo[u][1], lo[u][2], lo[u][3], hi[u][0], hi[u][1], hi[u][2], hi[u][3]};
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) o[rt][dt0 + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, part == 0 ? p[rt] : rest[rt], o[rt][dt0 + u], 0, 0, 0);
          }
      };
#pragma unroll
      for (int dt = 0; dt + 4 <= DT; dt += 4) {
        f16x4 lo[4], hi[4];
        read_v<DP>(tr_at + dt * 32, lo, hi);
        add(dt, lo, hi);
      }
      if constexpr (DT % 4 == 2) {
        f16x4 lo[2], hi[2];
        read_v<DP>(tr_at + (DT - 2) * 32, lo, hi);
        add(DT - 2, lo, hi);
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
      visit(here, next);
      here = next;
    }

    int tid_b = threadIdx.x;
    asm volatile("" : "+v"(tid_b));  // (nor is anything of what follows computed ahead of the visits)
    const int lane_b = tid_b & 63, quarter_b = lane_b >> 4, i16_b = lane_b & 15;
    // ---- what the wavefronts summed, joined in their order.  A row that saw nothing says so by a sum of -1 (its weight is zero where another's is not)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      sum[rt] = sum_of_row(sum[rt]);
      if (quarter_b == 0) {
        stat_m[wave][rt * 16 + i16_b] = top[rt];
        stat_l[wave][rt * 16 + i16_b] = saw[rt] ? sum[rt] : -1.f;
      }
    }
    if constexpr (GROUP) {
      const uint64_t some = __builtin_amdgcn_ballot_w64(taken_out != 0);
      if (lane_b == 0) took_out[wave] = some != 0;
    }
    __syncthreads();
    auto best_of = [&](int r) {
      float best = stat_m[0][r];
#pragma unroll
      for (int w = 1; w < W; ++w) best = fmaxf(best, stat_m[w][r]);
      return best;
    };
    const int my_rows = R - rg * kRows < kRows ? R - rg * kRows : kRows;
    // a piece's sums: of the one that begins a problem among the last ones of the workgroups, of others among the first ones
    float *firsts = grid.ws + kind * 2 * grid.shares * kShare, *lasts = firsts + static_cast<int64_t>(grid.shares) * kShare;
    auto sums_of = [&](int y) { return y == 0 ? lasts + static_cast<int64_t>(first_cut - 1) * kShare : firsts + static_cast<int64_t>(first_cut - 1 + y) * kShare; };
    float* handed = parts > 1 ? sums_of(z) : nullptr;
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
        const float w = weight_of(top[rt], best_of(row0 + i16_b), a.scale_log2);
        float* to = reinterpret_cast<float*>(mine) + i16_b * kPitch + 4 * quarter_b;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(to + dt * 16) = f32x4{o[rt][dt][0] * w, o[rt][dt][1] * w, o[rt][dt][2] * w, o[rt][dt][3] * w};
      }
      __syncthreads();
      for (int at = tid_b; at < 16 * (DP / 4); at += 64 * W) {
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
        const float all = (v[0] + v[1]) + (v[2] + v[3]);
        bool odd = all != all && l == l;
        if constexpr (GROUP)
          for (int w = 0; w < W; ++w) odd = odd || took_out[w] != 0;
        if (odd) {
          const int at_r = rg * kRows + r, beam_of = GROUP ? at_r / g : 0;
          const f32x4 fresh = values_no_numbers(a, Visited{names, b0, nb, common, first, last, p_blocks, hk}, beam_of,
                                                a.Q + (static_cast<int64_t>(b0 + beam_of) * a.heads + hk * g + (at_r - beam_of * g)) * a.d, c, best);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = fresh[j] + (v[j] == v[j] || l != l ? v[j] : 0.f);
        }
        if (parts > 1) {
          store_out(v, reinterpret_cast<f32x4*>(handed + r * DP + c), true);
          if (c == 0) store_stat(handed, kRows, DP, r, best, any ? l : -1.f);
        } else {
          store_row4(out_row(r) + c, v, any ? 1.f / l : 0.f);
        }
      }
      __syncthreads();
    }
    if (parts == 1 || !last_to_arrive(grid.arrivals + kind * grid.problems + p, parts, &flag)) continue;

    // ---- whoever is last joins the parts in their order: a wavefront per row finds the parts' weights, then a thread has four channels of a row, of every S-th part
    // where there are threads left
    constexpr int kItems = DP / 4, kAtOnce = 8;  // parts requested before the first is used: a trip to memory per eight
    const int items_all = my_rows * kItems;
    int spread = 1;
    while (spread * 2 * items_all <= 64 * W && spread < parts) spread *= 2;
    const int lot = tid_b / items_all, mine_of = tid_b - lot * items_all;
    f32x4 some[kAtOnce];
    const __amdgpu_buffer_rsrc_t pieces = make_rsrc(firsts, 8u * grid.shares * kShare);
    auto request = [&](int at, int y0) {
      const int offset = at / kItems * DP + 4 * (at % kItems);
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int y = y0 + u * spread < parts ? y0 + u * spread : parts - 1;
        some[u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(pieces, 4u * (((y == 0 ? grid.shares : y) + first_cut - 1) * kShare + offset), 0, kAgent));
      }
    };
    if (lot < spread) request(mine_of, lot);  // (on their way while the statistics come)
    constexpr int kMost = most_shares(RT);
    float* weights = reinterpret_cast<float*>(lds);  // [row][part]
    static_assert(kRows * kMost * 4 + 64 * W * 16 <= W * kWave, "the parts' weights and the threads' sums fit the LDS");
    for (int i = wave; i < my_rows; i += W) {
      float tops[kMost / 64], sums[kMost / 64], best = -INFINITY, total = 0.f;
      bool any = false;
#pragma unroll
      for (int c = 0; c < kMost / 64; ++c) {
        const int y = c * 64 + lane_b;
        uint64_t two = pair_of(-INFINITY, -1.f);
        if (y < parts) two = __hip_atomic_load(reinterpret_cast<const uint64_t*>(sums_of(y) + kRows * DP) + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        tops[c] = __builtin_bit_cast(float, static_cast<unsigned>(two));
        sums[c] = __builtin_bit_cast(float, static_cast<unsigned>(two >> 32));
        any = any || !(sums[c] < 0.f);
        best = fmaxf(best, tops[c]);
      }
      best = wave_max(best);
#pragma unroll
      for (int c = 0; c < kMost / 64; ++c) {
        tops[c] = weight_of(tops[c], best, a.scale_log2);
        total = fmaf(tops[c], sums[c], total);
      }
      total = wave_sum(total);
      const float inv = __builtin_amdgcn_ballot_w64(any) != 0 ? 1.f / total : 0.f;
#pragma unroll
      for (int c = 0; c < kMost / 64; ++c)
        if (c * 64 + lane_b < parts) weights[i * kMost + c * 64 + lane_b] = tops[c] * inv;
    }
    __syncthreads();
    if (spread > 1) {
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (lot < spread) {
        const float* w = weights + mine_of / kItems * kMost;
        for (int y0 = lot; y0 < parts; y0 += kAtOnce * spread) {
          if (y0 != lot) request(mine_of, y0);
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) {
            const int y = y0 + u * spread;
            if (y >= parts) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = fmaf(w[y], some[u][j], v[j]);
          }
        }
      }
      f32x4* sums = reinterpret_cast<f32x4*>(lds + kRows * kMost * 4);
      sums[tid_b] = v;
      __syncthreads();
      if (lot == 0) {
        for (int s = 1; s < spread; ++s) {
          const f32x4 one = sums[s * items_all + mine_of];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] += one[j];
        }
        const int c = 4 * (mine_of % kItems);
        if (c < a.d) store_row4(out_row(mine_of / kItems) + c, v, 1.f);
      }
    } else {
      for (int at = tid_b; at < items_all; at += 64 * W) {
        const float* w = weights + at / kItems * kMost;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        for (int y0 = 0; y0 < parts; y0 += kAtOnce) {
          if (y0 > 0 || at != tid_b) request(at, y0);
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) {
            if (y0 + u >= parts) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = fmaf(w[y0 + u], some[u][j], v[j]);
          }
        }
        const int c = 4 * (at % kItems);
        if (c < a.d) store_row4(out_row(at / kItems) + c, v, 1.f);
      }
    }
    __syncthreads();  // (the LDS is the next problem's)
  }
}

// Blocks of all sequences on all key heads whose reading once per sequence instead of once per group would cost each CU kSaved bytes
constexpr double kSaved = 200e3;
inline int64_t worth_grouping(const PagedArgs& a, int sub) {
  const double bytes = 128.0 * a.d * a.kv_heads * (1.0 - 1.0 / sub) / 256.0, blocks = sub > 1 ? kSaved / bytes : 1e9;
  return static_cast<int64_t>(blocks < 1e9 ? blocks : 1e9);
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
  const int64_t kinds = a.kv_heads * static_cast<int64_t>(grid.row_groups), blocks = a.room < 32 ? 1 : ceil_div(a.room, 32), most = GROUP ? batch : problems;
  if (problems * grid.sub > (int64_t{1} << 30) / blocks) return fail("attn_paged: the tables hold too many positions");
  grid.problems = static_cast<int>(problems);
  grid.batch = static_cast<int>(batch);
  grid.worth = GROUP ? static_cast<int>(worth_grouping(a, grid.sub)) : 0;
  grid.least = 8;
  grid.whole = 24;
  // workgroups of four wavefronts share a CU, but for those of large heads: 16 sequences on 32 heads of 80 after up to 10000 keys 148 us, with 256 of them 174
  constexpr int64_t kWorkgroups = DP <= 128 && W == 4 ? 512 : 256;
  int64_t shares = kinds < kWorkgroups ? kWorkgroups / kinds : 1;
  shares = shares < most_shares(RT) ? shares : most_shares(RT);
  if (blocks <= grid.whole || most > 4096) shares = 1;  // (nothing that could be cut; so many sequences that reading all their lengths in each workgroup costs more than it gives: 8192 after 30 keys, in tables of 4096, 326 us, 543 without)
  const int64_t slots = most > shares ? most : shares;
  if (slots > INT32_MAX / kinds || slots > int64_t{kSlotsY} * 65535) return fail("attn_paged: the launch has too many workgroups");
  grid.shares = static_cast<int>(shares);
  grid.one_of = 1.000001f / static_cast<float>(shares);
  std::unique_lock<std::recursive_mutex> lock;
  if (shares > 1 && split_scratch(s, static_cast<size_t>(kinds * 2 * shares) * 16 * RT * (DP + 2) * sizeof(float), static_cast<size_t>(kinds * most), static_cast<int>(shares),
                                  &grid.ws, &grid.arrivals, &lock) != 0)
    return -1;
  hipLaunchKernelGGL((attn_paged_kernel<DP, RT, W, GROUP>), dim3(static_cast<unsigned>(kinds), static_cast<unsigned>(slots < kSlotsY ? slots : kSlotsY), static_cast<unsigned>(ceil_div(slots, kSlotsY))), dim3(64 * W), 0, s, a, grid);
  return check_launch("attn_paged");
}
template <int DP>
int launch_paged_rows(const PagedArgs& a, int64_t batch, int beams, hipStream_t s) {
  const int g = a.heads / a.kv_heads;
  // A problem holds as many sequences of a group as make sixteen rows; with heads of more than 128 they are read one by one.  (32 rows read what more of them share once, but a problem's
  // own pages are then in fewer workgroups, and for heads of 128 in four wavefronts each, for want of registers: 45 sequences in groups of 5 after 675 keys 48.0 us / 29.2, 8 beams after
  // 16000 on 4 heads of 80 38.3 / 25.4; only 7 such groups after 53876 gain, 104 / 125.)
  if constexpr (DP <= 128) {
    if (g <= 16) {
      int sub = beams > 1 ? (16 / g < beams ? 16 / g : beams) : 1;
      // Read together where that saves each CU 200 KB at least, in sequences of 1536 keys or more (the tables say it could, and the lengths then that it does): groups on their way have
      // more trips to memory and fewer, longer problems.  Apart / together: 32 sequences in groups of 4, 32 heads on 8 of 128, after 500 keys 11.1 us / 17.0, 2000 26.6 / 28.4, 8000 89.1 / 46.7;
      // 8 beams on 32 heads of 128 after 120 7.2 / 21.8, 1000 16.6 / 22.4, 4000 48.2 / 30.3; 4 beams, 32 heads on 8, after 2000 16.8 / 17.1, 16000 41.5 / 28.2.
      if (a.room < 32u * kLong || batch * ceil_div(a.room, 32) < worth_grouping(a, sub)) sub = beams = 1;
      // Eight wavefronts where few problems are cut, four, and two workgroups per CU, where each CU has several to itself: 4 beams after 32749 keys 43.2 us / 48.6, 61 sequences after
      // up to 2047 on 8 heads 47.2 / 52.1; 64 on 32 heads of 80 after up to 300 55.4 / 30.2, 300 on 8 of 128 after up to 100 61.6 / 28.8.
      const bool many = batch / beams * ((beams + sub - 1) / sub) * a.kv_heads >= 512;
      if (beams > 1) return many ? launch_paged<DP, 1, 4, true>(a, batch, beams, sub, s) : launch_paged<DP, 1, 8, true>(a, batch, beams, sub, s);
      return many ? launch_paged<DP, 1, 4, false>(a, batch, beams, 1, s) : launch_paged<DP, 1, 8, false>(a, batch, beams, 1, s);
    }
    // 32 rows at a time
    return launch_paged<DP, 2, 4, false>(a, batch, beams, 1, s);
  } else {
    // Registers leave room for one wavefront per SIMD: four to a problem, or two where there are many: heads of 256, 52 sequences on 32 after 3 keys 40.3 us / 24.0, after 1000 164 / 151, 64 on 8 of 192
    // after 60 12.5 / 8.0; but 40 on 8 of 192 after 3000 71.4 / 89.6, one on 8 after 8000 21.0 / 23.4.
    return batch * a.kv_heads >= 512 ? launch_paged<DP, 1, 2, false>(a, batch, beams, 1, s) : launch_paged<DP, 1, 4, false>(a, batch, beams, 1, s);
  }
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
              static_cast<unsigned>(page), 0, 0, static_cast<unsigned>(columns * page < INT32_MAX ? columns * page : INT32_MAX), columns, scale == 0.f ? 1.f : fabsf(scale) * 1.4426950408889634f, static_cast<half_t>(scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d % 8 == 0 && page % 16 == 0 && pages > 0 && aligned(Q, 16) && aligned(K_pages, 16) && aligned(V_pages, 16) && aligned(out, 16)) {
    // 2^31 <= 2^(32 + shift) / page, rounded up, < 2^32: off by less than 1 in 2^31 page
    while ((int64_t{1} << (a.shift + 1)) < page) ++a.shift;
    a.magic = static_cast<unsigned>(((uint64_t{1} << (32 + a.shift)) + page - 1) / page);
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
