// Requests served together from one pool of pages, for gfx950: pages and slots for the rows that join, the rows into their slots, and the tables, lengths and
// part-filled pages of the beams that were chosen.  What lies in the buffers of indices is checked against its range wherever it is used.
#include "gemm_common.h"

namespace dtas {
namespace {

// Sums over the threads up to this one; sums past 2^32 - 1 stay there (a sequence that far behind is not served either way).
__device__ __forceinline__ unsigned add_sat(unsigned a, unsigned b) { return __builtin_elementwise_add_sat(a, b); }
template <int CTRL, int MASK>
__device__ __forceinline__ unsigned add_dpp(unsigned v) {
  return add_sat(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, MASK, 0xf, true)));
}
__device__ __forceinline__ unsigned upto_in_wave(unsigned v) {
  v = add_dpp<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
  v = add_dpp<0x112, 0xf>(v);
  v = add_dpp<0x114, 0xf>(v);
  v = add_dpp<0x118, 0xf>(v);
  v = add_dpp<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
  v = add_dpp<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}
// (every thread calls; `slots`: a float's room per wavefront; `total` becomes the sum of all)
template <int THREADS>
__device__ __forceinline__ unsigned upto_in_block(unsigned v, unsigned* slots, unsigned& total) {
  const int wave = threadIdx.x >> 6;
  v = upto_in_wave(v);
  __syncthreads();  // (what the last call left has been read)
  if ((threadIdx.x & 63) == 63) slots[wave] = v;
  __syncthreads();
  unsigned before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w == wave) before = total;
    total = add_sat(total, slots[w]);
  }
  return add_sat(v, before);
}

// ---- pages and slots --------------------------------------------------------------------------------------------------
// A thread per sequence finds out what it needs and, from the sums over the sequences before it, whether the pool has it; then a thread per row looks up its sequence
// (packed rows: by halving the starts, which lie in the LDS) and its slot.  The row that begins a page writes it into the table, so that no two threads write one entry,
// and nobody reads an entry that this launch writes.  Every workgroup repeats the sums for itself: no hand-over between workgroups, whose
// trip through memory costs more than the sums of a thousand sequences.  3.5 to 4.2 us, a launch's time, for 64 sequences of a row; 5.7 for 16384 packed rows of 37.
struct AssignArgs {
  const int *lens, *count;
  int* table;
  const int *free, *free_count;
  int *starts, *slots, *new_lens, *left;
  int64_t batch;
  unsigned rows;
  int64_t columns;
  unsigned page;
  int pages;
};

template <int THREADS>
__global__ void __launch_bounds__(THREADS) page_assign_kernel(AssignArgs a, bool maps, bool settles) {
  __shared__ unsigned begin[THREADS], base[THREADS], slots[THREADS / 64];
  __shared__ int length[THREADS], held[THREADS];  // (held: columns in use before; -1: not served)
  __shared__ unsigned joins[THREADS];
  __shared__ unsigned most_taken;
  const unsigned tid = threadIdx.x;
  const bool packed = a.starts != nullptr, first = blockIdx.x == 0;
  const int stack = *a.free_count;
  const unsigned there = stack < 0 ? 0u : stack > a.pages ? static_cast<unsigned>(a.pages) : static_cast<unsigned>(stack);
  const int64_t room = a.columns * a.page;
  unsigned asked_before = 0, needed_before = 0;
  if (tid == 0) most_taken = 0;
  for (int64_t c = 0; c < a.batch; c += THREADS) {
    const int64_t b = c + tid;
    const int len = b < a.batch ? a.lens[b] : -1, cnt = b < a.batch ? a.count[b] : 0;
    const unsigned asked = cnt > 0 ? cnt : 0;
    unsigned behind = asked, total = 0;
    if (packed) {
      behind = add_sat(asked_before, upto_in_block<THREADS>(asked, slots, total));
      begin[tid] = behind == ~0u ? ~0u : behind - asked;
      if (settles && first && b < a.batch) {
        const unsigned from = behind - asked;  // (a sum past the type's end: the rest of the starts say 2^31 - 1)
        a.starts[b] = behind == ~0u || from > 0x7fffffffu ? 0x7fffffff : static_cast<int>(from);
        if (b == a.batch - 1) a.starts[a.batch] = behind > 0x7fffffffu ? 0x7fffffff : static_cast<int>(behind);
      }
    }
    const int64_t all = static_cast<int64_t>(len) + static_cast<int64_t>(asked);
    const bool fits = len >= 0 && cnt >= 0 && all <= room && all <= INT32_MAX && behind <= a.rows;
    const unsigned have = len > 0 ? (static_cast<unsigned>(len) + a.page - 1) / a.page : 0u;
    const unsigned need = fits ? (static_cast<unsigned>(all) + a.page - 1) / a.page - have : 0u;
    unsigned needed = 0;
    const unsigned upto = add_sat(needed_before, upto_in_block<THREADS>(need, slots, needed));
    const bool served = fits && (need == 0 || upto <= there);
    base[tid] = upto - need;
    length[tid] = len;
    held[tid] = served ? static_cast<int>(have) : -1;
    joins[tid] = asked;
    if (served && need > 0) atomicMax(&most_taken, upto);
    if (settles && first && b < a.batch) a.new_lens[b] = served ? static_cast<int>(all) : len;
    const unsigned asked_upto = add_sat(asked_before, total);
    __syncthreads();
    if (maps) {
      const unsigned here = a.batch - c < THREADS ? static_cast<unsigned>(a.batch - c) : THREADS;
      const unsigned from = packed ? asked_before : static_cast<unsigned>(c) * a.rows, to = packed ? asked_upto < a.rows ? asked_upto : a.rows : from + here * a.rows;
      for (unsigned r = from + blockIdx.x * THREADS + tid; r < to; r += gridDim.x * THREADS) {
        unsigned i, t;
        if (packed) {  // the last sequence that begins at this row or before
          unsigned low = 0, high = here;
          while (high - low > 1) {
            const unsigned mid = (low + high) / 2;
            if (begin[mid] <= r) low = mid;
            else high = mid;
          }
          i = low;
          t = r - begin[i];
        } else {
          i = (r - from) / a.rows;
          t = (r - from) - i * a.rows;
        }
        int slot = -1;
        if (held[i] >= 0 && t < joins[i]) {
          const unsigned at = static_cast<unsigned>(length[i]) + t, column = at / a.page, in_page = at - column * a.page;
          int* entry = a.table + (c + i) * a.columns + column;
          int page;
          if (column >= static_cast<unsigned>(held[i])) {
            page = a.free[there - 1 - (base[i] + (column - static_cast<unsigned>(held[i])))];
            if (in_page == 0) *entry = page;
          } else {
            page = *entry;
          }
          if (page >= 0 && page < a.pages) slot = static_cast<int>(static_cast<unsigned>(page) * a.page + in_page);
        }
        a.slots[r] = slot;
      }
    }
    __syncthreads();
    asked_before = asked_upto;
    needed_before = add_sat(needed_before, needed);
  }
  if (maps && packed)
    for (uint64_t r = static_cast<uint64_t>(asked_before) + blockIdx.x * THREADS + tid; r < a.rows; r += gridDim.x * THREADS) a.slots[r] = -1;
  if (settles && first && tid == 0) {
    *a.left = static_cast<int>(there - most_taken);
    if (packed && a.batch == 0) a.starts[0] = 0;
  }
}

// ---- rows into their slots ----------------------------------------------------------------------------------------------
// A workgroup has `run` rows of one layer, of K and of V, in 16-byte pieces (or elements): a row of all key heads at least, two pieces per thread and turn.
// 2047 packed rows of 32 heads of 80 (42 MB read and written): 8.4 us, 5.0 TB/s, the rate of a large copy; 64 rows: 3.2 to 3.8 us, a launch's time.
template <typename U>
__global__ void __launch_bounds__(256) page_append_kernel(const U* __restrict__ K, const U* __restrict__ V, const int* __restrict__ slots, U* __restrict__ Kp,
                                                          U* __restrict__ Vp, int64_t rows, int kv_heads, int per_row, unsigned page, int64_t pages, int run, unsigned runs) {
  const int64_t l = blockIdx.x / runs, n0 = static_cast<int64_t>(blockIdx.x % runs) * run;
  const int64_t here = rows - n0 < run ? rows - n0 : run;
  const unsigned row = static_cast<unsigned>(kv_heads) * per_row, all = static_cast<unsigned>(here) * row, head = page * static_cast<unsigned>(per_row);
  const U* from_k = K + (l * rows + n0) * row;
  const U* from_v = V + (l * rows + n0) * row;
  U* to_k = Kp + l * pages * kv_heads * head;
  U* to_v = Vp + l * pages * kv_heads * head;
  for (unsigned t = threadIdx.x; t < all; t += 256) {
    const unsigned i = t / row, in_row = t - i * row, h = in_row / static_cast<unsigned>(per_row), e = in_row - h * per_row;
    const int slot = slots[n0 + i];
    if (slot < 0 || slot >= pages * page) continue;
    const unsigned p = static_cast<unsigned>(slot) / page, in_page = static_cast<unsigned>(slot) - p * page;
    const int64_t sink = (static_cast<int64_t>(p) * kv_heads + h) * head + in_page * static_cast<unsigned>(per_row) + e;
    const U k = from_k[t], v = from_v[t];
    to_k[sink] = k;
    to_v[sink] = v;
  }
}

// ---- tables of the beams that were chosen --------------------------------------------------------------------------------
// A workgroup per group, its wavefronts with a range of columns each, S >= beams lanes (a power of two) to a column: lane w reads the old entry of row w, takes its
// parent's from that lane, and compares its own with all others: what no parent names goes onto the stack, once.  Where on the stack is known when all groups have
// counted: the pages wait in the workspace, and whoever is last among the workgroups puts them down in their order, and takes the pages for copies from the top
// (in this order: a pool that has a page too few for the moment would lose a row otherwise).  The copies are a second launch.
// What binds are trips to memory, one behind the other: lengths, entries, the arrival, the lists' sizes, the lists: 4.9 us for one group of 4 beams, 7.8 for 24 of 8 (18.8 with a
// wavefront per list of pages in settle_pool instead of a thread per page).
struct ReorderArgs {
  const int *parents, *table, *lens;
  int* free;
  const int* free_count;
  int *new_table, *new_lens, *left;
  int64_t groups, columns;
  int beams, shift;  // S = 1 << shift
  unsigned page;
  int pages, waves;
  int64_t share;     // entries of `back` per wavefront
  int* back;         // [groups][waves][share]: pages given back by a wavefront's columns, in their order
  unsigned* backs;   // [groups][waves]: how many
  uint64_t* wanted;  // [groups][beams]: a row that takes a copy: its length << 32 | the page; ~0: none
  int* copies;       // [groups * beams][4]: page, its copy, rows
  unsigned* count;   // how many
  unsigned* arrivals;
};
template <typename T>
__device__ __forceinline__ void put(T* at, T v) { __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename T>
__device__ __forceinline__ T get(const T* at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned most_dpp(unsigned v) {
  const unsigned o = static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, true));
  return v > o ? v : o;
}
__device__ __forceinline__ unsigned most_in_wave(unsigned v) {
  v = most_dpp<0x118, 0xf>(most_dpp<0x114, 0xf>(most_dpp<0x112, 0xf>(most_dpp<0x111, 0xf>(v))));  // row_shr:1, 2, 4, 8
  return static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(most_dpp<0x143, 0xc>(most_dpp<0x142, 0xa>(v))), 63));
}

constexpr int kReorderThreads = 1024;
static_assert(DTAS_MAX_BEAMS <= 32, "a bit of a word for each");
__device__ void settle_pool(const ReorderArgs& a) {
  __shared__ unsigned slots[kReorderThreads / 64], before[kReorderThreads];
  __shared__ int top[kReorderThreads];  // (what was put down last, by its place in the stack)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nwaves = blockDim.x >> 6;
  const int64_t threads = blockDim.x;
  const int stack = *a.free_count;
  const uint64_t old_height = stack < 0 ? 0 : stack > a.pages ? a.pages : stack;
  uint64_t height = old_height;
  const int64_t rows = a.groups * a.beams;
  const uint64_t first_wanted = tid < rows ? get(a.wanted + tid) : ~uint64_t{0};  // (with the lists' sizes, in one trip)
  auto upto = [&](unsigned v, unsigned& total) {  // (a workgroup of any number of wavefronts)
    v = upto_in_wave(v);
    __syncthreads();
    if (lane == 63) slots[wave] = v;
    __syncthreads();
    unsigned front = 0;
    total = 0;
    for (int w = 0; w < nwaves; ++w) {
      if (w == wave) front = total;
      total = add_sat(total, slots[w]);
    }
    return add_sat(v, front);
  };
  const int64_t segments = a.groups * a.waves;
  for (int64_t c = 0; c < segments; c += threads) {
    const unsigned n = c + tid < segments ? get(a.backs + c + tid) : 0u;
    unsigned total;
    const unsigned behind = upto(n, total);
    before[tid] = behind - n;
    __syncthreads();
    // a thread per page: the last list that begins at it or before (an empty one begins where the next does)
    const unsigned lists = segments - c < threads ? static_cast<unsigned>(segments - c) : static_cast<unsigned>(threads);
    for (unsigned j = tid; j < total; j += static_cast<unsigned>(threads)) {
      unsigned low = 0, high = lists;
      while (high - low > 1) {
        const unsigned mid = (low + high) / 2;
        if (before[mid] <= j) low = mid;
        else high = mid;
      }
      if (height + j < static_cast<uint64_t>(a.pages)) {
        const int page = get(a.back + (c + low) * a.share + (j - before[low]));
        put(a.free + height + j, page);
        if (total - j <= kReorderThreads) top[(height + j) % kReorderThreads] = page;
      }
    }
    height += total;
    __syncthreads();
  }
  bool drained = false;
  auto drain = [&] {
    if (drained) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    drained = true;
  };
  if (height > static_cast<uint64_t>(a.pages)) {  // (more pages than there are: some table names one that is not its own)
    height = a.pages;
    drain();
  }
  uint64_t taken = 0;
  for (int64_t c = 0; c < rows; c += threads) {
    const int64_t r = c + tid;
    if (taken + threads > kReorderThreads) drain();
    const uint64_t one = c == 0 ? first_wanted : r < rows ? get(a.wanted + r) : ~uint64_t{0};
    const bool copy = one != ~uint64_t{0};
    unsigned total;
    const unsigned behind = upto(copy ? 1u : 0u, total);
    if (copy) {
      const uint64_t k = taken + behind - 1;
      const unsigned len = static_cast<unsigned>(one >> 32);
      const uint64_t place = height - 1 - k;
      const int to = k >= height ? -1 : drained || place < old_height ? get(a.free + place) : top[place % kReorderThreads];
      const bool good = to >= 0 && to < a.pages;
      a.new_lens[r] = good ? static_cast<int>(len) : -1;
      if (good) a.new_table[r * a.columns + len / a.page] = to;
      if (k < height) {
        a.copies[4 * k] = static_cast<int>(one & 0xffffffffu);
        a.copies[4 * k + 1] = to;
        a.copies[4 * k + 2] = good ? static_cast<int>(len % a.page) : 0;
      }
    }
    taken += total;
  }
  if (tid == 0) {
    const uint64_t n = taken < height ? taken : height;
    *a.count = static_cast<unsigned>(n);
    *a.left = static_cast<int>(height - n);
  }
}

__global__ void __launch_bounds__(kReorderThreads) page_reorder_kernel(ReorderArgs a) {
  __shared__ uint64_t copy[DTAS_MAX_BEAMS];
  __shared__ int flag, front[DTAS_MAX_BEAMS];  // (the first row of each parent)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int S = 1 << a.shift, w = lane & (S - 1), sub = lane >> a.shift, first = lane - w;
  const int64_t g = blockIdx.x, room = a.columns * a.page;
  const bool row = w < a.beams;
  const int raw = row ? a.lens[g * a.beams + w] : 0, parent = row ? a.parents[g * a.beams + w] : -1;
  const unsigned len = raw < 0 ? 0u : raw > room ? static_cast<unsigned>(room) : static_cast<unsigned>(raw);
  const unsigned named = (len + a.page - 1) / a.page;
  const bool has = parent >= 0 && parent < a.beams;
  const int from = first + (has ? parent : 0);
  const unsigned their_len = __shfl(len, from), their_named = __shfl(named, from), new_len = has ? their_len : 0u, new_named = has ? their_named : 0u;
  if (tid < DTAS_MAX_BEAMS) {
    copy[tid] = ~uint64_t{0};
    front[tid] = DTAS_MAX_BEAMS;
  }
  __syncthreads();
  if (wave == 0 && sub == 0 && has) atomicMin(&front[parent], w);
  __syncthreads();  // (also: the lengths have been read)
  const bool later = has && front[parent] < w;  // (a row of the same parent stands in front)
  const unsigned followed = static_cast<unsigned>(__builtin_amdgcn_ballot_w64(row && front[w] < DTAS_MAX_BEAMS)) & (S == 32 ? ~0u : (1u << S) - 1u);  // rows that are a parent
  const bool part_filled = has && later && new_len % a.page != 0;
  const unsigned most = most_in_wave(named);
  // this wavefront's columns
  const unsigned per = (most + a.waves - 1) / a.waves, lo = per * wave < most ? per * wave : most, hi = lo + per < most ? lo + per : most;
  const int* old = a.table + (g * a.beams + (row ? w : 0)) * a.columns;
  int* fresh = a.new_table + (g * a.beams + (row ? w : 0)) * a.columns;
  int* back = a.back + (g * a.waves + wave) * a.share;
  unsigned given = 0;
  const unsigned step = 64u >> a.shift;
  auto read = [&](unsigned c) { return row && c < hi && c < named ? old[c] : -1; };
  int entry = read(lo + sub);
  for (unsigned c0 = lo; c0 < hi; c0 += step) {
    const unsigned c = c0 + sub;
    const int next = read(c + step);
    const int theirs = __shfl(entry, from);
    const bool mine = has && c < hi && c < new_named;
    bool kept = false, again = false;  // (a row that is a parent names the same page; a row in front does)
#pragma unroll 4
    for (int i = 0; i < a.beams; ++i) {
      const bool same = __shfl(entry, first + i) == entry;
      kept = kept || (same && ((followed >> i) & 1) != 0);
      again = again || (same && i < w);
    }
    const bool give = entry >= 0 && entry < a.pages && !kept && !again;
    const uint64_t all = __builtin_amdgcn_ballot_w64(give);
    if (give) put(back + given + __builtin_popcountll(all & ((uint64_t{1} << lane) - 1)), entry);
    given += __builtin_popcountll(all);
    if (mine) {
      if (part_filled && c == new_len / a.page && theirs >= 0 && theirs < a.pages) copy[w] = static_cast<uint64_t>(new_len) << 32 | static_cast<unsigned>(theirs);
      else fresh[c] = theirs;
    }
    entry = next;
  }
  if (lane == 0 && wave < a.waves) put(a.backs + g * a.waves + wave, given);
  __syncthreads();
  if (wave == 0 && row && sub == 0) {
    const uint64_t one = copy[w];
    put(a.wanted + g * a.beams + w, one);
    if (one == ~uint64_t{0}) a.new_lens[g * a.beams + w] = static_cast<int>(new_len);
  }
  // whoever is last: what the others left has drained before it is counted
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const unsigned before = __hip_atomic_fetch_add(a.arrivals, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    flag = before == gridDim.x - 1;
    if (flag) put(a.arrivals, 0u);  // re-armed for the next launch
  }
  __syncthreads();
  if (flag) settle_pool(a);
}

// without a row the stack's height is handed on, as far as the stack can be that high
__global__ void stack_height_kernel(const int* free_count, int* left, int pages) {
  const int stack = *free_count;
  *left = stack < 0 ? 0 : stack > pages ? pages : stack;
}

// The copies: a wavefront per copy, layer, key head and K or V, four pieces per lane on their way at a time.  24 groups of 8 beams, 16 layers of 8 heads of 128, pages of 32 (95 MB
// read and written): 24 us of the call's 31 to 34 (when that was 33.7, eight pieces: 35.3; four times the workgroups: 1 us more; loads and stores past the L2: 2 more; a workgroup for all heads of K and V: 29).
template <typename U>
__global__ void __launch_bounds__(256) page_copy_kernel(U* __restrict__ Kp, U* __restrict__ Vp, const int* __restrict__ copies, const unsigned* __restrict__ count,
                                                        unsigned layers, int64_t pages, unsigned kv_heads, unsigned per_row, unsigned page) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint64_t each = uint64_t{2} * kv_heads * layers, items = *count * each, head = static_cast<uint64_t>(page) * per_row;
  for (uint64_t item = static_cast<uint64_t>(blockIdx.x) * 4 + wave; item < items; item += static_cast<uint64_t>(gridDim.x) * 4) {
    const uint64_t k = item / each, of = item - k * each;  // (neighbours: the heads of a page)
    const uint64_t tensor = of / (each / 2), l = (of - tensor * (each / 2)) / kv_heads, h = of % kv_heads;
    const int from = copies[4 * k], to = copies[4 * k + 1];
    const unsigned some = static_cast<unsigned>(copies[4 * k + 2]) * per_row;
    U* base = tensor ? Vp : Kp;
    const U* source = base + ((l * pages + from) * kv_heads + h) * head;
    U* sink = base + ((l * pages + to) * kv_heads + h) * head;
    constexpr int kAhead = 4;
    unsigned t = lane;
    for (; t + (kAhead - 1) * 64 < some; t += kAhead * 64) {
      U v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) v[u] = source[t + u * 64];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) sink[t + u * 64] = v[u];
    }
    U v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (t + u * 64 < some) v[u] = source[t + u * 64];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (t + u * 64 < some) sink[t + u * 64] = v[u];
  }
}

struct Span { const void* at; int64_t bytes; };
// outputs against inputs and against each other; an output may be the input that `same` names
template <int IN, int OUT>
int check_spans(const char* what, const Span (&in)[IN], const Span (&out)[OUT], const void* const (&same)[OUT]) {
  for (int i = 0; i < OUT; ++i) {
    if (!out[i].at) continue;
    for (const Span& o : in)
      if (o.at && !(o.at == same[i] && o.at == out[i].at) && overlaps(out[i].at, out[i].bytes, o.at, o.bytes)) return fail("%s: output overlaps an input", what);
    for (int j = 0; j < i; ++j)
      if (out[j].at && overlaps(out[i].at, out[i].bytes, out[j].at, out[j].bytes)) return fail("%s: the outputs overlap", what);
  }
  return 0;
}
constexpr int64_t kMost = int64_t{1} << 60;

}  // namespace
}  // namespace dtas

extern "C" int dtas_page_assign_i32(const void* lens, const void* count, void* table, const void* free, const void* free_count, void* starts, void* slots,
                                    void* new_lens, void* left, int64_t batch, int64_t rows, int64_t columns, int64_t page, int64_t pages, void* stream) {
  using namespace dtas;
  clear_error();
  if (batch < 0 || rows < 0 || columns < 0 || pages < 0)
    return fail("page_assign: negative extent batch=%lld rows=%lld columns=%lld pages=%lld", (long long)batch, (long long)rows, (long long)columns, (long long)pages);
  if (page < 1) return fail("page_assign: a page holds at least one position, got %lld", (long long)page);
  if (batch > INT32_MAX || rows > INT32_MAX || columns > INT32_MAX || page > INT32_MAX || pages > INT32_MAX / page || (!starts && rows > 0 && batch > INT32_MAX / rows) ||
      (columns > 0 && batch > kMost / columns))
    return fail("page_assign: the extents overflow");
  const int64_t all = starts ? rows : batch * rows;
  if (!free_count || !left) return fail("page_assign: NULL buffer");
  if (batch > 0 && (!lens || !count || !new_lens || (columns > 0 && !table))) return fail("page_assign: NULL buffer");
  if ((pages > 0 && !free) || (all > 0 && !slots)) return fail("page_assign: NULL buffer");
  const Span in[] = {{lens, batch * 4}, {count, batch * 4}, {free, pages * 4}, {free_count, 4}};
  const Span out[] = {{table, batch * columns * 4}, {starts, starts ? (batch + 1) * 4 : 0}, {slots, all * 4}, {new_lens, batch * 4}, {left, 4}};
  if (check_spans("page_assign", in, out, {nullptr, nullptr, nullptr, lens, free_count}) != 0) return -1;
  AssignArgs a{static_cast<const int*>(lens), static_cast<const int*>(count), static_cast<int*>(table), static_cast<const int*>(free), static_cast<const int*>(free_count),
               static_cast<int*>(starts), static_cast<int*>(slots), static_cast<int*>(new_lens), static_cast<int*>(left), batch, static_cast<unsigned>(rows), columns,
               static_cast<unsigned>(page), static_cast<int>(pages)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  constexpr int kThreads = 1024;
  const unsigned groups = all <= 8 * kThreads ? 1u : static_cast<unsigned>(all / (2 * kThreads) < 64 ? ceil_div(all, 2 * kThreads) : 64);
  // Several workgroups read the lengths and the stack's height: where the new ones take their place, a launch behind them writes those
  const bool apart = groups > 1 && (new_lens == lens || left == free_count);
  hipLaunchKernelGGL(page_assign_kernel<kThreads>, dim3(groups), dim3(kThreads), 0, s, a, true, !apart);
  if (check_launch("page_assign") != 0 || !apart) return check_launch("page_assign");
  hipLaunchKernelGGL(page_assign_kernel<kThreads>, dim3(1), dim3(kThreads), 0, s, a, false, true);
  return check_launch("page_assign");
}

extern "C" int dtas_page_append_f16(const void* K, const void* V, const void* slots, void* K_pages, void* V_pages, int64_t layers, int64_t rows, int64_t kv_heads,
                                    int64_t d, int64_t page, int64_t pages, void* stream) {
  using namespace dtas;
  clear_error();
  if (layers < 0 || rows < 0 || kv_heads < 0 || d < 0 || page < 0 || pages < 0)
    return fail("page_append: negative extent layers=%lld rows=%lld kv_heads=%lld d=%lld page=%lld pages=%lld", (long long)layers, (long long)rows, (long long)kv_heads,
                (long long)d, (long long)page, (long long)pages);
  if (layers == 0 || rows == 0 || kv_heads == 0 || d == 0 || page == 0 || pages == 0) return 0;
  if (rows > INT32_MAX || kv_heads > INT32_MAX || d > INT32_MAX || pages > INT32_MAX / page || kv_heads * d > INT32_MAX / 2 || page * d > INT32_MAX ||
      layers > kMost / kv_heads / d / (pages * page) || layers > kMost / kv_heads / d / rows)
    return fail("page_append: the extents overflow");
  if (!K || !V || !slots || !K_pages || !V_pages) return fail("page_append: NULL buffer");
  const int64_t new_bytes = layers * rows * kv_heads * d * 2, page_bytes = layers * pages * kv_heads * page * d * 2;
  const Span in[] = {{K, new_bytes}, {V, new_bytes}, {slots, rows * 4}}, out[] = {{K_pages, page_bytes}, {V_pages, page_bytes}};
  if (check_spans("page_append", in, out, {nullptr, nullptr}) != 0) return -1;
  const bool wide = d % 8 == 0 && aligned(K, 16) && aligned(V, 16) && aligned(K_pages, 16) && aligned(V_pages, 16);
  const int64_t per_row = wide ? d / 8 : d, row = kv_heads * per_row, run = row >= 256 ? 1 : 256 / row, runs = ceil_div(rows, run);
  // as many layers, or runs of one layer, to a launch as a grid holds: less than 2^32 threads
  constexpr int64_t kMostRuns = int64_t{1} << 23;
  const int64_t some_layers = runs < kMostRuns ? kMostRuns / runs : 1, some_rows = runs < kMostRuns ? rows : kMostRuns * run;
  auto go = [&](auto* tag) {
    using U = std::remove_pointer_t<decltype(tag)>;
    for (int64_t l = 0; l < layers; l += some_layers)
      for (int64_t n = 0; n < rows; n += some_rows) {
        const int64_t here = layers - l < some_layers ? layers - l : some_layers, rows_here = rows - n < some_rows ? rows - n : some_rows, runs_here = ceil_div(rows_here, run);
        const int64_t from = (l * rows + n) * row, to = l * pages * page * row;
        hipLaunchKernelGGL(page_append_kernel<U>, dim3(static_cast<unsigned>(here * runs_here)), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const U*>(K) + from,
                           static_cast<const U*>(V) + from, static_cast<const int*>(slots) + n, static_cast<U*>(K_pages) + to, static_cast<U*>(V_pages) + to, rows_here,
                           static_cast<int>(kv_heads), static_cast<int>(per_row), static_cast<unsigned>(page), pages, static_cast<int>(run), static_cast<unsigned>(runs_here));
        if (check_launch("page_append") != 0) return -1;
      }
    return 0;
  };
  return wide ? go(static_cast<u32x4*>(nullptr)) : go(static_cast<half_t*>(nullptr));
}

extern "C" int dtas_page_reorder_f16(const void* parents, const void* table, const void* lens, void* free, const void* free_count, void* new_table, void* new_lens,
                                     void* left, void* K_pages, void* V_pages, int64_t layers, int64_t groups, int64_t beams, int64_t columns, int64_t kv_heads,
                                     int64_t d, int64_t page, int64_t pages, void* stream) {
  using namespace dtas;
  clear_error();
  if (layers < 0 || groups < 0 || beams < 0 || columns < 0 || kv_heads < 0 || d < 0 || pages < 0)
    return fail("page_reorder: negative extent layers=%lld groups=%lld beams=%lld columns=%lld kv_heads=%lld d=%lld pages=%lld", (long long)layers, (long long)groups,
                (long long)beams, (long long)columns, (long long)kv_heads, (long long)d, (long long)pages);
  if (page < 1) return fail("page_reorder: a page holds at least one position, got %lld", (long long)page);
  if (beams > DTAS_MAX_BEAMS) return fail("page_reorder: up to %d beams, got %lld", DTAS_MAX_BEAMS, (long long)beams);
  if (layers > INT32_MAX || groups > INT32_MAX / DTAS_MAX_BEAMS || columns > INT32_MAX || page > INT32_MAX || pages > INT32_MAX / page || kv_heads > INT32_MAX || d > INT32_MAX ||
      (columns > 0 && groups > kMost / DTAS_MAX_BEAMS / columns) || (d > 0 && page * d > INT32_MAX) ||
      (layers > 0 && kv_heads > 0 && d > 0 && pages > 0 && layers > kMost / kv_heads / d / (pages * page)))
    return fail("page_reorder: the extents overflow");
  // a step of a wavefront's columns, two from eight wavefronts on, and the 32-bit words of the workspace: wanted, copies, backs, back, the count
  int shift = 0;
  while ((1 << shift) < beams) ++shift;
  const int64_t steps = ceil_div(columns << shift, 64), waves = steps < 2 ? 1 : steps < 8 ? steps : steps < 16 ? 8 : steps / 2 < kReorderThreads / 64 ? steps / 2 : kReorderThreads / 64;
  const int64_t share = ceil_div(columns, waves) * beams, lists = groups * beams * 6 + groups * waves * (share + 1) + 2;
  if (lists > (int64_t{1} << 28)) return fail("page_reorder: tables of %lld entries are too large", (long long)(groups * beams * columns));
  const int64_t rows = groups * beams, page_bytes = layers * pages * kv_heads * page * d * 2;
  if (!free_count || !left || (pages > 0 && !free) || (rows > 0 && (!parents || !lens || !new_lens)) || (rows > 0 && columns > 0 && (!table || !new_table)) ||
      (page_bytes > 0 && (!K_pages || !V_pages)))
    return fail("page_reorder: NULL buffer");
  const Span in[] = {{parents, rows * 4}, {table, rows * columns * 4}, {lens, rows * 4}, {free_count, 4}};
  const Span out[] = {{new_table, rows * columns * 4}, {new_lens, rows * 4}, {left, 4}, {free, pages * 4}, {K_pages, page_bytes}, {V_pages, page_bytes}};
  if (check_spans("page_reorder", in, out, {table, lens, free_count, nullptr, nullptr, nullptr}) != 0) return -1;
  ReorderArgs a{static_cast<const int*>(parents), static_cast<const int*>(table), static_cast<const int*>(lens), static_cast<int*>(free),
                static_cast<const int*>(free_count), static_cast<int*>(new_table), static_cast<int*>(new_lens), static_cast<int*>(left), groups, columns,
                static_cast<int>(beams), 0, static_cast<unsigned>(page), static_cast<int>(pages), 1, 0, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows == 0) {  // (nothing to sort out, and no workspace to do it in)
    if (left == free_count) return 0;
    hipLaunchKernelGGL(stack_height_kernel, dim3(1), dim3(1), 0, s, a.free_count, a.left, a.pages);
    return check_launch("page_reorder");
  }
  a.shift = shift;
  a.waves = static_cast<int>(waves);
  a.share = share;
  float* room = nullptr;
  std::unique_lock<std::recursive_mutex> lock;
  if (split_scratch(s, static_cast<size_t>(lists) * 4, 1, 1, &room, &a.arrivals, &lock) != 0) return -1;
  a.wanted = reinterpret_cast<uint64_t*>(room);
  a.copies = reinterpret_cast<int*>(room) + 2 * rows;
  a.count = reinterpret_cast<unsigned*>(room) + 6 * rows;
  a.backs = a.count + 2;
  a.back = reinterpret_cast<int*>(a.backs + groups * a.waves);
  // Whoever settles the pool has use for more wavefronts than the columns have, where there are many groups; but a launch has less than 2^32 threads.  (Those of the columns always fit: n of them, n > 1, take
  // more than 32 (n - 1) entries of a group's lists, one takes 8 words, and the lists are limited above.)
  const int64_t useful = groups * waves < 8 ? groups * waves : 8, fit = ((int64_t{1} << 32) - 1) / groups / 64, spare = useful < fit ? useful : fit;
  const unsigned threads = 64u * static_cast<unsigned>(waves > spare ? waves : spare);
  hipLaunchKernelGGL(page_reorder_kernel, dim3(static_cast<unsigned>(groups)), dim3(threads), 0, s, a);
  if (check_launch("page_reorder") != 0) return -1;
  if (beams < 2 || page_bytes == 0 || page == 1) return 0;
  const int64_t most = groups * (beams - 1), each = 2 * layers * kv_heads;  // copies at most, and a copy's items
  const unsigned grid = each < 8192 / most ? static_cast<unsigned>(ceil_div(most * each, 4)) : 2048;
  const bool wide = d % 8 == 0 && aligned(K_pages, 16) && aligned(V_pages, 16);
  auto go = [&](auto* tag) {
    using U = std::remove_pointer_t<decltype(tag)>;
    hipLaunchKernelGGL(page_copy_kernel<U>, dim3(grid), dim3(256), 0, s, static_cast<U*>(K_pages), static_cast<U*>(V_pages), a.copies, a.count,
                       static_cast<unsigned>(layers), pages, static_cast<unsigned>(kv_heads), static_cast<unsigned>(wide ? d / 8 : d), static_cast<unsigned>(page));
  };
  if (wide) go(static_cast<u32x4*>(nullptr));
  else go(static_cast<half_t*>(nullptr));
  return check_launch("page_reorder");
}
