// Drafted tokens against the target's probabilities, and what is accepted into the key/value cache, for gfx950.
#include "gemm_common.h"

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
//
// What happens at a node does not depend on the way there: a workgroup per node finds out which child is accepted there, or the token behind it, and
// whoever is last among a sequence's workgroups follows the path.  Nodes that cannot be on it are left out beforehand: the first child of a node
// is settled by accept * q < p alone, and a later one (c >= 1 by then) is out of the question where its first brother is accepted or p <= q.  So the rows that
// are read are few more than those of the path (32 trees of 31 nodes over 50280 tokens: 68 us with a workgroup per tree that walked it).
constexpr int kVerifyThreads = 1024, kVerifyWaves = kVerifyThreads / 64;

// sums over the lanes up to this one, on the DPP datapath (through the LDS crossbar the six steps take six times as long); ROWS: of 16 lanes each, or of all
template <int CTRL, int MASK>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits), CTRL, MASK, 0xf, true);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits >> 32), CTRL, MASK, 0xf, true);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double lane64(double v, int lane) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const unsigned lo = __builtin_amdgcn_readlane(static_cast<int>(bits), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(bits >> 32), lane);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double upto16(double v) {
  v += dpp64<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
  v += dpp64<0x112, 0xf>(v);
  v += dpp64<0x114, 0xf>(v);
  v += dpp64<0x118, 0xf>(v);
  return v;
}
__device__ __forceinline__ double upto64(double v) {
  v = upto16(v);
  v += dpp64<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
  v += dpp64<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}

__device__ __forceinline__ double rest_of(float p, float q, double c) {
  const double w = fma(-c, static_cast<double>(q), static_cast<double>(p));
  return w > 0.0 ? w : 0.0;  // (NaN too)
}

// four consecutive probabilities (rows of an odd vocabulary begin off 16 bytes)
__device__ __forceinline__ f32x4 load4(const float* p) {
  f32x4 v;
  __builtin_memcpy(&v, __builtin_assume_aligned(p, 4), 16);
  return v;
}

// The sum of max(p - c q, 0) over [from, to), by one wavefront; q is not read where c is 0.  `from` is a multiple of 4 of the row, and so is `to` unless it
// is the row's end.  A refusal, a pass of a workgroup over both rows of 50280 tokens, takes 4.4 us: a CU draws them from its
// L2 in 3.7 (with a maximum in the place of the sums), the 64-bit arithmetic alone takes 3.1, and with sums in fp32 it is 3.9.
__device__ __forceinline__ double sum_rest(const float* p, const float* q, double c, int64_t from, int64_t to, int lane) {
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  constexpr int kAtOnce = 3;
  for (int64_t base = from; base < to; base += 256 * kAtOnce) {
    f32x4 a[kAtOnce], b[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int64_t v = base + 256 * u + 4 * lane;
      const bool in = v + 4 <= to;
      a[u] = b[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (base + 256 * u >= to) continue;
      if (in) a[u] = load4(p + v);
      if (in && c != 0.0) b[u] = load4(q + v);
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (base + 256 * u >= to) break;
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += rest_of(a[u][j], b[u][j], c);
    }
  }
  const int64_t end = to - ((to - from) & 3) + lane;  // the last one to three
  if (end < to) s[0] += rest_of(p[end], c != 0.0 ? q[end] : 0.f, c);
  return lane64(upto64((s[0] + s[1]) + (s[2] + s[3])), 63);
}

struct VerifyArgs {
  const float *target, *draft;
  const int *tokens, *parents;
  const float *accept, *sample;
  int *path, *count, *next;
  int T;
  int64_t V;
  int* outcomes;       // [batch, T]: an accepted child, or -2 - the next token
  unsigned* arrivals;  // [batch]
};

__global__ void __launch_bounds__(kVerifyThreads) verify_tree_kernel(VerifyArgs a) {
  __shared__ float at_p[DTAS_MAX_TREE_NODES], at_q[DTAS_MAX_TREE_NODES], at_u[DTAS_MAX_TREE_NODES];
  __shared__ int eldest[DTAS_MAX_TREE_NODES];
  __shared__ uint64_t at_reach, at_mine;
  __shared__ double part[2][kVerifyWaves];
  __shared__ int flag;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, node = blockIdx.x, T = a.T;
  const int64_t b = blockIdx.y, V = a.V;
  // ---- the edges, and which nodes the walk can reach
  if (wave == 0) {
    const int parent = lane < T ? a.parents[b * T + lane] : -1, token = lane < T ? a.tokens[b * T + lane] : -1;
    const float u = lane < T ? a.accept[b * T + lane] : 0.f;
    const bool offered = lane > 0 && parent >= 0 && parent < lane && token >= 0 && token < V;
    const int above = offered ? parent : 0;
    const float p0 = offered ? a.target[(b * T + above) * V + token] : 0.f, q0 = offered ? a.draft[(b * T + above) * V + token] : 0.f;
    eldest[lane] = 64;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (offered) atomicMin(&eldest[above], lane);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int first = eldest[above];  // (of this lane's node and its brothers)
    at_p[lane] = p0;
    at_q[lane] = q0;
    at_u[lane] = u;
    const bool at_once = static_cast<double>(u) * static_cast<double>(q0) < static_cast<double>(p0 > 0.f ? p0 : 0.f);
    const uint64_t settled = __builtin_amdgcn_ballot_w64(offered && at_once);
    const bool can = offered && (first == lane ? at_once : !((settled >> (first & 63)) & 1) && p0 > q0);
    uint64_t reach = 1, fresh = 1;  // from node 0 on, a generation at a time
    while (fresh) {
      const uint64_t more = __builtin_amdgcn_ballot_w64(can && ((fresh >> above) & 1)) & ~reach;
      reach |= more;
      fresh = more;
    }
    const uint64_t mine = __builtin_amdgcn_ballot_w64(offered && parent == node);
    if (lane == 0) {
      at_reach = reach;
      at_mine = mine;
    }
  }
  __syncthreads();
  const uint64_t reach = at_reach;
  if (!((reach >> node) & 1)) return;
  uint64_t mine = at_mine;

  // ---- this node: its children in their order, then the token
  const float* p = a.target + (b * T + node) * V;
  const float* q = a.draft + (b * T + node) * V;
  int phase = 0;
  // the sums of the wavefronts' pieces of [lo, hi): lane w of a row of sixteen returns with piece w's
  auto sums = [&](double c, int64_t lo, int64_t piece, int64_t hi) -> double {
    const int64_t from = lo + wave * piece < hi ? lo + wave * piece : hi, to = from + piece < hi ? from + piece : hi;
    const double s = sum_rest(p, q, c, from, to, lane);
    double* bank = part[phase++ & 1];
    if (lane == 0) bank[wave] = s;
    __syncthreads();
    return bank[lane & 15];
  };
  static_assert(kVerifyWaves == 16, "a row of lanes");
  const int64_t whole = ((V + kVerifyWaves - 1) / kVerifyWaves + 3) / 4 * 4;
  int outcome = -1;
  bool accepted = false;
  double c = 0.0, left = 1.0;
  double pieces = 0.0;  // with the present c: lane w of sixteen holds the sum of piece w ...
  bool summed = false;
  for (; mine; mine &= mine - 1) {
    const int i = __builtin_ctzll(mine);
    if (static_cast<double>(at_u[i]) * static_cast<double>(at_q[i]) * left < rest_of(at_p[i], at_q[i], c)) {
      outcome = i;
      accepted = true;
      break;
    }
    c += left;
    pieces = sums(c, 0, whole, V);
    summed = true;
    left = lane64(upto16(pieces), 15);
  }
  if (!accepted) {
    if (!summed) pieces = sums(c, 0, whole, V);
    double total = lane64(upto16(pieces), 15);
    if (!(total > 0.0) && c != 0.0) {  // nothing is left of the target (its rows equal the draft's): the target itself
      c = 0.0;
      pieces = sums(c, 0, whole, V);
      total = lane64(upto16(pieces), 15);
    }
    if (total > 0.0) {  // (a row of zeros has no token: outcome -1)
      const double r = static_cast<double>(a.sample[b]), goal = (r > 0.0 ? r < 1.0 ? r : 1.0 : 0.0) * total;
      // the piece that the goal falls into: the first whose end lies behind it, or (where rounding leaves it behind all) the last with a sum
      int64_t lo = 0, hi = V, piece = whole;
      double base = 0.0;
      for (;;) {
        const double upto = upto16(pieces);
        const unsigned some = static_cast<unsigned>(__builtin_amdgcn_ballot_w64(pieces > 0.0)) & 0xffffu;
        const unsigned behind = static_cast<unsigned>(__builtin_amdgcn_ballot_w64(pieces > 0.0 && base + upto > goal)) & 0xffffu;
        const int at = behind ? __builtin_ctz(behind) : 31 - __builtin_clz(some | 1u);
        if (at > 0) base += lane64(upto, at - 1);
        lo += at * piece;
        hi = lo + piece < hi ? lo + piece : hi;
        if (hi - lo <= 256) break;
        piece = ((hi - lo + kVerifyWaves - 1) / kVerifyWaves + 3) / 4 * 4;
        pieces = sums(c, lo, piece, hi);
      }
      // four tokens a lane
      double w[4], mine4 = 0.0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t v = lo + 4 * lane + j;
        w[j] = v < hi ? rest_of(p[v], c != 0.0 ? q[v] : 0.f, c) : 0.0;
        mine4 += w[j];
      }
      const double upto = upto64(mine4);
      const uint64_t some = __builtin_amdgcn_ballot_w64(mine4 > 0.0), behind = __builtin_amdgcn_ballot_w64(mine4 > 0.0 && base + upto > goal);
      const int l = behind ? __builtin_ctzll(behind) : 63 - __builtin_clzll(some | 1);
      double before = base + (upto - mine4);
      int token_at = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (w[j] > 0.0 && !(token_at > 0 && before > goal)) token_at = j + 1;  // (the first whose end lies behind the goal, else the last with a weight)
        before += w[j];
      }
      outcome = -2 - static_cast<int>(lo + 4 * l + __shfl(token_at, l) - 1);
    }
  }

  // ---- whoever is last follows the path.  The outcomes pass the L2 (the XCDs' are not coherent); an arrival is counted once its own has drained
  if (tid == 0) {
    __hip_atomic_store(a.outcomes + b * T + node, outcome, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const unsigned arrived = __hip_atomic_fetch_add(a.arrivals + b, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    flag = arrived == static_cast<unsigned>(__builtin_popcountll(reach)) - 1;
    if (flag) __hip_atomic_store(a.arrivals + b, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // re-armed for the next launch
  }
  if (wave != 0) return;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if (!__builtin_amdgcn_readfirstlane(flag)) return;
  const int found = (reach >> lane) & 1 ? __hip_atomic_load(a.outcomes + b * T + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : -1;
  int at = 0, steps = 1, way = lane == 0 ? 0 : -1;
  for (;;) {
    const int o = __builtin_amdgcn_readlane(found, at);
    if (o < 1) {
      if (lane == 0) {
        a.next[b] = -2 - o;
        a.count[b] = steps;
      }
      break;
    }
    at = o;
    if (lane == steps) way = o;
    ++steps;
  }
  if (lane < T) a.path[b * T + lane] = way;
}

// ---- the accepted rows into the cache -------------------------------------------------------------------------------
// cache[l, b, h, lens[b] + j, :] = new[l, b, path[b, j], h, :] for j < count[b]; no path: all rows in their order.  Rows that would
// fall outside [0, capacity), and path entries outside [0, T), are left out.  A workgroup has `run` slots of one sequence and layer, of K and of V, in 16-byte
// pieces (or elements): what it needs to know of the sequence are scalars, and a workgroup behind the last kept slot ends at once.
template <typename U>
__global__ void __launch_bounds__(256) cache_append_kernel(const U* __restrict__ K, const U* __restrict__ V, const int* __restrict__ path,
                                                           const int* __restrict__ count, U* __restrict__ Kc, U* __restrict__ Vc,
                                                           const int* __restrict__ lens, int B, int T, int slots, int H, int per_row, int64_t capacity,
                                                           int run, int runs) {
  const int64_t lb = blockIdx.x / static_cast<unsigned>(runs);
  const int b = static_cast<int>(lb % B), j0 = static_cast<int>(blockIdx.x % static_cast<unsigned>(runs)) * run;
  int kept = slots;
  if (count) kept = count[b] < slots ? count[b] : slots;
  if (j0 >= kept) return;
  const int64_t len = lens[b];
  const int here = kept - j0 < run ? kept - j0 : run;
  const unsigned row = static_cast<unsigned>(H) * per_row, all = static_cast<unsigned>(here) * row;
  const U* from_k = K + lb * T * static_cast<int64_t>(row);
  const U* from_v = V + lb * T * static_cast<int64_t>(row);
  U* to_k = Kc + lb * H * capacity * per_row;
  U* to_v = Vc + lb * H * capacity * per_row;
  for (unsigned t = threadIdx.x; t < all; t += 256) {
    const unsigned i = t / row, in_row = t - i * row, h = in_row / static_cast<unsigned>(per_row), e = in_row - h * per_row;
    const int j = j0 + static_cast<int>(i), node = path ? path[static_cast<int64_t>(b) * slots + j] : j;
    const int64_t at = len + j;
    if (node < 0 || node >= T || at < 0 || at >= capacity) continue;
    const int64_t source = static_cast<int64_t>(node) * row + in_row, sink = (static_cast<int64_t>(h) * capacity + at) * per_row + e;
    const U k = from_k[source], v = from_v[source];
    to_k[sink] = k;
    to_v[sink] = v;
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
  constexpr int64_t kMost = int64_t{1} << 60;
  if (V > INT32_MAX || batch > INT32_MAX || V > kMost / nodes / batch) return fail("verify_tree: the extents overflow");
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
  VerifyArgs args{static_cast<const float*>(target), static_cast<const float*>(draft), static_cast<const int*>(tokens), static_cast<const int*>(parents),
                  static_cast<const float*>(accept), static_cast<const float*>(sample), static_cast<int*>(path), static_cast<int*>(count), static_cast<int*>(next),
                  static_cast<int>(nodes), V, nullptr, nullptr};
  hipStream_t s = static_cast<hipStream_t>(stream);
  // a grid holds 65535 sequences: more are further launches
  for (int64_t b = 0; b < batch; b += 65535) {
    const int64_t some = batch - b < 65535 ? batch - b : 65535;
    float* room = nullptr;
    std::unique_lock<std::recursive_mutex> lock;
    if (split_scratch(s, static_cast<size_t>(some * nodes) * sizeof(int), static_cast<size_t>(some), static_cast<int>(nodes), &room, &args.arrivals, &lock) != 0) return -1;
    args.outcomes = reinterpret_cast<int*>(room);
    hipLaunchKernelGGL(verify_tree_kernel, dim3(static_cast<unsigned>(nodes), static_cast<unsigned>(some)), dim3(kVerifyThreads), 0, s, args);
    if (check_launch("verify_tree") != 0) return -1;
    const int64_t n = some * nodes;
    args.target += n * V;
    args.draft += n * V;
    args.tokens += n;
    args.parents += n;
    args.accept += n;
    args.sample += some;
    args.path += n;
    args.count += some;
    args.next += some;
  }
  return 0;
}

extern "C" int dtas_cache_append_f16(const void* K, const void* V, const void* path, const void* count, void* K_cache, void* V_cache,
                                     const void* lens, int64_t layers, int64_t batch, int64_t nodes, int64_t slots, int64_t kv_heads, int64_t d,
                                     int64_t capacity, void* stream) {
  using namespace dtas;
  clear_error();
  if (layers < 0 || batch < 0 || nodes < 0 || slots < 0 || kv_heads < 0 || d < 0 || capacity < 0)
    return fail("cache_append: negative extent layers=%lld batch=%lld nodes=%lld slots=%lld kv_heads=%lld d=%lld capacity=%lld", (long long)layers,
                (long long)batch, (long long)nodes, (long long)slots, (long long)kv_heads, (long long)d, (long long)capacity);
  if (layers == 0 || batch == 0 || nodes == 0 || slots == 0 || kv_heads == 0 || d == 0 || capacity == 0) return 0;
  if ((path == nullptr) != (count == nullptr)) return fail("cache_append: path and count go together");
  if (!path && slots != nodes) return fail("cache_append: without a path every row has its slot (%lld rows, %lld slots)", (long long)nodes, (long long)slots);
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
  const int64_t per_row = wide ? d / 8 : d, row = kv_heads * per_row;
  // a slot of all heads at least, two pieces (of K and V) per thread and turn where the rows are short; a workgroup's pieces are counted in 32 bits
  if (row > INT32_MAX / 2) return fail("cache_append: the rows of a position are too long");
  const int64_t run = row >= 256 ? 1 : 256 / row, runs = ceil_div(slots, run);
  if (layers * batch * runs > INT32_MAX) return fail("cache_append: the launch has too many workgroups");
  auto go = [&](auto* tag) {
    using U = std::remove_pointer_t<decltype(tag)>;
    hipLaunchKernelGGL(cache_append_kernel<U>, dim3(static_cast<unsigned>(layers * batch * runs)), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const U*>(K), static_cast<const U*>(V), static_cast<const int*>(path), static_cast<const int*>(count),
                       static_cast<U*>(K_cache), static_cast<U*>(V_cache), static_cast<const int*>(lens), static_cast<int>(batch),
                       static_cast<int>(nodes), static_cast<int>(slots), static_cast<int>(kv_heads), static_cast<int>(per_row), capacity, static_cast<int>(run),
                       static_cast<int>(runs));
  };
  if (wide) go(static_cast<u32x4*>(nullptr));
  else go(static_cast<half_t*>(nullptr));
  return check_launch("cache_append");
}
