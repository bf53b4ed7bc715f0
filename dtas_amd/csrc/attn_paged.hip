// Attention of one new token per sequence over keys and values in pages, for gfx950.
//
//   row (b, h): query head h of sequence b, which shares key head h / (heads / kv_heads), sees the positions j < lens[b];
//   position j lies in page table[b][j / page], row j % page
//   out[b, h, :] = sum_j softmax_j(scale * Q[b, h, :] . k_j) v_j                         fp32 scores, statistics and sums
//
// Positions in pages outside [0, pages) are not seen; a row that sees nothing is zeros.
#include "gemm_common.h"

namespace dtas {
namespace {

struct PagedArgs {
  const half_t *Q, *K, *V;
  const int *table, *lens;
  half_t* out;
  int heads, kv_heads, d, pages;
  unsigned page;
  int64_t columns;
  float scale_log2;  // |scale| * log2(e): the softmax is taken in powers of two
  half_t sign;       // the scale's: 1, -1, or 0 (scale_log2 is 1 then)
};

// positions of a sequence (its table holds no more)
__device__ __forceinline__ unsigned length_of(const PagedArgs& a, int64_t b) {
  const int len = a.lens[b];
  const int64_t room = a.columns * a.page;
  return len < 0 ? 0u : len > room ? static_cast<unsigned>(room) : static_cast<unsigned>(len);
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
              static_cast<unsigned>(page), columns, scale == 0.f ? 1.f : fabsf(scale) * 1.4426950408889634f, static_cast<half_t>(scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t total = batch * heads;
  const int64_t grid = total < (int64_t{1} << 22) ? total : int64_t{1} << 22;
  hipLaunchKernelGGL(attn_paged_scalar_kernel, dim3(static_cast<unsigned>(grid)), dim3(64), 0, s, a, total);
  return check_launch("attn_paged");
}
