// Causal attention of new tokens over a paged key / value cache.
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j   over the positions j <= context - new + i of the sequence; no position: o_i = 0.
//
// One warp per (token, head): the lanes share the head's elements, the running maximum m and sum l of the softmax and the output
// row stay in registers in fp32 and every key is read once.  e4m3 pages: the key's scale multiplies its score, the value's scale
// its probability.
#include "paged.cuh"

namespace lbi {
namespace paged {

struct AttnArgs {
  lbi_paged_batch b;
  const void* q;
  int64_t q_stride;
  void* out;
  int heads, zero_tail, page_shift;
  float scale_log2;
};

template <int TYPE, bool E4M3>
__global__ void __launch_bounds__(128) attn_row_kernel(const AttnArgs a) {
  using T = typename Elem<TYPE>::T;
  using C = typename Elem<E4M3 ? LBI_E4M3 : TYPE>::T;
  const lbi_paged_batch& p = a.b;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, dim = p.head_dim;
  const int row = (int)(unit / a.heads), head = (int)(unit % a.heads);
  if (row >= p.rows) return;
  T* out = (T*)a.out + ((int64_t)row * a.heads + head) * dim;
  float q[8], o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = o[e] = 0.f;
  float l = 0.f;
  if (row < last_row(p)) {
    const int b = seq_of_row(p, row);
    const int2 r = seq_rows(p, b);
    const int ctx = __ldg(p.context + b);
    const int keys = min(ctx - (r.y - row) + 1, p.table_width << a.page_shift);
    const int kh = head / (a.heads / p.kv_heads);
    const T* src = (const T*)a.q + (int64_t)row * a.q_stride + head * dim;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane + 32 * e < dim) q[e] = to_f<T>(src[lane + 32 * e]) * a.scale_log2;
    float m = -INFINITY;
    for (int j = 0; j < keys; ++j) {
      const int page = page_of(p, b, j, a.page_shift);
      if (page < 0) continue;
      const int64_t slot = ((int64_t)page * p.kv_heads + kh) * p.page_size + (j & (p.page_size - 1));
      const C* kp = (const C*)p.k + slot * dim;
      const C* vp = (const C*)p.v + slot * dim;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (lane + 32 * e < dim) s += q[e] * to_f<C>(kp[lane + 32 * e]);
      s = warp_sum(s);
      if (E4M3) s *= __ldg(p.k_scale + slot);
      const float mn = fmaxf(m, s);
      const float keep = exp2f(m - mn);
      float w = exp2f(s - mn);
      l = l * keep + w;
      m = mn;
      if (E4M3) w *= __ldg(p.v_scale + slot);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (lane + 32 * e < dim) o[e] = o[e] * keep + w * to_f<C>(vp[lane + 32 * e]);
    }
  } else if (!a.zero_tail) {
    return;
  }
  const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (lane + 32 * e < dim) out[lane + 32 * e] = from_f<T>(o[e] * inv);
}

}  // namespace paged
}  // namespace lbi

extern "C" int lbi_paged_attention(const lbi_paged_batch* p, const void* q, int64_t q_stride, void* out, int type, int heads, float scale,
                                   int zero_tail, cudaStream_t st) {
  using namespace lbi::paged;
  if (p->head_dim % 16 != 0 || p->head_dim > 256 || type < 0 || type > LBI_F16 || heads % p->kv_heads != 0) return (int)cudaErrorInvalidValue;
  if (p->rows == 0) return 0;
  AttnArgs a{*p, q, q_stride, out, heads, zero_tail, shift_of(p->page_size), scale * 1.4426950408889634f};
  const int64_t blocks = ((int64_t)p->rows * heads + 3) / 4;
  if (blocks >= (1ll << 31)) return (int)cudaErrorInvalidValue;
#define LBI_ATTN(T, E) attn_row_kernel<T, E><<<(unsigned)blocks, 128, 0, st>>>(a)
  const bool e4m3 = p->cache_type == LBI_E4M3;
  if (type == LBI_F32) { if (e4m3) LBI_ATTN(LBI_F32, true); else LBI_ATTN(LBI_F32, false); }
  else if (type == LBI_BF16) { if (e4m3) LBI_ATTN(LBI_BF16, true); else LBI_ATTN(LBI_BF16, false); }
  else { if (e4m3) LBI_ATTN(LBI_F16, true); else LBI_ATTN(LBI_F16, false); }
#undef LBI_ATTN
  return (int)cudaGetLastError();
}
