// Rules on the logits of the next token: penalties for tokens that occurred already, a bias and a grammar mask, in one pass.
//
//   seen  = the token occurs in the row's history, made = how often it occurs behind the prompt
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - presence * [made > 0] - frequency * made + bias;   not allowed -> -inf (whatever the logit was, NaN included)
//
// Bound by memory (logits in, fp32 out).  A block owns a tile of the vocabulary of one row: it counts the history's tokens that
// fall into the tile in shared memory (whole numbers: the order of the atomics does not matter), bit 31 marks a token that occurs
// in the prompt only.  Every block of a row reads the row's history again, which stays in L2.
#include "paged.cuh"

namespace lbi {
namespace paged {

constexpr int TILE_V = 4096;
constexpr int LOGIT_THREADS = 256;

template <int TYPE>
__global__ void __launch_bounds__(LOGIT_THREADS) logits_kernel(const lbi_logit_rules p) {
  using T = typename Elem<TYPE>::T;
  __shared__ uint32_t count[TILE_V];
  const int b = blockIdx.y, v0 = blockIdx.x * TILE_V, n = min(TILE_V, p.vocab - v0);
  for (int i = threadIdx.x; i < TILE_V; i += LOGIT_THREADS) count[i] = 0;
  __syncthreads();
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.history) : p.history;
  const int prompt = p.prompt_lengths ? p.prompt_lengths[b] : 0;
  const int64_t* hist = p.tokens + (int64_t)b * p.tokens_stride;
  for (int i = threadIdx.x; i < len; i += LOGIT_THREADS) {
    const int64_t t = hist[i] - v0;
    if (t >= 0 && t < n) {
      if (i < prompt) atomicOr(&count[t], 0x80000000u);
      else atomicAdd(&count[t], 1u);
    }
  }
  __syncthreads();
  const float rep = p.repetition_row ? p.repetition_row[b] : p.repetition;
  const float pres = p.presence_row ? p.presence_row[b] : p.presence;
  const float freq = p.frequency_row ? p.frequency_row[b] : p.frequency;
  const T* x = (const T*)p.logits + (int64_t)b * p.logits_stride + v0;
  float* out = p.out + (int64_t)b * p.out_stride + v0;
  const float* bias = p.bias ? p.bias + (int64_t)b * p.bias_stride + v0 : nullptr;
  const int* allowed = p.allowed ? p.allowed + (int64_t)b * p.allowed_stride + (v0 >> 5) : nullptr;
  for (int i = threadIdx.x; i < n; i += LOGIT_THREADS) {
    float f = to_f<T>(x[i]);
    const uint32_t c = count[i];
    if (c) {
      f = f > 0.f ? __fdiv_rn(f, rep) : f * rep;
      const uint32_t made = c & 0x7fffffffu;
      if (made) f = __fsub_rn(__fsub_rn(f, pres), __fmul_rn(freq, (float)made));
    }
    if (bias) f += bias[i];
    if (allowed && !((uint32_t)allowed[i >> 5] >> (i & 31) & 1u)) f = -INFINITY;
    out[i] = f;
  }
}

}  // namespace paged
}  // namespace lbi

extern "C" int lbi_adjust_logits(const lbi_logit_rules* p, cudaStream_t st) {
  using namespace lbi::paged;
  if (p->batch == 0 || p->vocab == 0) return 0;
  if (p->batch > 65535 || p->type < 0 || p->type > LBI_F16) return (int)cudaErrorInvalidValue;
  dim3 grid((p->vocab + TILE_V - 1) / TILE_V, p->batch);
  if (p->type == LBI_F32) logits_kernel<LBI_F32><<<grid, LOGIT_THREADS, 0, st>>>(*p);
  else if (p->type == LBI_BF16) logits_kernel<LBI_BF16><<<grid, LOGIT_THREADS, 0, st>>>(*p);
  else logits_kernel<LBI_F16><<<grid, LOGIT_THREADS, 0, st>>>(*p);
  return (int)cudaGetLastError();
}
