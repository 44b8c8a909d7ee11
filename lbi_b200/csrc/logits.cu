// Rules on the logits of the next token: penalties for tokens that occurred already, a bias and a grammar mask, in one pass.
//
//   seen  = the token occurs in the row's history, made = how often it occurs behind the prompt
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - presence * [made > 0] - frequency * made + bias;   not allowed -> -inf (whatever the logit was, NaN included)
//
// Bound by memory (logits in, fp32 out).  A block owns a tile of the vocabulary of one row: it counts the history's tokens that
// fall into the tile in shared memory (whole numbers: the order of the atomics does not matter); the count's highest bit marks a token
// that occurs in the prompt.  Every block of a row reads the row's history again, which stays in L2, so tiles are large: 16-bit counts,
// two to a word, while the history is shorter than 2^15, else 32-bit counts of half as many tokens.
//
// Measured on a B200: 192 rows of 128001 fp32 logits, histories of up to 4096 tokens, bias and mask: 58 us against 32 us for reading and
// writing the logits once (207 MB).  The rest is the blocks' start, during which no logit is loaded: counters to zero, a walk over the
// history (9 tiles read it), two barriers; 65 % of the issue slots are busy, DRAM at 35 %.  A row of 32768: launch and call, 5.3 to 6.4 us.
#include <algorithm>

#include "paged.cuh"

namespace lbi {
namespace paged {

constexpr int COUNT_BYTES = 32768;
// Three blocks per SM leave registers for the loads of EACH elements at once.  Measured with 192 x 128001: 58 us; four blocks 63 us; three
// blocks with 2 or 8 elements 66 and 64 us; two blocks 71 us; six blocks of 256 threads 60 us, one of 1024 86 us.
constexpr int LOGIT_THREADS = 512, LOGIT_BLOCKS = 3, EACH = 4;

template <int TYPE, typename COUNT>
__global__ void __launch_bounds__(LOGIT_THREADS, LOGIT_BLOCKS) logits_kernel(const lbi_logit_rules p, int tile, unsigned tiles) {
  using T = typename Elem<TYPE>::T;
  constexpr bool WIDE = sizeof(COUNT) == 4;
  constexpr uint32_t PROMPT = WIDE ? 0x80000000u : 0x8000u;
  __shared__ alignas(16) COUNT count[COUNT_BYTES / sizeof(COUNT)];
  const int b = blockIdx.x / tiles, v0 = (blockIdx.x % tiles) * tile, n = min(tile, p.vocab - v0);
  for (int i = threadIdx.x; i < tile * (int)sizeof(COUNT) / 16; i += LOGIT_THREADS) reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.history) : p.history;
  const int prompt = p.prompt_lengths ? p.prompt_lengths[b] : 0;
  const float rep = p.repetition_row ? p.repetition_row[b] : p.repetition;
  const float pres = p.presence_row ? p.presence_row[b] : p.presence;
  const float freq = p.frequency_row ? p.frequency_row[b] : p.frequency;
  const int64_t* hist = p.tokens + (int64_t)b * p.tokens_stride;
  __syncthreads();
  for (int i0 = threadIdx.x; i0 < len; i0 += 4 * LOGIT_THREADS) {
    int64_t t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = i0 + e * LOGIT_THREADS < len ? __ldg(hist + i0 + e * LOGIT_THREADS) - v0 : -1;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (t[e] >= 0 && t[e] < n) {
        uint32_t* word = reinterpret_cast<uint32_t*>(count) + (WIDE ? t[e] : t[e] >> 1);
        const int shift = WIDE ? 0 : (int)(t[e] & 1) * 16;
        // text repeats itself: what the prompt has set already is not set again
        if (i0 + e * LOGIT_THREADS >= prompt) atomicAdd(word, 1u << shift);
        else if (!(*reinterpret_cast<volatile uint32_t*>(word) >> shift & PROMPT)) atomicOr(word, PROMPT << shift);
      }
  }
  __syncthreads();
  const T* x = (const T*)p.logits + (int64_t)b * p.logits_stride + v0;
  float* out = p.out + (int64_t)b * p.out_stride + v0;
  const float* bias = p.bias ? p.bias + (int64_t)b * p.bias_stride + v0 : nullptr;
  const int* allowed = p.allowed ? p.allowed + (int64_t)b * p.allowed_stride + (v0 >> 5) : nullptr;
  // Rows of odd vocabularies start anywhere, so an element per thread and access, several in flight; the tile's end is a case of its
  // own.  A tile starts at a multiple of 32, so a warp's 32 elements share a word of the mask.
  auto rules = [&](int i, float f, float add, uint32_t bits) {
    const uint32_t c = count[i];
    if (c) {
      f = f > 0.f ? __fdiv_rn(f, rep) : f * rep;
      const uint32_t made = c & (PROMPT - 1);
      if (made) f = __fsub_rn(__fsub_rn(f, pres), __fmul_rn(freq, (float)made));
    }
    if (bias) f += add;
    out[i] = bits >> (threadIdx.x & 31) & 1u ? f : -INFINITY;
  };
  int i = threadIdx.x;
  for (; i + (EACH - 1) * LOGIT_THREADS < n; i += EACH * LOGIT_THREADS) {
    float f[EACH], add[EACH];
    uint32_t bits[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) f[e] = to_f<T>(x[i + e * LOGIT_THREADS]);
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      add[e] = bias ? __ldg(bias + i + e * LOGIT_THREADS) : 0.f;
      bits[e] = allowed ? (uint32_t)__ldg(allowed + ((i + e * LOGIT_THREADS) >> 5)) : 0xffffffffu;
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) rules(i + e * LOGIT_THREADS, f[e], add[e], bits[e]);
  }
  for (; i < n; i += LOGIT_THREADS)
    rules(i, to_f<T>(x[i]), bias ? __ldg(bias + i) : 0.f, allowed ? (uint32_t)__ldg(allowed + (i >> 5)) : 0xffffffffu);
}

template <int TYPE>
static int launch_logits(const lbi_logit_rules& p, int sm_count, cudaStream_t st) {
  // As few tiles as the counts allow, then so many more as fit into the same number of rounds of blocks (192 x 128001: 9
  // instead of 8 per row), of 1024 tokens at least.
  const bool wide = p.history >= 32768;
  const int64_t most = COUNT_BYTES / (wide ? 4 : 2), slots = (int64_t)LOGIT_BLOCKS * sm_count;
  const int64_t fewest = (p.vocab + most - 1) / most, rounds = (fewest * p.batch + slots - 1) / slots;
  const int64_t wanted = std::max(fewest, rounds * slots / p.batch);
  const int tile = (int)std::min<int64_t>(most, std::max<int64_t>(1024, ((p.vocab + wanted - 1) / wanted + 31) / 32 * 32));
  const unsigned tiles = (unsigned)((p.vocab + tile - 1) / tile);
  if ((int64_t)tiles * p.batch >= (1ll << 31)) return (int)cudaErrorInvalidValue;
  const unsigned grid = tiles * p.batch;
  static lbi::PerDeviceOnce narrow_once, wide_once;
  narrow_once.all_shared(logits_kernel<TYPE, uint16_t>);
  wide_once.all_shared(logits_kernel<TYPE, uint32_t>);
  if (wide) logits_kernel<TYPE, uint32_t><<<grid, LOGIT_THREADS, 0, st>>>(p, tile, tiles);
  else logits_kernel<TYPE, uint16_t><<<grid, LOGIT_THREADS, 0, st>>>(p, tile, tiles);
  return (int)cudaGetLastError();
}

}  // namespace paged
}  // namespace lbi

extern "C" int lbi_adjust_logits(const lbi_logit_rules* p, int sm_count, cudaStream_t st) {
  using namespace lbi::paged;
  if (p->batch == 0 || p->vocab == 0) return 0;
  if (p->type < 0 || p->type > LBI_F16) return (int)cudaErrorInvalidValue;
  return p->type == LBI_F32 ? launch_logits<LBI_F32>(*p, sm_count, st)
       : p->type == LBI_BF16 ? launch_logits<LBI_BF16>(*p, sm_count, st) : launch_logits<LBI_F16>(*p, sm_count, st);
}
