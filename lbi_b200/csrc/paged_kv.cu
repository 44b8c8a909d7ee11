// Writing the paged key / value cache (rotary turn and 8-bit quantisation included) and reading it back.
//
// append:  row = (q | k | v).  (a, b) -> (a cos - b sin, a sin + b cos) on the heads of q and k, in fp32; k and v rows go to
//          slot position % page_size of page table[position / page_size].  e4m3: scale = max |x| / 448 of the head row (the largest
//          e4m3 value), code = round(x / scale); a row of zeros has scale 0 and codes 0.
// gather:  out[b, h, j] = code * scale (or the stored value), 0 behind the context.
//
// Both are bound by memory: a head row of head_dim elements belongs to head_dim / 16 threads of 16 elements each.  In append a
// thread's 16 elements are 8 of each half of the head (the two partners of 8 turns) or 16 neighbours when the pairs are
// interleaved, so a turn needs no exchange between threads; a block owns one token, so a thread loads its 8 cosines and sines once
// for all heads.
//
// Measured on a B200: 24617 tokens of 32 + 2 x 8 heads of 128, bf16, into e4m3 pages (559 MB) 122 to 126 us, 4.5 TB/s, 0.69 of the
// copy bandwidth: latency of the chain load - maximum over the head row - division - store (46 % of the warps resident, 60 % of the issue
// slots busy, DRAM at 53 %).  12 contexts of up to 16384 tokens from e4m3 (8 heads of 128, 1.05 GB) 178 to 185 us, 0.87 to 0.90 of the copy
// bandwidth.  One token per call: launch and call, 7 us.
#include "paged.cuh"

namespace lbi {
namespace paged {

// A token's threads: 128 while blocks are few, for fewer passes over its heads (12 tokens of 48 heads of 128 11.1 us, 64 threads 13.3; 240
// tokens 11.2 / 13.4), 64 from FEW_TOKENS on, for a block's start spread over more passes (1200 tokens 17.4 / 16.4 us, 24624 tokens
// 130 / 122).  Other shapes were not measured.
constexpr int APPEND_THREADS = 128, FEW_TOKENS = 600;

struct AppendArgs {
  lbi_paged_batch b;
  const void* qkv;
  int64_t qkv_stride;
  void* q_out;
  int heads, zero_tail, page_shift, group_shift;   // 1 << group_shift threads serve one head row
  const float* cos_tab;
  const float* sin_tab;
  int64_t rope_rows;
};

// PAIRED: the turn's partners are neighbours (2 i, 2 i + 1), else i and i + head_dim / 2.
template <int TYPE, bool E4M3, bool PAIRED>
__global__ void __launch_bounds__(APPEND_THREADS, 8) append_kernel(const AppendArgs a) {
  using T = typename Elem<TYPE>::T;
  using C = typename Elem<E4M3 ? LBI_E4M3 : TYPE>::T;
  const lbi_paged_batch& p = a.b;
  const int row = blockIdx.x, dim = p.head_dim, half = dim >> 1;
  const int group = 1 << a.group_shift, lane = threadIdx.x & (group - 1);
  const int d0 = PAIRED ? lane * 16 : lane * 8, d1 = PAIRED ? d0 + 8 : d0 + half;   // two runs of 8 elements
  const bool active = lane * 16 < dim;
  const int total = a.heads + 2 * p.kv_heads, per_pass = blockDim.x >> a.group_shift, first = threadIdx.x >> a.group_shift;
  const T* src = (const T*)a.qkv + (int64_t)row * a.qkv_stride;
  T* q_out = (T*)a.q_out + (int64_t)row * a.heads * dim;

  Vec<T, 8> next[2] = {};
  bool dead = false;   // no position: q is zero, nothing is written
  auto load = [&](int h) {
    if (h < total && active && !dead) {
      next[0] = *reinterpret_cast<const Vec<T, 8>*>(src + h * dim + d0);
      next[1] = *reinterpret_cast<const Vec<T, 8>*>(src + h * dim + d1);
    }
  };
  load(first);   // before anything is known about the token, and then one head row ahead

  int pos = -1, page = -1;
  bool turn_ok = true;
  Place at = {0, 0, 0, false};
  if (p.batch > 0) at = place_of_row(p, row);
  if (!at.owned && !a.zero_tail) return;
  if (at.owned) {
    pos = __ldg(p.context + at.b) - (at.last - row);
    if (pos >= 0) page = page_of(p, at.b, pos, a.page_shift);
    if (a.cos_tab && pos >= a.rope_rows) {
      turn_ok = false;
      if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, 83);
    }
  }
  dead = pos < 0 || !turn_ok;
  if (dead) next[0] = next[1] = Vec<T, 8>{};
  union Eight {
    float f[8];
    float2 f2[4];
  } cs, sn;
#pragma unroll
  for (int i = 0; i < 8; ++i) cs.f[i] = 1.f, sn.f[i] = 0.f;
  if (a.cos_tab && !dead && active) {
    load_f<float, 8>(a.cos_tab + (int64_t)pos * half + lane * 8, cs.f);
    load_f<float, 8>(a.sin_tab + (int64_t)pos * half + lane * 8, sn.f);
  }
#pragma unroll 1
  for (int h0 = 0; h0 < total; h0 += per_pass) {
    const int h = h0 + first;
    const bool here = h < total && active;
    Eight u, w;   // the partners of eight turns (or 16 elements of a value row)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      u.f[e] = PAIRED ? to_f<T>(next[e >> 2].v[2 * (e & 3)]) : to_f<T>(next[0].v[e]);
      w.f[e] = PAIRED ? to_f<T>(next[e >> 2].v[2 * (e & 3) + 1]) : to_f<T>(next[1].v[e]);
    }
    load(h + per_pass);
    if (a.cos_tab && h < a.heads + p.kv_heads) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 un = u.f2[e], wn = w.f2[e], minus = make_float2(-sn.f2[e].x, -sn.f2[e].y);
        u.f2[e] = fma2(wn, minus, mul2(un, cs.f2[e]));
        w.f2[e] = fma2(un, sn.f2[e], mul2(wn, cs.f2[e]));
      }
    }
    float top = 0.f;
    if (E4M3) {   // every thread of the warp takes part in the exchange
      // as whole numbers, magnitudes are in order, with a NaN (which has to reach the scale) above all
      int most = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) most = max(most, max(__float_as_int(u.f[e]) & 0x7fffffff, __float_as_int(w.f[e]) & 0x7fffffff));
      for (int o = 1; o < group; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      top = __int_as_float(most);
    }
    if (!here) continue;
    float x[16];   // in the order of memory: run d0, run d1
    auto in_order = [&] {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[PAIRED ? 2 * e : e] = u.f[e];
        x[PAIRED ? 2 * e + 1 : 8 + e] = w.f[e];
      }
    };
    if (h < a.heads) {
      in_order();
      store_f<T, 8>(q_out + h * dim + d0, x);
      store_f<T, 8>(q_out + h * dim + d1, x + 8);
      continue;
    }
    if (dead || page < 0) continue;
    const bool is_k = h - a.heads < p.kv_heads;
    const int kh = is_k ? h - a.heads : h - a.heads - p.kv_heads;
    const int slot = (page * p.kv_heads + kh) * p.page_size + (pos & (p.page_size - 1));
    C* dst = (C*)(is_k ? p.k : p.v) + (int64_t)slot * dim;
    if (E4M3) {
      const float scale = __fmul_rn(top, 1.f / 448.f);
      // One reciprocal per head row: x * (1 / scale) is within 2^-22 of x / scale, some millionths of the code's half step.  A scale
      // below the normal range has no reciprocal: those rows divide.
      if (scale < 1.17549435e-38f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          u.f[e] = scale == 0.f ? 0.f : __fdiv_rn(u.f[e], scale);
          w.f[e] = scale == 0.f ? 0.f : __fdiv_rn(w.f[e], scale);
        }
      } else {
        float inv;
        asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(scale));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u.f2[e] = mul2(u.f2[e], make_float2(inv, inv));
          w.f2[e] = mul2(w.f2[e], make_float2(inv, inv));
        }
      }
      in_order();
      uint32_t code[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * e], x[4 * e + 1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * e + 2], x[4 * e + 3]), __NV_SATFINITE, __NV_E4M3);
        code[e] = __byte_perm(lo, hi, 0x5410);
      }
      *reinterpret_cast<uint2*>(dst + d0) = make_uint2(code[0], code[1]);
      *reinterpret_cast<uint2*>(dst + d1) = make_uint2(code[2], code[3]);
      if (lane == 0) (is_k ? p.k_scale : p.v_scale)[slot] = scale;
    } else {
      in_order();
      store_f<T, 8>((T*)dst + d0, x);
      store_f<T, 8>((T*)dst + d1, x + 8);
    }
  }
}

template <int TYPE, bool E4M3>
__global__ void __launch_bounds__(256) gather_kernel(const lbi_paged_batch p, void* k_out, void* v_out, int max_len, int page_shift, int bh0) {
  using T = typename Elem<TYPE>::T;
  using C = typename Elem<E4M3 ? LBI_E4M3 : TYPE>::T;
  const unsigned dim = p.head_dim, parts = dim >> 4;   // 16 elements per thread
  const int bh = bh0 + blockIdx.y, b = bh / p.kv_heads, h = bh % p.kv_heads;
  const unsigned i = blockIdx.x * 256 + threadIdx.x;
  const int pos = (int)(i / parts), d = (int)(i % parts) * 16;
  if (pos >= max_len) return;
  float x[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = 0.f;
  const bool is_k = blockIdx.z == 0;
  if (pos < __ldg(p.context + b)) {
    const int page = page_of(p, b, pos, page_shift);
    if (page >= 0) {
      const int64_t slot = ((int64_t)page * p.kv_heads + h) * p.page_size + (pos & (p.page_size - 1));
      load_f<C, 16>((const C*)(is_k ? p.k : p.v) + slot * dim + d, x);
      if (E4M3) {
        const float scale = __ldg((is_k ? p.k_scale : p.v_scale) + slot);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] *= scale;
      }
    }
  }
  store_f<T, 16>((T*)(is_k ? k_out : v_out) + ((int64_t)bh * max_len + pos) * dim + d, x);
}

}  // namespace paged
}  // namespace lbi

#define LBI_BY_TYPE(type, e4m3, CALL)                                              \
  do {                                                                             \
    if ((type) == LBI_F32) { if (e4m3) { CALL(LBI_F32, true); } else { CALL(LBI_F32, false); } }      \
    else if ((type) == LBI_BF16) { if (e4m3) { CALL(LBI_BF16, true); } else { CALL(LBI_BF16, false); } } \
    else { if (e4m3) { CALL(LBI_F16, true); } else { CALL(LBI_F16, false); } }     \
  } while (0)

extern "C" int lbi_kv_append(const lbi_paged_batch* p, const void* qkv, int64_t qkv_stride, void* q_out, int type, int heads,
                             const float* cos_tab, const float* sin_tab, int64_t rope_rows, int interleaved, int zero_tail, cudaStream_t st) {
  using namespace lbi::paged;
  if (p->head_dim % 16 != 0 || p->head_dim > 256 || p->rows < 0 || type < 0 || type > LBI_F16) return (int)cudaErrorInvalidValue;
  if (p->rows == 0) return 0;
  AppendArgs a{*p, qkv, qkv_stride, q_out, heads, zero_tail, shift_of(p->page_size), shift_of(p->head_dim / 16), cos_tab, sin_tab, rope_rows};
  const int threads = p->rows < FEW_TOKENS ? APPEND_THREADS : APPEND_THREADS / 2;
#define LBI_APPEND(T, E)                                                             \
  do {                                                                                \
    if (interleaved) append_kernel<T, E, true><<<p->rows, threads, 0, st>>>(a); \
    else append_kernel<T, E, false><<<p->rows, threads, 0, st>>>(a);            \
  } while (0)
  LBI_BY_TYPE(type, p->cache_type == LBI_E4M3, LBI_APPEND);
#undef LBI_APPEND
  return (int)cudaGetLastError();
}

extern "C" int lbi_kv_gather(const lbi_paged_batch* p, void* k_out, void* v_out, int64_t max_len, int type, cudaStream_t st) {
  using namespace lbi::paged;
  if (p->head_dim % 16 != 0 || p->head_dim > 256 || type < 0 || type > LBI_F16) return (int)cudaErrorInvalidValue;
  if (max_len <= 0 || p->batch == 0) return 0;
  const int64_t pairs = (int64_t)p->batch * p->kv_heads;
  if (max_len * (p->head_dim / 16) >= (1ll << 31) || pairs >= (1ll << 31)) return (int)cudaErrorInvalidValue;
  const int shift = shift_of(p->page_size);
  for (int64_t bh0 = 0; bh0 < pairs; bh0 += 65535) {   // what one grid holds in its second dimension
    const dim3 grid((unsigned)((max_len * (p->head_dim / 16) + 255) / 256), (unsigned)(pairs - bh0 < 65535 ? pairs - bh0 : 65535), 2);
#define LBI_GATHER(T, E) gather_kernel<T, E><<<grid, 256, 0, st>>>(*p, k_out, v_out, (int)max_len, shift, (int)bh0)
    LBI_BY_TYPE(type, p->cache_type == LBI_E4M3, LBI_GATHER);
#undef LBI_GATHER
  }
  return (int)cudaGetLastError();
}
