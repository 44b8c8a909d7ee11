// Device helpers shared by the operators over a paged key / value cache: element types, the batch's geometry, page lookup.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "api_paged.h"
#include "common.cuh"

namespace lbi {
namespace paged {

struct AttnArgs {
  lbi_paged_batch b;
  const void* q;
  int64_t q_stride;
  void* out;
  float* part_o;      // [rows * heads, splits, head_dim] results of the parts, null when there is one
  float* part_lse;    // [rows * heads, splits] base-2 logarithm of the sum of exponentials
  int heads, group, zero_tail, page_shift, splits, split_keys;
  float scale_log2;
};

int launch_attn_tiles(const AttnArgs& a, int type, cudaStream_t st);   // paged_attn_tc.cu

template <int TYPE> struct Elem;
template <> struct Elem<LBI_F32> { using T = float; };
template <> struct Elem<LBI_BF16> { using T = __nv_bfloat16; };
template <> struct Elem<LBI_F16> { using T = __half; };
template <> struct Elem<LBI_E4M3> { using T = __nv_fp8_storage_t; };

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(float x) { return x; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f(__nv_fp8_storage_t x) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(x, __NV_E4M3))); }

template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }

// N elements of T (N * sizeof(T) a multiple of 4) as fp32, loaded and stored in the widest words that fit.
template <typename T, int N>
struct alignas(sizeof(T) * N >= 16 ? 16 : sizeof(T) * N) Vec {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ void load_f(const T* p, float* f) {
  Vec<T, N> x = *reinterpret_cast<const Vec<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = to_f<T>(x.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_f(T* p, const float* f) {
  Vec<T, N> x;
#pragma unroll
  for (int i = 0; i < N; ++i) x.v[i] = from_f<T>(f[i]);
  *reinterpret_cast<Vec<T, N>*>(p) = x;
}

// [first, last) rows of the new tokens of sequence b.  Offsets are clamped to the rows that exist: a wrong one can leave tokens
// out but never reach outside q.
__device__ __forceinline__ int2 seq_rows(const lbi_paged_batch& p, int b) {
  if (!p.cu) {
    const int each = p.rows / p.batch;
    return make_int2(b * each, (b + 1) * each);
  }
  const int lo = min(max(__ldg(p.cu + b), 0), p.rows);
  return make_int2(lo, min(max(__ldg(p.cu + b + 1), lo), p.rows));
}

// The last b of [0, n) with below(b), which holds for a first part of them (0 if for none); a full warp calls, 32 candidates are tried
// at a time.
template <typename F>
__device__ __forceinline__ int last_below(int n, F below) {
  int lo = 0;
  const int lane = threadIdx.x & 31;
  while (n > 1) {
    const int step = (n + 31) >> 5;
    const bool yes = lane * step < n && below(lo + lane * step);
    const int hit = max(__popc(__ballot_sync(0xffffffffu, yes)) - 1, 0);
    n = min(step, n - hit * step);
    lo += hit * step;
  }
  return lo;
}

// Sequence of row `row`, its rows [first, last), and whether the row belongs to any; a full warp calls.  Batches of up to 31 sequences
// read all offsets at once.
struct Place {
  int b, first, last;
  bool owned;
};
__device__ __forceinline__ Place place_of_row(const lbi_paged_batch& p, int row) {
  if (!p.cu) {
    const int each = p.rows / p.batch, b = row / each;
    return {b, b * each, (b + 1) * each, true};
  }
  if (p.batch < 32) {
    const int lane = threadIdx.x & 31;
    const int v = min(max(__ldg(p.cu + min(lane, p.batch)), 0), p.rows);
    const int b = min(max(__popc(__ballot_sync(0xffffffffu, lane < p.batch && v <= row)) - 1, 0), p.batch - 1);
    const int lo = __shfl_sync(0xffffffffu, v, b), hi = max(__shfl_sync(0xffffffffu, v, b + 1), lo);
    return {b, lo, hi, row >= lo && row < hi};
  }
  const int b = last_below(p.batch, [&](int i) { return __ldg(p.cu + i) <= row; });
  const int2 r = seq_rows(p, b);
  return {b, r.x, r.y, row >= r.x && row < r.y};
}

// The rows [x, y) from the first sequence's to the last's; those in front and behind belong to nobody.
__device__ __forceinline__ int2 owned_rows(const lbi_paged_batch& p) {
  if (!p.cu) return make_int2(0, p.rows);
  const int last = min(max(__ldg(p.cu + p.batch), 0), p.rows);
  return make_int2(min(max(__ldg(p.cu), 0), last), last);
}
// Zeros in the rows of nobody of `out` [rows, width], shared among all blocks.
template <typename T>
__device__ __forceinline__ void zero_rows_of_nobody(const lbi_paged_batch& p, T* out, int width) {
  const int2 own = owned_rows(p);
  const int nobody = own.x + p.rows - own.y;
  for (int64_t i = blockIdx.x; i < nobody; i += gridDim.x) {
    const int64_t row = i < own.x ? i : i + own.y - own.x;
    for (int e = threadIdx.x; e < width; e += blockDim.x) out[row * width + e] = from_f<T>(0.f);
  }
}

// Page of position pos of sequence b, or -1 (recorded as status 84) where the table or the pool ends.
__device__ __forceinline__ int page_of(const lbi_paged_batch& p, int b, int pos, int page_shift) {
  const int i = pos >> page_shift;
  int page = -1;
  if (i < p.table_width) page = __ldg(p.table + (int64_t)b * p.table_stride + i);
  if (page < 0 || page >= p.num_pages) {
    if (p.status) atomicCAS(p.status, 0, 84);
    return -1;
  }
  return page;
}

// Work is cut into tiles of `per_tile` rows (row r of a sequence's tile space = token * group + head of the group); sequence b owns
// the tiles from cu[b] * group / per_tile + b on, which is never less than the tiles of the sequences before it need, so a tile finds
// its sequence without a prefix sum over the batch and the host needs only rows and batch to size the grid.
__device__ __forceinline__ int64_t first_tile(const lbi_paged_batch& p, int b, int group, int per_tile) {
  const int64_t start = p.cu ? min(max(__ldg(p.cu + b), 0), p.rows) : (int64_t)b * (p.rows / p.batch);
  return start * group / per_tile + b;
}
inline int64_t tile_bound(const lbi_paged_batch& p, int group, int per_tile) { return (int64_t)p.rows * group / per_tile + p.batch; }

// Sequence of tile `tile`; a full warp calls.
__device__ __forceinline__ int seq_of_tile(const lbi_paged_batch& p, int64_t tile, int group, int per_tile) {
  return last_below(p.batch, [&](int b) { return first_tile(p, b, group, per_tile) <= tile; });
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 values as one 32-bit word of a 16-bit type (a in the low half).
template <int TYPE>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  uint32_t d;
  if (TYPE == LBI_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  return d;
}

// Four e4m3 codes -> two words of a 16-bit type, exactly: sign, exponent and mantissa are moved to their places, which divides the value
// by 2^120 (bf16) or 2^8 (fp16), codes below the normal range included, and the quotient is multiplied back.  (fp16 has a conversion
// instruction, but it runs on the unit of the exponentials.)  A NaN code comes out as 480: rows with a NaN carry a NaN scale.
template <int TYPE>
__device__ __forceinline__ void codes_to_16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t a = __byte_perm(w, 0, 0x1404), b = __byte_perm(w, 0, 0x3424);
  if (TYPE == LBI_F16) {
    const uint32_t x = ((a >> 1) & 0x3f803f80u) | (a & 0x80008000u), y = ((b >> 1) & 0x3f803f80u) | (b & 0x80008000u);
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(x), "r"(0x5c005c00u));
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(y), "r"(0x5c005c00u));
  } else {
    const uint32_t x = ((a >> 4) & 0x07f007f0u) | (a & 0x80008000u), y = ((b >> 4) & 0x07f007f0u) | (b & 0x80008000u);
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(x), "r"(0x7b807b80u));
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(y), "r"(0x7b807b80u));
  }
}

// The same by the conversion instruction, for kernels that have time on its unit.
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations per instruction (packed pairs, sm_100).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)),
        "l"(reinterpret_cast<const unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
  return d;
}

// Scale of a value row: a row of zeros has scale 0, which has no logarithm and no reciprocal; its codes are 0, so any positive
// scale serves.  A NaN stays.  A row whose largest element is below 4.5e-28 is read as one of up to that size.
__device__ __forceinline__ float positive_scale(float s) { return s < 1e-30f ? 1e-30f : s; }

__host__ __device__ __forceinline__ int shift_of(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

}  // namespace paged
}  // namespace lbi
