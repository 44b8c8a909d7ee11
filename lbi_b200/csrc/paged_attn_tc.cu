// Causal attention of a chunk of new tokens over a paged cache, on tcgen05 / TMEM / TMA: 16-bit queries, head_dim 64 or 128.
//
// A block owns 256 rows (token x head of a group, heads fastest, so that a key is loaded once for all heads of its group): two tiles
// of 128 rows, each with a softmax warpgroup of its own, and walks the keys KEYS (64 or 128) at a time:
//     S_g = Q_g K_j^T        M 128 x N KEYS, TMEM columns [KEYS g, ..)
//     P_g = 2^(S_g - m)      rounded to the queries' type and stored over S_g in TMEM: the second product takes its left operand
//                            from there, so P never passes through shared memory (half a step per weight, as the result itself is
//                            rounded: 2.3e-3 of the result in bf16, 2.9e-4 in fp16, against 1.7e-3 and 2.1e-4 for the result's
//                            rounding alone; a second term of P would double the products with V)
//     O_g += P_g V_j         M 128 x N head_dim, accumulated in TMEM columns [2 KEYS + head_dim g, ..)
// Products of a thread run in the order in which they are issued, so S_g of the next tile may be issued right behind the product that
// still reads P_g, and the barrier that announces S_g(j + 1) also says that O_g holds tile j.  The running maximum follows the row only
// when it has grown by more than 2^8 (fp16: 2^4): P stays in (0, 2^8], and O is rescaled (a read and a write of TMEM) in the first tiles
// only.  fp16 has half a step of 2^-11 only down to 2^-14, and the keys of a long context may all weigh less than that beside one heavy
// key: there P is held times 2^11, up to 2^15, so that the half step holds down to 2^-25 of the heaviest key.
// While one warpgroup computes exponentials the tensor core works for the other.
//
// What bounds it: the chain S -> maximum -> exponentials -> P -> products of a row tile, of which two (or, with 16-bit pages at head_dim
// 64, four: two blocks per SM, 256 columns of TMEM each) run at a time.  The special-function unit would be the next bound (16
// exponentials per clock and SM: 1024 cycles per 128 x 128 tile, as long as the products take at head_dim 128), so a part of the
// exponentials is computed by a polynomial on the FMA units.  Measured on a B200 with 2368 new tokens over 8192 keys, 32 heads on 8,
// L2 flushed: head_dim 128 fp16 pages 250 us, 1090 TFLOP/s (0.66 of the measured bf16 product rate), bf16 246 us, e4m3 336 us, 810 TFLOP/s;
// head_dim 64 209 us, 651 TFLOP/s, and 291 us.  Two warpgroups per row tile, each with half of the columns, were slower (261 against
// 231 us at head_dim 128, side by side): the exchange of the maxima costs more than the shorter chain gives.
//
// Keys and values: 16-bit pages come by TMA, one box per page and 64 columns (128-byte swizzle), the ids of a tile's pages read one
// tile ahead, a lane per page.  Slots behind the context and pages that do not exist are masked out of S, and their rows of V are
// cleared before the product (0 * NaN would reach every row).  Codes of e4m3 pages come 64 keys at a time; converting warps store
// them as 16-bit values (exact) and prepare the scales: with u_j = scale s_j k_scale_j + log2 v_scale_j the weights 2^(u_j - m) carry
// the value's scale, and the sum of exponentials takes 2^(u_j - m) / v_scale_j.
// Every wait is bounded (tcgen05.cuh).
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "paged.cuh"
#include "tcgen05.cuh"

namespace lbi {
namespace paged {

using namespace tc;

constexpr int ROWS = 128;                  // rows of a tile
constexpr int COPY_KEYS = 64;              // keys of one copy of codes

template <bool E4M3, int DH>
struct TcConfig {
  static constexpr int BLOCKS = DH == 64 && !E4M3 ? 2 : 1;        // per SM
  static constexpr int KEYS = DH == 64 && !E4M3 ? 64 : 128;       // of a tile
  static constexpr int SLOTS = DH == 128 ? 4 : E4M3 ? 8 : 6;      // K_0, V_0, K_1, V_1, ...
  // Masks and scales of a key tile: K_j is stored when S_(j - SLOTS / 2) is complete, which follows the softmax of the tile before
  // that one, so SLOTS / 2 + 2 entries never meet one that is still read.
  static constexpr int META = SLOTS / 2 + 2;
  static constexpr int RAW = E4M3 ? (DH == 128 ? 3 : 6) : 1;        // copies of codes on their way to the converting warps
  // warps 0-3, 4-7 softmax; 8 products; 9 copies; 16-bit pages: 10 clears V; e4m3: 10 and 11 scales, 12-15 conversion
  static constexpr int CONVERT = E4M3 ? 4 : 0, FIRST_CONVERT = 12;
  static constexpr int THREADS = 384 + CONVERT * 32;
  // Registers at launch and of the warpgroups afterwards (softmax, warps 8-11, conversion): claimed ones come from those that the
  // block was launched with and others have released, so the shares add up to at most threads x LAUNCH.
  static constexpr int LAUNCH = E4M3 ? 128 : DH == 64 ? 80 : 168;
  static constexpr int SOFTMAX = E4M3 ? 200 : DH == 64 ? 96 : 224, ISSUE = E4M3 || DH == 64 ? 48 : 56, WIDE = 64;
  static_assert(256 * SOFTMAX + 128 * ISSUE + CONVERT * 32 * WIDE <= THREADS * LAUNCH, "register shares");
  static constexpr int TMEM = DH == 64 && !E4M3 ? 256 : 512;
  // Of every 8 pairs of exponentials so many by the polynomial.  Measured at 0 / 2 / 3 / 4, 2368 tokens over 8192 keys, 32 heads:
  // head_dim 128 261 / 232 / 229 / 235 us, head_dim 64 206 / 201 / 217 / 224 us.  e4m3: none; the conversion takes the issue slots (2:
  // 464 against 314 us).
  static constexpr int POLY = E4M3 ? 0 : DH == 64 ? 2 : 3;
  // e4m3, where the columns suffice: Q is read from TMEM, too.  Shared memory is what runs short there (the conversion writes 2 bytes
  // per code, the softmax reads scales).
  static constexpr bool Q_IN_TMEM = E4M3 && DH == 64;
  static_assert(2 * KEYS + 2 * DH + (Q_IN_TMEM ? DH : 0) <= TMEM, "columns");
};

template <int KEYS>
struct alignas(16) KeyMeta {
  uint32_t there[4];                       // which of the tile's keys exist
  // e4m3, for two neighbouring keys: scale * log2(e) * k_scale of both, log2 v_scale of both; 1 / v_scale
  float ks_lv[KEYS / 2][4], iv[KEYS];
};

template <bool E4M3, int DH>
struct TcSmem {
  using C = TcConfig<E4M3, DH>;
  alignas(1024) uint8_t q[2][C::Q_IN_TMEM ? 512 : ROWS * DH * 2];
  alignas(1024) uint8_t kv[C::SLOTS][C::KEYS * DH * 2];
  alignas(1024) uint8_t raw[C::RAW][E4M3 ? COPY_KEYS * DH : 16];
  KeyMeta<E4M3 ? C::KEYS : 4> meta[C::META];
  uint64_t bar_raw_full[C::RAW];
  uint64_t bar_raw_empty[C::RAW];
  uint64_t bar_q;
  uint64_t bar_full[C::SLOTS];
  uint64_t bar_empty[C::SLOTS];
  uint64_t bar_clean[C::SLOTS];            // 16-bit pages: V without the rows that belong to no key
  uint64_t bar_s[2];                       // S_g(j) is there (and O_g holds tile j - 1)
  uint64_t bar_p[2];                       // P_g(j) is there, O_g is scaled for it
  uint64_t bar_o[2];                       // O_g is complete
  uint32_t tmem_base;
  volatile int abort_flag;
};

// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 32 lanes x 16 consecutive 32-bit columns, from registers.
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15 "
      "};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 16 lanes x 128 columns: thread t gets, for every 8 columns, columns 2 (t % 4) and + 1 of rows t / 4 and t / 4 + 8.
__device__ __forceinline__ void tmem_ld_16x128(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x16.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63 "
      "}, [%64];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}
// 16 lanes x 32 columns in the same spread: column t % 4 of every 4, rows t / 4 and t / 4 + 8.
__device__ __forceinline__ void tmem_st_16x32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%16], {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15 "
      "};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
template <int N>
__device__ __forceinline__ void claim_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void release_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// 2^x for x in [-126, 128) on the FMA units, for the share of the exponentials that the special-function unit has no time for:
// x = n + f with n the nearest whole number, 2^f by the minimax polynomial of degree 3 (bf16; relative error 7.5e-5, a fiftieth of the
// half step to which P is rounded) or 4 (fp16; 2.6e-6) on [-1/2, 1/2], n added to the exponent.
template <int TYPE>
__device__ __forceinline__ float2 exp2_by_polynomial(float2 x) {
  x = make_float2(fmaxf(x.x, -126.f), fmaxf(x.y, -126.f));
  const float2 t = add2(x, make_float2(12582912.f, 12582912.f));   // 1.5 * 2^23: n in the low bits
  const float2 n = add2(t, make_float2(-12582912.f, -12582912.f));
  const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
  float2 r;
  if (TYPE == LBI_F16) {
    r = fma2(make_float2(0.009570102207362652f, 0.009570102207362652f), f, make_float2(0.05591785907745361f, 0.05591785907745361f));
    r = fma2(r, f, make_float2(0.240247443318367f, 0.240247443318367f));
    r = fma2(r, f, make_float2(0.6931217908859253f, 0.6931217908859253f));
    r = fma2(r, f, make_float2(0.9999992847442627f, 0.9999992847442627f));
  } else {
    r = fma2(make_float2(0.0551716685295105f, 0.0551716685295105f), f, make_float2(0.2426111251115799f, 0.2426111251115799f));
    r = fma2(r, f, make_float2(0.6932609677314758f, 0.6932609677314758f));
    r = fma2(r, f, make_float2(0.9999280571937561f, 0.9999280571937561f));
  }
  return make_float2(__int_as_float(__float_as_int(r.x) + (__float_as_int(t.x) << 23)), __int_as_float(__float_as_int(r.y) + (__float_as_int(t.y) << 23)));
}

// Two weights as a word of P.  The largest is 2^15 or 2^8, but behind scores so large that their steps are whole binades the rounding of
// score and maximum may add some: fp16 then takes its largest number, not infinity.
template <int TYPE>
__device__ __forceinline__ uint32_t pack_weights(float a, float b) {
  if (TYPE != LBI_F16) return pack16<TYPE>(a, b);
  uint32_t d;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  return d;
}

template <int TYPE, bool E4M3, int DH>
__global__ void __launch_bounds__(TcConfig<E4M3, DH>::THREADS, TcConfig<E4M3, DH>::BLOCKS)
attn_tiles_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttnArgs a) {
  using T = typename Elem<TYPE>::T;
  using C = TcConfig<E4M3, DH>;
  using Smem = TcSmem<E4M3, DH>;
  constexpr int KEYS = C::KEYS, SLOTS = C::SLOTS, META = C::META, RAW = C::RAW, PANELS = DH / 64;
  constexpr float UP = TYPE == LBI_F16 ? 11.f : 0.f;        // P is held times 2^UP
  constexpr float GROWTH = UP + (TYPE == LBI_F16 ? 4.f : 8.f);   // binary logarithm of the largest P
  // ... the sum of exponentials of e4m3 pages without the factor, which its range (1 / v_scale) has no room for
  constexpr float DOWN = E4M3 && TYPE == LBI_F16 ? 1.f / 2048.f : 1.f;
  constexpr int Q_BYTES = ROWS * DH * 2, Q_PANEL = ROWS * 128, KV_BYTES = KEYS * DH * 2, KV_PANEL = KEYS * 128;   // panels of 64 columns
  extern __shared__ uint8_t raw_smem[];
  Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  const lbi_paged_batch& p = a.b;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (a.zero_tail && !a.part_o) zero_rows_of_nobody(p, (T*)a.out, a.heads * DH);

  // ------------------------------------------------------------------ the block's rows and keys
  const int64_t unit_block = (int64_t)gridDim.x - 1 - blockIdx.x;   // late tokens walk more keys: first
  const int split = (int)(unit_block % a.splits);
  const int64_t unit = unit_block / a.splits;
  const int kh = (int)(unit % p.kv_heads);
  const int64_t tile = unit / p.kv_heads;
  const int b = seq_of_tile(p, tile, a.group, 2 * ROWS);
  const int2 r = seq_rows(p, b);
  const int64_t local64 = (tile - first_tile(p, b, a.group, 2 * ROWS)) * (2 * ROWS);
  const int64_t rows_b = (int64_t)(r.y - r.x) * a.group;
  if (local64 < 0 || local64 >= rows_b) return;
  const int local = (int)local64, n_rows = (int)min((int64_t)2 * ROWS, rows_b - local64);
  const int first_pos = __ldg(p.context + b) - (r.y - r.x);
  const int64_t capacity = (int64_t)p.table_width << a.page_shift;
  const int k0 = split * a.split_keys;
  int k_end = 0;            // one behind the last key that any row sees
  auto key_tiles = [&](int g) {   // of row tile g

    const int last = min(n_rows, (g + 1) * ROWS) - 1;   // the tile's last row
    const int64_t seen = last < g * ROWS ? 0 : (int64_t)first_pos + (local + last) / a.group + 1;
    const int keys = (int)min(seen, capacity);
    if (seen > capacity && split == 0 && threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, 84);   // the table ends before the context
    const int k1 = split == a.splits - 1 ? keys : min(keys, k0 + a.split_keys);
    k_end = max(k_end, k1);
    return k1 > k0 ? (k1 - k0 + KEYS - 1) / KEYS : 0;
  };
  // two variables, not an array, which an index known at run time only would put into local memory
  const int n_kv0 = key_tiles(0), n_kv1 = key_tiles(1), n_j = max(n_kv0, n_kv1);

  if (threadIdx.x == 0) {
    s.abort_flag = 0;
    mbar_init(&s.bar_q, 8);
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&s.bar_full[i], E4M3 ? C::CONVERT + (i % 2 == 0 ? 2 : 0) : 1);   // K comes with its scales
      mbar_init(&s.bar_empty[i], 1);
      mbar_init(&s.bar_clean[i], 1);
    }
    for (int i = 0; i < RAW; ++i) {
      mbar_init(&s.bar_raw_full[i], 1);
      mbar_init(&s.bar_raw_empty[i], E4M3 ? C::CONVERT : 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.bar_s[i], 1);
      mbar_init(&s.bar_p[i], 4);
      mbar_init(&s.bar_o[i], 1);
    }
    fence_barrier_init();
    prefetch_tmap(&map_k);
    prefetch_tmap(&map_v);
  }
  if (warp == 8) tmem_alloc(&s.tmem_base, C::TMEM);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = s.tmem_base;
  volatile int* abortp = &s.abort_flag;

  if (warp >= 12) {
    // ======================================================================== converting warps: codes -> 16-bit values
    release_registers<C::WIDE>();
    if constexpr (E4M3) {
      constexpr int THREADS = C::CONVERT * 32, CHUNKS = COPY_KEYS * DH / 16 / THREADS;    // 16-byte chunks of codes per thread and copy
      const int tid = threadIdx.x - C::FIRST_CONVERT * 32;
      // Which row and 16-byte chunk of codes a thread takes: eight neighbouring threads read and write without bank conflicts.
      // head_dim 64: two rows of four chunks.  head_dim 128: four chunks of the rows r and r ^ 5, which differ in the bit that decides
      // between the halves of the swizzled row of codes and in the lowest, which decides between the even and the odd chunks of the
      // converted row.
      const int row0 = DH == 128 ? (tid >> 6) * 8 + (tid & 4 ? (tid >> 3 & 3) ^ 5 : tid >> 3 & 3) : tid >> 2;
      const int chunk = DH == 128 ? (tid >> 5 & 1) * 4 + (tid & 3) : tid & 3;
      const int from = row0 * DH + ((DH == 128 ? chunk ^ (row0 & 7) : chunk) << 4);
      const int to0 = (chunk >> 2) * KV_PANEL + row0 * 128 + (((2 * (chunk & 3)) ^ (row0 & 7)) << 4), to1 = to0 ^ 16;
      constexpr int STEP = THREADS * 16 / DH;          // rows between a thread's chunks: a multiple of 8
      static_assert(STEP % 8 == 0, "the swizzle repeats");
      bool ok = true;
      for (int n = 0; n < 2 * n_j && ok; ++n) {        // K_0, V_0, K_1, ...
        const int st = n % SLOTS;
        for (int half = 0; half < KEYS / COPY_KEYS && ok; ++half) {
          const int nr = n * (KEYS / COPY_KEYS) + half, sr = nr % RAW;
          ok = mbar_wait(&s.bar_raw_full[sr], (nr / RAW) & 1, abortp, p.status, 48);
          if (!ok) break;
          uint4 raw[CHUNKS];
#pragma unroll
          for (int i = 0; i < CHUNKS; ++i) raw[i] = *reinterpret_cast<const uint4*>(s.raw[sr] + from + i * STEP * DH);
          if (half == 0 && n >= SLOTS) ok = mbar_wait(&s.bar_empty[st], ((n / SLOTS) - 1) & 1, abortp, p.status, 47);
          if (!ok) break;
          uint8_t* to = s.kv[st] + half * COPY_KEYS * 128;
#pragma unroll
          for (int i = 0; i < CHUNKS; ++i) {
            uint32_t x[8];
            codes_to_16<TYPE>(raw[i].x, x[0], x[1]);
            codes_to_16<TYPE>(raw[i].y, x[2], x[3]);
            codes_to_16<TYPE>(raw[i].z, x[4], x[5]);
            codes_to_16<TYPE>(raw[i].w, x[6], x[7]);
            *reinterpret_cast<uint4*>(to + to0 + i * STEP * 128) = make_uint4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<uint4*>(to + to1 + i * STEP * 128) = make_uint4(x[4], x[5], x[6], x[7]);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.bar_raw_empty[sr]);
        }
        if (!ok) break;
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.bar_full[st]);
      }
    }
  } else if (warp >= 8) {
    release_registers<C::ISSUE>();
    if (warp == 8) {
      // ====================================================================== MMA issuer (one thread)
      // The loop over g stays a loop, so that not all descriptors are kept in registers.
      if (elect_one()) {
        constexpr uint32_t F16_BITS = (1u << 7) | (1u << 10);
        constexpr uint32_t idesc_s = make_idesc_bf16(ROWS, KEYS, 0, 0) & (TYPE == LBI_F16 ? ~F16_BITS : ~0u);
        constexpr uint32_t idesc_o = make_idesc_bf16(ROWS, DH, 0, 1) & (TYPE == LBI_F16 ? ~F16_BITS : ~0u);
        const uint64_t kmajor = make_smem_desc(0, 16, 1024), mnmajor = make_smem_desc(0, KV_PANEL, 1024);
        const uint32_t q16 = smem_u32(s.q[0]) >> 4, kv16 = smem_u32(s.kv[0]) >> 4;
        auto issue_s = [&](int g, int n) {   // n: index of K_j in the slot sequence
          const uint64_t da = kmajor + (q16 + g * (Q_BYTES >> 4)), db = kmajor + (kv16 + (n % SLOTS) * (KV_BYTES >> 4));
#pragma unroll
          for (int kk = 0; kk < DH / 16; ++kk) {
            if (C::Q_IN_TMEM) mma_ts(tmem + g * KEYS, tmem + 2 * KEYS + 2 * DH + g * (DH / 2) + kk * 8, db + ((kk >> 2) * (KV_PANEL >> 4) + (kk & 3) * 2), idesc_s, kk);
            else mma_bf16(tmem + g * KEYS, da + ((kk >> 2) * (Q_PANEL >> 4) + (kk & 3) * 2), db + ((kk >> 2) * (KV_PANEL >> 4) + (kk & 3) * 2), idesc_s, kk);
          }
          mma_commit(&s.bar_s[g]);
        };
        auto wait_full = [&](int n) { return mbar_wait(&s.bar_full[n % SLOTS], (n / SLOTS) & 1, abortp, p.status, 41); };
        bool ok = n_j == 0 || (mbar_wait(&s.bar_q, 0, abortp, p.status, 42) && wait_full(0));
        if (ok && n_j > 0) {
          fence_after_sync();
#pragma unroll 1
          for (int g = 0; g < 2; ++g)
            if ((g == 0 ? n_kv0 : n_kv1) > 0) issue_s(g, 0);
          mma_commit(&s.bar_empty[0]);
        }
        for (int j = 0; j < n_j && ok; ++j) {
          const int nv = 2 * j + 1, nk = 2 * j + 2;
          const bool next_k = j + 1 < n_j;
          ok = wait_full(nv) && (E4M3 || mbar_wait(&s.bar_clean[nv % SLOTS], (nv / SLOTS) & 1, abortp, p.status, 51)) && (!next_k || wait_full(nk));
#pragma unroll 1
          for (int g = 0; g < 2 && ok; ++g) {
            const int n_g = g == 0 ? n_kv0 : n_kv1;
            if (j >= n_g) continue;
            ok = mbar_wait(&s.bar_p[g], j & 1, abortp, p.status, 43);
            if (!ok) break;
            fence_after_sync();
            const uint64_t db = mnmajor + (kv16 + (nv % SLOTS) * (KV_BYTES >> 4));
#pragma unroll
            for (int kk = 0; kk < KEYS / 16; ++kk)
              mma_ts(tmem + 2 * KEYS + g * DH, tmem + g * KEYS + kk * 8, db + 128 * kk, idesc_o, (j > 0 || kk > 0) ? 1u : 0u);
            if (j + 1 == n_g) mma_commit(&s.bar_o[g]);
            else issue_s(g, nk);
          }
          if (ok) {
            mma_commit(&s.bar_empty[nv % SLOTS]);
            if (next_k) mma_commit(&s.bar_empty[nk % SLOTS]);
          }
        }
      }
    } else if (warp == 9) {
      // ====================================================================== TMA producer: one lane per page
      constexpr int COPY = E4M3 ? COPY_KEYS : KEYS, COPIES = KEYS / COPY, RING = E4M3 ? RAW : SLOTS;   // keys of a ring entry
      const int box = min(p.page_size, COPY);    // rows of a box: a page, or an entry's part of it
      const int per = KEYS / box;                // boxes of a tile, 1 .. 16
      const int* table = p.table + (int64_t)b * p.table_stride;
      auto load_page = [&](int j) {
        const int pos = k0 + j * KEYS + lane * box;
        return j < n_j && lane < per && pos < k_end ? __ldg(table + (pos >> a.page_shift)) : -1;
      };
      int page = load_page(0);
      bool ok = true;
      for (int j = 0; j < n_j && ok; ++j) {
        const int next = load_page(j + 1);
        const int base = k0 + j * KEYS, pos = base + lane * box;
        const bool wanted = lane < per && pos < k_end;
        const bool good = wanted && page >= 0 && page < p.num_pages;
        if (wanted && !good && p.status) atomicCAS(p.status, 0, 84);
        const uint32_t boxes = __ballot_sync(0xffffffffu, good);
        const int row = (max(page, 0) * p.kv_heads + kh) * p.page_size + (pos & (p.page_size - 1));
        for (int i = 0; i < 2 * COPIES && ok; ++i) {
          const int v = i / COPIES, n = 2 * COPIES * j + i, st = n % RING;
          uint64_t* full = E4M3 ? &s.bar_raw_full[st] : &s.bar_full[st];
          if (n >= RING) ok = mbar_wait(E4M3 ? &s.bar_raw_empty[st] : &s.bar_empty[st], ((n / RING) - 1) & 1, abortp, p.status, 44);
          if (!ok) break;
          if (!E4M3 && v == 0 && lane < 4) {
            uint32_t there = 0;
            if (lane >= KEYS / 32 || (boxes == (1u << per) - 1u && base + KEYS <= k_end)) {
              there = 0xffffffffu;
            } else {
              for (int e = 0; e < 32; ++e) {
                const int key = lane * 32 + e;
                if ((boxes >> (key / box) & 1u) && base + key < k_end) there |= 1u << e;
              }
            }
            s.meta[j % META].there[lane] = there;
          }
          __syncwarp();   // the words of all four lanes before lane 0's arrival, which the readers wait for
          const int at = lane * box - (i % COPIES) * COPY;   // row in the entry
          const bool here = good && at >= 0 && at < COPY;
          const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, here)) * (uint32_t)box * DH * (E4M3 ? 1 : 2);
          if (lane == 0) mbar_arrive_expect_tx(full, bytes);
          __syncwarp();
          if (here) {
            if (E4M3) {
              tma_load_2d(s.raw[st] + at * DH, v ? &map_v : &map_k, full, 0, row);
            } else {
#pragma unroll
              for (int c = 0; c < PANELS; ++c) tma_load_2d(s.kv[st] + c * KV_PANEL + at * 128, v ? &map_v : &map_k, full, c * 64, row);
            }
          }
          __syncwarp();
        }
        page = next;
      }
    } else if (E4M3) {
      // ====================================================================== scales and presence of the keys, two per thread
      constexpr int EACH = KEYS / 64;
      const int key0 = threadIdx.x - 320;              // 0 .. 63
      const int* table = p.table + (int64_t)b * p.table_stride;
      int page[EACH];
      float k_scale[EACH], v_scale[EACH];
      bool good[EACH];
      auto load_pages = [&](int j) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          const int pos = k0 + j * KEYS + key0 + i * 64;
          page[i] = j < n_j && pos < k_end ? __ldg(table + (pos >> a.page_shift)) : -1;
        }
      };
      auto look_up = [&](int j) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          good[i] = page[i] >= 0 && page[i] < p.num_pages;
          const int slot = good[i] ? (page[i] * p.kv_heads + kh) * p.page_size + ((k0 + j * KEYS + key0 + i * 64) & (p.page_size - 1)) : 0;
          k_scale[i] = good[i] ? __ldg(p.k_scale + slot) : 0.f;
          v_scale[i] = good[i] ? __ldg(p.v_scale + slot) : 0.f;
        }
      };
      load_pages(0);
      look_up(0);
      load_pages(1);
      bool ok = true;
      for (int j = 0; j < n_j && ok; ++j) {
        const int n = 2 * j, st = n % SLOTS;
        if (n >= SLOTS) ok = mbar_wait(&s.bar_empty[st], ((n / SLOTS) - 1) & 1, abortp, p.status, 49);   // see META
        if (!ok) break;
        auto& meta = s.meta[j % META];
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          const int key = key0 + i * 64;
          const float vs = positive_scale(v_scale[i]);
          const uint32_t there = __ballot_sync(0xffffffffu, good[i]);
          meta.ks_lv[key >> 1][key & 1] = k_scale[i] * a.scale_log2;
          meta.ks_lv[key >> 1][2 + (key & 1)] = lg2(vs);
          meta.iv[key] = __frcp_rn(vs) * DOWN;
          if (lane == 0) meta.there[key >> 5] = there;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.bar_full[st]);
        look_up(j + 1);
        load_pages(j + 2);
      }
    } else if (warp == 10) {
      // ====================================================================== rows of V that belong to no key: 0 * NaN is NaN
      // (codes become finite values whatever they are)
      bool ok = true;
      for (int j = 0; j < n_j && ok; ++j) {
        const int nv = 2 * j + 1, st = nv % SLOTS;
        ok = mbar_wait(&s.bar_full[st], (nv / SLOTS) & 1, abortp, p.status, 52);
        if (!ok) break;
        const uint32_t* there = s.meta[j % META].there;
        if ((there[0] & there[1] & there[2] & there[3]) != 0xffffffffu) {
          for (int row = lane; row < KEYS; row += 32)
            if (!(there[row >> 5] >> (row & 31) & 1u)) {
              const uint32_t at = smem_u32(s.kv[st]) + row * 128;
#pragma unroll
              for (int c = 0; c < PANELS * 8; ++c)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at + (c >> 3) * KV_PANEL + (c & 7) * 16), "r"(0) : "memory");
            }
          fence_proxy_async();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.bar_clean[st]);
      }
    }
  } else {
    // ======================================================================== softmax warpgroups
    claim_registers<C::SOFTMAX>();
    const int g = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;             // of the tile
    const bool live = g * ROWS + row < n_rows;
    if constexpr (C::Q_IN_TMEM) {   // a thread's row into its lane, two elements per column
      const int at = local + g * ROWS + row;
      const T* src = (const T*)a.q + (int64_t)(r.x + (live ? at / a.group : 0)) * a.q_stride + (kh * a.group + (live ? at % a.group : 0)) * DH;
#pragma unroll
      for (int c = 0; c < DH / 32; ++c) {
        uint4 x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = live ? __ldg(reinterpret_cast<const uint4*>(src) + c * 4 + e) : make_uint4(0, 0, 0, 0);
        tmem_st_32x16(tmem + ((uint32_t)(quarter * 32) << 16) + 2 * KEYS + 2 * DH + g * (DH / 2) + c * 16, reinterpret_cast<const uint32_t*>(x));
      }
      tmem_st_wait();
      fence_before_sync();
    } else {   // 16-byte chunks of the warp's 32 rows, neighbouring lanes on neighbouring chunks, into the swizzled tile
      for (int i = lane; i < 32 * (DH / 8); i += 32) {
        const int rr = quarter * 32 + i / (DH / 8), c = i % (DH / 8);
        const int at = g * ROWS + rr;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (at < n_rows) {
          const int tok = (local + at) / a.group, head = kh * a.group + (local + at) % a.group;
          x = __ldg(reinterpret_cast<const uint4*>((const T*)a.q + (int64_t)(r.x + tok) * a.q_stride + head * DH) + c);
        }
        *reinterpret_cast<uint4*>(s.q[g] + (c >> 3) * Q_PANEL + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = x;
      }
      fence_proxy_async();
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.bar_q);

    const int mine = g == 0 ? n_kv0 : n_kv1;
    const uint32_t t_s = tmem + ((uint32_t)(quarter * 32) << 16) + g * KEYS;   // P too
    const uint32_t t_o = tmem + ((uint32_t)(quarter * 32) << 16) + 2 * KEYS + g * DH;
    auto rescale = [&](float keep) {
#pragma unroll
      for (int c = 0; c < DH / 16; ++c) {
        uint32_t o[16];
        tmem_ld_32x16(t_o + c * 16, o);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
        tmem_st_32x16(t_o + c * 16, o);
      }
    };
    auto hand_over = [&] {
      tmem_st_wait();
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.bar_p[g]);
    };
    // of the thread's row: the point that exponents are relative to, in base-2 logarithms (UP below a maximum), and the sum
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    if constexpr (E4M3) {
      // Every column has its own scales.  A thread per row would read all of them from shared memory, 393 KB per 128 keys, which
      // takes longer than the exponentials; in the spread of the 16-lane loads a thread has a quarter of the columns for four rows
      // (t / 4 + 8 k of the warp's 32) and reads a quarter of that.  A row is shared by the four threads of a quad.
      const int t = lane & 3;
      int lim[4];
      float mr[4], lr[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int rr = g * ROWS + quarter * 32 + (lane >> 2) + 8 * k;
        lim[k] = rr < n_rows ? first_pos + (local + rr) / a.group : -1;
        mr[k] = -INFINITY;
        lr[k] = 0.f;
      }
      constexpr int N = KEYS / 8;
      static_assert(N == 16, "one load per 16 lanes");
      for (int j = 0; j < mine; ++j) {
        ok = mbar_wait(&s.bar_s[g], j & 1, abortp, p.status, 45);
        if (!ok) break;
        fence_after_sync();
        const auto& meta = s.meta[j % META];
        union {   // [16 rows][8 columns][row + 8][column]
          uint32_t w[2][N * 4];
          float2 f2[2][N][2];
        } x;
#pragma unroll
        for (int h = 0; h < 2; ++h) tmem_ld_16x128(t_s + ((uint32_t)(16 * h) << 16), x.w[h]);
        tmem_ld_wait();
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const float4 f = *reinterpret_cast<const float4*>(meta.ks_lv[4 * n + t]);
#pragma unroll
          for (int k = 0; k < 4; ++k) x.f2[k >> 1][n][k & 1] = fma2(x.f2[k >> 1][n][k & 1], make_float2(f.x, f.y), make_float2(f.z, f.w));
        }
        const int base = k0 + j * KEYS;
        const bool masked = __any_sync(0xffffffffu, (meta.there[0] & meta.there[1] & meta.there[2] & meta.there[3]) != 0xffffffffu ||
                                                        min(min(lim[0], lim[1]), min(lim[2], lim[3])) - base < KEYS - 1);
        if (masked) {
#pragma unroll
          for (int n = 0; n < N; ++n) {
            const uint32_t bits = meta.there[n >> 2] >> ((n & 3) * 8 + 2 * t);
            const int key = base + 8 * n + 2 * t;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float2& u = x.f2[k >> 1][n][k & 1];
              if (!(bits & 1u) || key > lim[k]) u.x = -INFINITY;
              if (!(bits & 2u) || key + 1 > lim[k]) u.y = -INFINITY;
            }
          }
        }
        float top[4];
        bool grow = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
          for (int n = 0; n < N; n += 2) {
            const float2 u = x.f2[k >> 1][n][k & 1], w = x.f2[k >> 1][n + 1][k & 1];
            t0 = fmaxf(t0, fmaxf(u.x, u.y));
            t1 = fmaxf(t1, fmaxf(w.x, w.y));
          }
          top[k] = fmaxf(t0, t1);
          top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 1));
          top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 2));
          grow = grow || top[k] - mr[k] > GROWTH;
        }
        if (__any_sync(0xffffffffu, grow)) {
          float row_keep = 1.f;   // of row `lane`, for O
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float m_new = top[k] - mr[k] > GROWTH ? (UP == 0.f ? top[k] : __fadd_ru(top[k], -UP)) : mr[k];
            const float keep = mr[k] == m_new ? 1.f : ex2(mr[k] - m_new);
            mr[k] = m_new;
            lr[k] *= keep;
            const float k_row = __shfl_sync(0xffffffffu, keep, (lane & 7) * 4);
            if (lane >> 3 == k) row_keep = k_row;
          }
          if (j > 0) rescale(row_keep);
        }
        float2 neg[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float ref = mr[k] == -INFINITY ? 0.f : mr[k];
          neg[k] = make_float2(-ref, -ref);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int n0 = 0; n0 < N; n0 += 8) {
            uint32_t w[16];
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                float2& u = x.f2[h][n0 + n][k];
                u = add2(u, neg[2 * h + k]);
                u = make_float2(ex2(u.x), ex2(u.y));
                w[2 * n + k] = pack_weights<TYPE>(u.x, u.y);
              }
            tmem_st_16x32(t_s + ((uint32_t)(16 * h) << 16) + n0 * 4, w);
          }
        hand_over();
        // the sums are needed by nobody yet: behind the arrival
        float2 sum[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] = make_float2(lr[k], 0.f);
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const float2 iv = *reinterpret_cast<const float2*>(meta.iv + 8 * n + 2 * t);
#pragma unroll
          for (int k = 0; k < 4; ++k) sum[k] = fma2(x.f2[k >> 1][n][k & 1], iv, sum[k]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) lr[k] = sum[k].x + sum[k].y;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {   // to the thread of the row
        lr[k] += __shfl_xor_sync(0xffffffffu, lr[k], 1);
        lr[k] += __shfl_xor_sync(0xffffffffu, lr[k], 2);
        const float l_row = __shfl_sync(0xffffffffu, lr[k], (lane & 7) * 4), m_row = __shfl_sync(0xffffffffu, mr[k], (lane & 7) * 4);
        if (lane >> 3 == k) {
          l = l_row;
          m = m_row;
        }
      }
    } else {
      const int limit = live ? first_pos + (local + g * ROWS + row) / a.group : -1;
      float2 l2 = make_float2(0.f, 0.f);
      for (int j = 0; j < mine; ++j) {
        ok = mbar_wait(&s.bar_s[g], j & 1, abortp, p.status, 45);
        if (!ok) break;
        fence_after_sync();
        const auto& meta = s.meta[j % META];
        union {   // the row of S
          uint32_t w[KEYS];
          float f[KEYS];
          float2 f2[KEYS / 2];
        } x;
#pragma unroll
        for (int c = 0; c < KEYS / 32; ++c) tmem_ld_32x32(t_s + c * 32, x.w + c * 32);
        tmem_ld_wait();
        const int rel = limit - (k0 + j * KEYS);     // the row's last key, counted from the tile's first
        const uint4 there = *reinterpret_cast<const uint4*>(meta.there);
        const bool masked = __any_sync(0xffffffffu, (there.x & there.y & there.z & there.w) != 0xffffffffu || rel < KEYS - 1);
        if (masked) {
#pragma unroll
          for (int c = 0; c < KEYS / 32; ++c) {
            const int e0 = rel - 32 * c;
            const uint32_t seen = meta.there[c] & (e0 >= 31 ? 0xffffffffu : e0 < 0 ? 0u : (2u << e0) - 1u);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(seen >> e & 1u)) x.f[c * 32 + e] = -INFINITY;
          }
        }
        float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < KEYS; e += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i) t4[i] = fmaxf(t4[i], fmaxf(x.f[e + i], x.f[e + 4 + i]));
        const float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * a.scale_log2;   // positive, see the choice of the kernel
        // the reference point follows only a growth to more than 2^GROWTH
        const bool grow = top - m > GROWTH;
        if (__any_sync(0xffffffffu, grow)) {
          const float m_new = grow ? (UP == 0.f ? top : __fadd_ru(top, -UP)) : m;
          const float keep = m == m_new ? 1.f : ex2(m - m_new);
          m = m_new;
          l2.x *= keep;
          l2.y *= keep;
          if (j > 0) rescale(keep);
        }
        const float ref = m == -INFINITY ? 0.f : m;
        const float2 neg = make_float2(-ref, -ref), sc = make_float2(a.scale_log2, a.scale_log2);
        auto exponentials = [&](auto by_polynomial) {
#pragma unroll
          for (int c = 0; c < KEYS / 32; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float2& u = x.f2[c * 16 + e];
              u = fma2(u, sc, neg);
              if (decltype(by_polynomial)::value && e % 8 < C::POLY) u = exp2_by_polynomial<TYPE>(u);
              else u = make_float2(ex2(u.x), ex2(u.y));
              w[e] = pack_weights<TYPE>(u.x, u.y);
            }
            tmem_st_32x16(t_s + c * 16, w);
          }
        };
        if (masked) exponentials(std::false_type{});   // 2^-inf is 0 there, the polynomial's smallest value is 2^-126
        else exponentials(std::true_type{});
        hand_over();
        // the sum is needed by nobody yet: behind the arrival
        float2 sum[4] = {l2, make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int e = 0; e < KEYS / 2; ++e) sum[e & 3] = add2(sum[e & 3], x.f2[e]);
        l2 = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
      }
      l = l2.x + l2.y;
    }
    if (ok && mine > 0) ok = mbar_wait(&s.bar_o[g], 0, abortp, p.status, 46);
    if (ok) {
      fence_after_sync();
      const float inv = l == 0.f ? 0.f : DOWN / l;
      const int at = local + g * ROWS + row;
      const int64_t o_row = (int64_t)(r.x + at / a.group) * a.heads + kh * a.group + at % a.group;
#pragma unroll
      for (int c = 0; c < DH / 32; ++c) {
        uint32_t x[32];
        if (mine > 0) {
          tmem_ld_32x32(t_o + c * 32, x);
          tmem_ld_wait();
        }
        if (live) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = mine > 0 ? __uint_as_float(x[e + i]) * inv : 0.f;
            if (a.part_o) store_f<float, 8>(a.part_o + (o_row * a.splits + split) * DH + c * 32 + e, f);
            else store_f<T, 8>((T*)a.out + o_row * DH + c * 32 + e, f);
          }
        }
      }
      if (live && a.part_o) a.part_lse[o_row * a.splits + split] = l == 0.f ? -INFINITY : m + log2f(l);
    }
  }

  // ---------------------------------------------------------------------- teardown
  __syncwarp();
  if (s.abort_flag) {
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 2000000ull) __nanosleep(1000);  // let copies in flight land before smem is released
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 8) {
    fence_after_sync();
    tmem_dealloc(tmem, C::TMEM);
  }
}

// ------------------------------------------------------------------------------------------------ host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                  CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &res) == cudaSuccess && res == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

template <int TYPE, bool E4M3, int DH>
static int launch_tiles(const AttnArgs& a, cudaStream_t st) {
  CUtensorMap map[2];
  EncodeTiledFn fn = encode_fn();
  if (!fn) return 801;
  const cuuint64_t dims[2] = {DH, (cuuint64_t)a.b.num_pages * a.b.kv_heads * a.b.page_size};
  const cuuint64_t strides[1] = {E4M3 ? DH : DH * 2};
  const cuuint32_t box[2] = {E4M3 ? DH : 64, (cuuint32_t)std::min(a.b.page_size, E4M3 ? COPY_KEYS : TcConfig<E4M3, DH>::KEYS)}, estr[2] = {1, 1};
  for (int v = 0; v < 2; ++v) {
    const CUresult rc = fn(&map[v], E4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : TYPE == LBI_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                           v ? a.b.v : a.b.k, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           E4M3 && DH == 64 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return 1000 + (int)rc;
  }
  auto kernel = attn_tiles_kernel<TYPE, E4M3, DH>;
  const int smem = (int)sizeof(TcSmem<E4M3, DH>) + 1024;
  static lbi::PerDeviceOnce once;
  cudaError_t e = once.max_dynamic_smem(kernel, smem);
  if (e != cudaSuccess) return (int)e;
  // the claims of the warpgroups add up to what a block gets at launch only if the kernel was compiled to this many registers
  static const bool registers_add_up = [&] {
    cudaFuncAttributes attr;
    return cudaFuncGetAttributes(&attr, kernel) == cudaSuccess && attr.numRegs == TcConfig<E4M3, DH>::LAUNCH;
  }();
  if (!registers_add_up) return (int)cudaErrorInvalidConfiguration;
  const int64_t blocks = tile_bound(a.b, a.group, 2 * ROWS) * a.b.kv_heads * a.splits;
  if (blocks >= (1ll << 31)) return (int)cudaErrorInvalidValue;
  kernel<<<(unsigned)blocks, TcConfig<E4M3, DH>::THREADS, smem, st>>>(map[0], map[1], a);
  return (int)cudaGetLastError();
}

int launch_attn_tiles(const AttnArgs& a, int type, cudaStream_t st) {
  const bool e4m3 = a.b.cache_type == LBI_E4M3, wide = a.b.head_dim == 128;
  if (type == LBI_BF16)
    return e4m3 ? (wide ? launch_tiles<LBI_BF16, true, 128>(a, st) : launch_tiles<LBI_BF16, true, 64>(a, st))
                : (wide ? launch_tiles<LBI_BF16, false, 128>(a, st) : launch_tiles<LBI_BF16, false, 64>(a, st));
  return e4m3 ? (wide ? launch_tiles<LBI_F16, true, 128>(a, st) : launch_tiles<LBI_F16, true, 64>(a, st))
              : (wide ? launch_tiles<LBI_F16, false, 128>(a, st) : launch_tiles<LBI_F16, false, 64>(a, st));
}

}  // namespace paged
}  // namespace lbi
