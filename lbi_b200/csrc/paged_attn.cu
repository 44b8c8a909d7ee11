// Causal attention of new tokens over a paged key / value cache.
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j   over the positions j <= context - new + i of the sequence; no position: o_i = 0.
//
// Kernels:
//   attn_rows_kernel   8 or 16 query rows at a time (tokens x heads of a group) for 16-bit queries: decoding, a few new tokens.
//   attn_tiles_kernel  256 rows at a time on tcgen05 (paged_attn_tc.cu): chunks of a prompt.
//   attn_any_kernel    16 rows at a time in (almost) full precision: fp32 queries, and head sizes that the other tiles do not cover.
//   combine_kernel     joins the parts of a long context.
#include <algorithm>

#include "paged.cuh"

namespace lbi {
namespace paged {

// ------------------------------------------------------------------------------------------------ tiles of 8 and 16 rows
// Bound by reading the cache once: 2 head_dim sizeof(code) bytes per key and kv head.  All query heads of a group (and several new
// tokens, if there are) share a tile of 8 or 16 rows, so that one read of a key serves them all, and mma.sync m16n8k16 does the
// products with the keys (then the head's elements) as its 16 rows and the query rows as its 8 columns: S^T = K Q^T, O^T = V^T P^T.
// With at most 16 rows the tensor work is a few per cent of the time, and the operands come straight from the copies below, which
// tcgen05 (128 rows, operands through descriptors) would only add steps to.  P^T leaves the first product with a key's rows in one
// thread and enters the second with a row's keys in one thread: movmatrix turns it.  Every warp works alone on its own keys: a ring of
// cp.async tiles in shared memory (no block barrier in the loop), running maximum and sum, O^T in registers; the four warps of a block
// are joined through shared memory at the end.  The page ids of a tile are loaded one tile ahead of its copies.
//
// e4m3 pages: codes become fp16 values exactly.  With u_j = scale s_j k_scale_j + log2 v_scale_j the weights 2^(u_j - max u) carry
// the value's scale (fp16 has no range for p * v_scale); the sum of exponentials takes 2^(u_j - max u) / v_scale_j.
// P is rounded to the 16-bit type of the products before the second one (half a step of that type, as the result itself is rounded);
// maximum, sum and output stay in fp32.  fp16 keeps that half step only down to 2^-14, and the keys of a long context may all weigh
// less than that beside one heavy key: products in fp16 hold the weights times 2^15, so that the half step holds down to 2^-29 of
// the heaviest key and what is lost below, 2^-40 of it per key, is nothing to the result.
//
// Measured on a B200, 32 query heads on 8 of 128: 64 contexts of up to 8192 keys (ragged, 1.02 GB) 183 us, 5.6 TB/s, 0.85 of the copy
// bandwidth; all 8192 long 0.94 of it.  e4m3: 2 contexts of 131072 keys (0.55 GB) 115 to 117 us, 4.8 TB/s, 0.73: the codes' way to
// fp16 takes the issue slots (57 % busy) that the 16-bit pages leave free (26 %).

constexpr int ROW_TILE = 16;   // rows of attn_any_kernel; attn_rows_kernel has tiles of 8, too
constexpr int WARPS = 4;

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool fill) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(fill ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool fill) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(fill ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
template <int TYPE>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if (TYPE == LBI_F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16-byte chunk c of row r in a tile of RB-byte rows: eight rows that are read at the same chunk lie in eight different bank groups.
template <int RB>
__device__ __forceinline__ uint32_t swz(int r, int c) {
  constexpr int PER = RB / 16;                 // chunks per row
  constexpr int IN_LINE = PER < 8 ? PER : 8;   // ... of one 128-byte line
  constexpr int ROWS = 8 / IN_LINE;            // rows per line
  return (uint32_t)(r * RB + ((c ^ ((r / ROWS) & (IN_LINE - 1))) << 4));
}

// What a block of 16 rows works on.
struct RowsUnit {
  int split, kh, b, first_row, local, n_rows, first_pos, k0, k1;   // local: first row of the tile in the sequence's tile space
  bool any;
};
__device__ __forceinline__ RowsUnit rows_unit(const AttnArgs& a, int per_tile) {
  const lbi_paged_batch& p = a.b;
  RowsUnit u;
  u.split = blockIdx.x % a.splits;
  const int64_t unit = blockIdx.x / a.splits;
  u.kh = (int)(unit % p.kv_heads);
  const int64_t tile = unit / p.kv_heads;
  u.b = seq_of_tile(p, tile, a.group, per_tile);
  const int2 r = seq_rows(p, u.b);
  u.first_row = r.x;
  u.local = (int)(tile - first_tile(p, u.b, a.group, per_tile)) * per_tile;
  const int rows_b = (r.y - r.x) * a.group;
  u.any = u.local >= 0 && u.local < rows_b;
  u.n_rows = min(per_tile, rows_b - u.local);
  u.first_pos = __ldg(p.context + u.b) - (r.y - r.x);              // position of the sequence's first new token
  const int64_t capacity = (int64_t)p.table_width << a.page_shift;
  const int64_t seen = (int64_t)u.first_pos + (u.local + u.n_rows - 1) / a.group + 1;
  const int keys = (int)min(seen, capacity);
  if (u.any && seen > capacity && u.split == 0 && threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, 84);   // the table ends before the context
  u.k0 = u.split * a.split_keys;
  u.k1 = u.split == a.splits - 1 ? keys : min(keys, u.k0 + a.split_keys);
  return u;
}
// Slot of key `lane` of a tile that starts at `base`, or -1 where there is no such key or page.
__device__ __forceinline__ int key_slot(const AttnArgs& a, const RowsUnit& u, int pos, bool wanted, int page) {
  const lbi_paged_batch& p = a.b;
  if (!wanted) return -1;
  if (page >= 0 && page < p.num_pages) return (page * p.kv_heads + u.kh) * p.page_size + (pos & (p.page_size - 1));
  if (p.status) atomicCAS(p.status, 0, 84);
  return -1;
}
// Joins the warps of a block and stores the result (or the part): references and sums of the warps' rows in `ml`, the output row parts
// behind them as [warp][row][dim + 4].
template <typename T, int ROWS>
__device__ __forceinline__ void join_and_store(const AttnArgs& a, const RowsUnit& u, const float* ml, int dim) {
  const float* os = ml + 2 * WARPS * ROWS;
  for (int i = threadIdx.x; i < u.n_rows * (dim / 8); i += WARPS * 32) {
    const int rr = i / (dim / 8), d = i % (dim / 8) * 8;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, ml[w * ROWS + rr]);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f, acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = ex2(ml[w * ROWS + rr] - ref);
      sum += f * ml[(WARPS + w) * ROWS + rr];
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += f * os[(w * ROWS + rr) * (dim + 4) + d + e];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= inv;
    const int64_t at = (int64_t)(u.first_row + (u.local + rr) / a.group) * a.heads + u.kh * a.group + (u.local + rr) % a.group;
    if (a.part_o) {
      store_f<float, 8>(a.part_o + (at * a.splits + u.split) * dim + d, acc);
      if (d == 0) a.part_lse[at * a.splits + u.split] = sum == 0.f ? -INFINITY : top + log2f(sum);
    } else {
      store_f<T, 8>((T*)a.out + at * dim + d, acc);
    }
  }
}

template <bool E4M3, int DH, int KEYS, int STAGES, int NT>
struct RowsTile {
  static constexpr int ROWS = 8 * NT;
  static constexpr int RB = DH * (E4M3 ? 1 : 2);
  static constexpr int TILE = KEYS * RB;
  static constexpr int STAGE = 2 * TILE + (E4M3 ? 8 * KEYS : 0) + 16;   // K, V, scales, which keys exist
  static constexpr int RING = STAGES * STAGE;
  static constexpr int JOIN = WARPS * ROWS * (DH + 4) * 4 + WARPS * ROWS * 8;
  static constexpr int SMEM = WARPS * RING > JOIN ? WARPS * RING : JOIN;
};

// An 8 x 8 matrix of 16-bit values, two per thread, transposed across the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int TYPE, bool E4M3, int DH, int KEYS, int STAGES, int BLOCKS, int NT>
__global__ void __launch_bounds__(WARPS * 32, BLOCKS) attn_rows_kernel(const AttnArgs a) {
  using T = typename Elem<TYPE>::T;
  using L = RowsTile<E4M3, DH, KEYS, STAGES, NT>;
  constexpr int ROWS = L::ROWS, KT = KEYS / 16;
  constexpr int MATH = E4M3 ? LBI_F16 : TYPE;             // of the products
  constexpr float UP = MATH == LBI_F16 ? 15.f : 0.f;      // weights are held times 2^UP
  // ... the sum of exponentials of e4m3 pages without the factor, which its range (1 / v_scale) has no room for
  constexpr float DOWN = E4M3 ? 1.f / 32768.f : 1.f;
  extern __shared__ __align__(128) uint8_t smem[];
  const lbi_paged_batch& p = a.b;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (a.zero_tail && !a.part_o) zero_rows_of_nobody(p, (T*)a.out, a.heads * DH);
  const RowsUnit u = rows_unit(a, ROWS);
  if (!u.any) return;
  const int kh = u.kh, k0 = u.k0, k1 = u.k1;

  // Query fragments: row 8 n + g of the tile.  The order of the head's elements within a product of 16 is free as long as Q and K
  // agree: natural for 16-bit pages (ldmatrix), 4 neighbours per thread for codes (one 32-bit load).
  // e4m3: the products run in fp16, which holds the codes and, behind a power of two per row that brings its largest element to
  // [2^14, 2^15), a bf16 query as well (29 binades below the largest to the normal range's end: nothing that an fp32 sum would notice).
  uint32_t qf[NT][DH / 16][2];
  int limit[NT][2];         // of the rows 8 n + 2 t and + 1, whose scores the thread has
  float row_scale[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 8 * n + g, rr = u.local + r;
    const bool live = r < u.n_rows;
    const int token = live ? rr / a.group : 0, head = kh * a.group + (live ? rr % a.group : 0);
    const uint32_t* src = reinterpret_cast<const uint32_t*>((const T*)a.q + (int64_t)(u.first_row + token) * a.q_stride + head * DH);
#pragma unroll
    for (int ks = 0; ks < DH / 16; ++ks) {
      qf[n][ks][0] = live ? src[ks * 8 + (E4M3 ? 2 * t : t)] : 0u;
      qf[n][ks][1] = live ? src[ks * 8 + (E4M3 ? 2 * t + 1 : t + 4)] : 0u;
    }
    float scale = a.scale_log2;
    if (E4M3 && TYPE == LBI_BF16) {
      int most = 0;   // as whole numbers, magnitudes are in order
#pragma unroll
      for (int ks = 0; ks < DH / 16; ++ks)
#pragma unroll
        for (int i = 0; i < 2; ++i) most = max(most, max((int)(qf[n][ks][i] << 16 & 0x7fff0000u), (int)(qf[n][ks][i] & 0x7fff0000u)));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int e = min(max(14 + 127 - (most >> 23), -100), 120);
      const float up = __int_as_float((e + 127) << 23);
      scale *= __int_as_float((127 - e) << 23);
#pragma unroll
      for (int ks = 0; ks < DH / 16; ++ks)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t& w = qf[n][ks][i];
          w = pack16<LBI_F16>(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up);
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int at = 8 * n + 2 * t + e;
      row_scale[n][e] = __shfl_sync(0xffffffffu, scale, (2 * t + e) * 4);
      // rows that do not exist (queries of zero, never stored) ask for no mask
      limit[n][e] = at < u.n_rows ? u.first_pos + (u.local + at) / a.group : 0x7fffffff;
    }
  }
  int lowest = min(limit[0][0], limit[0][1]);
  if (NT == 2) lowest = min(lowest, min(limit[NT - 1][0], limit[NT - 1][1]));
  float o[DH / 16][NT][4];
#pragma unroll
  for (int i = 0; i < DH / 16; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][n][e] = 0.f;
  float m[NT][2], l[NT][2];   // what the exponents are relative to: the running maximum less UP
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) m[n][e] = -INFINITY, l[n][e] = 0.f;

  const uint32_t ring = smem_addr(smem) + warp * L::RING;
  const int n_tiles = k1 > k0 ? (k1 - k0 + KEYS - 1) / KEYS : 0;
  const int mine = n_tiles > warp ? (n_tiles - warp + WARPS - 1) / WARPS : 0;      // tiles warp, warp + 4, ...
  const int* table = p.table + (int64_t)u.b * p.table_stride;
  auto load_page = [&](int i) {   // page id of key `lane` of this warp's i-th tile; -1: not there
    const int pos = k0 + (warp + i * WARPS) * KEYS + lane;
    return i < mine && lane < KEYS && pos < k1 ? __ldg(table + (pos >> a.page_shift)) : -1;
  };
  auto copy_tile = [&](int i, int page) {
    const int st = i % STAGES;
    const int pos = k0 + (warp + i * WARPS) * KEYS + lane;
    const int slot = key_slot(a, u, pos, lane < KEYS && pos < k1, page);
    const uint32_t kd = ring + st * L::STAGE, vd = kd + L::TILE;
    constexpr int CH = L::RB / 16;
#pragma unroll
    for (int j = 0; j < KEYS * CH / 32; ++j) {
      const int row = (j * 32 + lane) / CH, c = lane % CH;
      const int s = __shfl_sync(0xffffffffu, slot, row);
      const int64_t off = (int64_t)max(s, 0) * L::RB + c * 16;
      cp_async16(kd + swz<L::RB>(row, c), (const uint8_t*)p.k + off, s >= 0);
      cp_async16(vd + swz<L::RB>(row, c), (const uint8_t*)p.v + off, s >= 0);
    }
    if (E4M3 && lane < KEYS) {
      cp_async4(vd + L::TILE + lane * 4, p.k_scale + max(slot, 0), slot >= 0);
      cp_async4(vd + L::TILE + (KEYS + lane) * 4, p.v_scale + max(slot, 0), slot >= 0);
    }
    const uint32_t there = __ballot_sync(0xffffffffu, slot >= 0);
    if (lane == 0) asm volatile("st.shared.b32 [%0], %1;" ::"r"(kd + L::STAGE - 16), "r"(there) : "memory");
  };

  int page = load_page(0);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    const int next = load_page(i + 1);
    if (i < mine) copy_tile(i, page);
    cp_async_commit();
    page = next;
  }
  for (int i = 0; i < mine; ++i) {
    cp_async_wait<STAGES - 2>();
    __syncwarp();
    const int next = load_page(i + STAGES);
    if (i + STAGES - 1 < mine) copy_tile(i + STAGES - 1, page);   // into the stage that tile i - 1 was read from
    cp_async_commit();
    page = next;
    const uint32_t kd = ring + (i % STAGES) * L::STAGE, vd = kd + L::TILE;
    const int base = k0 + (warp + i * WARPS) * KEYS;
    const int mi = lane >> 3, row = lane & 7;   // ldmatrix: which of the four matrices, which of its rows

    float s[KT][NT][4];   // keys 16 kt + g (0, 1) and + 8 (2, 3), rows 8 n + 2 t and + 1
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[kt][n][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < DH / 16; ++ks)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        uint32_t f[4];
        if (!E4M3) {
          ldsm4(kd + swz<L::RB>(kt * 16 + (mi & 1) * 8 + row, 2 * ks + (mi >> 1)), f);
        } else {
          codes_to_f16(lds32(kd + swz<L::RB>(kt * 16 + g, ks) + 4 * t), f[0], f[2]);
          codes_to_f16(lds32(kd + swz<L::RB>(kt * 16 + 8 + g, ks) + 4 * t), f[1], f[3]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<MATH>(s[kt][n], f, qf[n][ks][0], qf[n][ks][1]);
      }

    const uint32_t there = lds32(kd + L::STAGE - 16);
    float inv_vs[KT][2];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float ks = 1.f, lv = 0.f;
        if (E4M3) {
          const int key = kt * 16 + 8 * h + g;
          ks = __uint_as_float(lds32(vd + L::TILE + key * 4));
          const float vs = positive_scale(__uint_as_float(lds32(vd + L::TILE + (KEYS + key) * 4)));
          lv = lg2(vs);
          inv_vs[kt][h] = rcp(vs) * DOWN;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = s[kt][n][2 * h + e];
            x = E4M3 ? fmaf(x * row_scale[n][e], ks, lv) : x * row_scale[n][e];
          }
      }
    if (__any_sync(0xffffffffu, there != (KEYS == 32 ? 0xffffffffu : (1u << KEYS) - 1u) || base + KEYS - 1 > lowest)) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = kt * 16 + 8 * (e >> 1) + g;
            if (base + key > limit[n][e & 1] || !(there >> key & 1u)) s[kt][n][e] = -INFINITY;
          }
    }
    float keep[NT][2], ref[NT][2];
    bool changed = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) top = fmaxf(top, fmaxf(s[kt][n][e], s[kt][n][2 + e]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        // rounded up: however large the scores, no weight is above 2^UP
        const float mn = fmaxf(m[n][e], UP == 0.f ? top : __fadd_ru(top, -UP));
        ref[n][e] = mn == -INFINITY ? 0.f : mn;      // a row that has seen no key yet
        keep[n][e] = ex2(m[n][e] - ref[n][e]);
        m[n][e] = mn;
        l[n][e] *= keep[n][e];
        changed = changed || keep[n][e] != 1.f;
      }
    uint32_t pf[KT][NT][2];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float w[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            w[e] = ex2(s[kt][n][2 * h + e] - ref[n][e]);
            l[n][e] += E4M3 ? w[e] * inv_vs[kt][h] : w[e];
          }
          pf[kt][n][h] = transpose8x8(pack16<MATH>(w[0], w[1]));
        }
    if (__any_sync(0xffffffffu, changed)) {
#pragma unroll
      for (int d = 0; d < DH / 16; ++d)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][n][e] *= keep[n][e & 1];
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      if (!E4M3) {
#pragma unroll
        for (int d = 0; d < DH / 16; ++d) {
          uint32_t f[4];
          ldsm4_t(vd + swz<L::RB>(kt * 16 + (mi >> 1) * 8 + row, 2 * d + (mi & 1)), f);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<MATH>(o[d][n], f, pf[kt][n][0], pf[kt][n][1]);
        }
      } else {
#pragma unroll
        for (int c = 0; c < DH / 32; ++c) {   // elements 32 c + 4 g .. + 3 of four keys: rows g and g + 8 of two products
          uint32_t w[4], lo[4], hi[4];
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4)
            w[q4] = lds32(vd + swz<L::RB>(kt * 16 + 2 * t + (q4 & 1) + (q4 >> 1) * 8, 2 * c + (g >> 2)) + 4 * (g & 3));
          codes_to_f16(__byte_perm(w[0], w[1], 0x5140), lo[0], lo[1]);
          codes_to_f16(__byte_perm(w[0], w[1], 0x7362), lo[2], lo[3]);
          codes_to_f16(__byte_perm(w[2], w[3], 0x5140), hi[0], hi[1]);
          codes_to_f16(__byte_perm(w[2], w[3], 0x7362), hi[2], hi[3]);
#pragma unroll
          for (int i2 = 0; i2 < 2; ++i2) {
            const uint32_t f[4] = {lo[2 * i2], lo[2 * i2 + 1], hi[2 * i2], hi[2 * i2 + 1]};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816<MATH>(o[2 * c + i2][n], f, pf[kt][n][0], pf[kt][n][1]);
          }
        }
      }
    }
    __syncwarp();   // the stage may be overwritten
  }
  cp_async_wait<0>();
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], x);

  // ------------------------------------------------------------------ join the warps
  __syncthreads();
  float* ml = reinterpret_cast<float*>(smem);                     // [warp][row] maximum, then sum
  float* os = ml + 2 * WARPS * ROWS;                              // [warp][row][DH + 4]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (g == 0) {
        ml[warp * ROWS + 8 * n + 2 * t + e] = m[n][e];
        ml[(WARPS + warp) * ROWS + 8 * n + 2 * t + e] = l[n][e];
      }
      float* to = os + (warp * ROWS + 8 * n + 2 * t + e) * (DH + 4);
#pragma unroll
      for (int d = 0; d < DH / 16; ++d) {
        to[E4M3 ? 32 * (d >> 1) + 4 * g + 2 * (d & 1) : 16 * d + g] = o[d][n][e] * DOWN;
        to[E4M3 ? 32 * (d >> 1) + 4 * g + 2 * (d & 1) + 1 : 16 * d + g + 8] = o[d][n][2 + e] * DOWN;
      }
    }
  __syncthreads();
  join_and_store<T, ROWS>(a, u, ml, DH);
}

// Joins the parts of a context: o = sum_s 2^(lse_s - max) o_s / sum_s 2^(lse_s - max).  A group of LANES threads owns a (token, head),
// four elements each; with SHARE > 1 so many groups share its parts (few rows, many parts), which are then added in their order.
constexpr int COMBINE_THREADS = 128;

template <int TYPE, int LANES, int RUNS, int SHARE>
__global__ void __launch_bounds__(COMBINE_THREADS) combine_kernel(const AttnArgs a) {
  using T = typename Elem<TYPE>::T;
  constexpr int GROUPS = COMBINE_THREADS / LANES, ROWS = GROUPS / SHARE, WIDTH = LANES * 4 * RUNS;
  __shared__ float part[SHARE > 1 ? GROUPS : 1][SHARE > 1 ? WIDTH + 1 : 1];
  const lbi_paged_batch& p = a.b;
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, share = group % SHARE, dim = p.head_dim;
  const int64_t at = (int64_t)blockIdx.x * ROWS + group / SHARE;
  const bool exists = at < (int64_t)p.rows * a.heads;
  const int2 own = owned_rows(p);
  const bool owned = exists && at / a.heads >= own.x && at / a.heads < own.y;
  const float* lse = a.part_lse + at * a.splits;
  float top = -INFINITY;
  if (owned)
    for (int s = lane; s < a.splits; s += LANES) top = fmaxf(top, lse[s]);
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float ref = top == -INFINITY ? 0.f : top;
  float acc[RUNS][4], sum = 0.f;
#pragma unroll
  for (int r = 0; r < RUNS; ++r)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[r][e] = 0.f;
  if (owned) {
#pragma unroll 4
    for (int s = share; s < a.splits; s += SHARE) {
      const float w = ex2(__ldg(lse + s) - ref);
      sum += w;
#pragma unroll
      for (int r = 0; r < RUNS; ++r) {
        const int d = (r * LANES + lane) * 4;
        const float4 x = d < dim ? __ldg(reinterpret_cast<const float4*>(a.part_o + (at * a.splits + s) * dim + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
        acc[r][0] += w * x.x;
        acc[r][1] += w * x.y;
        acc[r][2] += w * x.z;
        acc[r][3] += w * x.w;
      }
    }
  }
  if (SHARE > 1) {
#pragma unroll
    for (int r = 0; r < RUNS; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[group][(r * LANES + lane) * 4 + e] = acc[r][e];
    if (lane == 0) part[group][WIDTH] = sum;
    __syncthreads();
    if (share == 0) {
#pragma unroll
      for (int g = 1; g < SHARE; ++g) {
#pragma unroll
        for (int r = 0; r < RUNS; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[r][e] += part[group + g][(r * LANES + lane) * 4 + e];
        sum += part[group + g][WIDTH];
      }
    }
  }
  if (share != 0 || !exists || (!owned && !a.zero_tail)) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int r = 0; r < RUNS; ++r) {
    const int d = (r * LANES + lane) * 4;
    if (d >= dim) break;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[r][e] *= inv;
    store_f<T, 4>((T*)a.out + at * dim + d, acc[r]);
  }
}

template <int TYPE>
int launch_combine(const AttnArgs& a, int sm_count, cudaStream_t st) {
  // several groups per row where the rows alone give less than two blocks per SM
  const int64_t rows = (int64_t)a.b.rows * a.heads;
  const bool few = rows < 2ll * sm_count * 4 && a.splits >= 8;
  const int dim = a.b.head_dim, lanes = dim <= 32 ? 8 : dim <= 64 ? 16 : 32;
  const int64_t per_block = COMBINE_THREADS / lanes / (few ? 4 : 1), blocks = (rows + per_block - 1) / per_block;
  if (blocks >= (1ll << 31)) return (int)cudaErrorInvalidValue;
#define LBI_COMBINE(L, R)                                                                          \
  do {                                                                                             \
    if (few) combine_kernel<TYPE, L, R, 4><<<(unsigned)blocks, COMBINE_THREADS, 0, st>>>(a);        \
    else combine_kernel<TYPE, L, R, 1><<<(unsigned)blocks, COMBINE_THREADS, 0, st>>>(a);            \
  } while (0)
  if (lanes == 8) LBI_COMBINE(8, 1);
  else if (lanes == 16) LBI_COMBINE(16, 1);
  else if (dim <= 128) LBI_COMBINE(32, 1);
  else LBI_COMBINE(32, 2);
#undef LBI_COMBINE
  return (int)cudaGetLastError();
}

// ------------------------------------------------------------------------------------------------ 16-row tiles, any type and size
// The same division of work (one warp, its own keys) for fp32 queries and head sizes without tiles of their own.  An fp32 value is the
// sum of three bf16 values (24 bits), an fp16 value of two, a bf16 value or a code is one; a product of two such sums is the products
// of their terms down to 2^-16 of the first (six for fp32 against fp32), by mma.sync m16n8k16 with bf16 operands.  (tf32 products
// would take two terms, but m16n8k8 occupies the tensor pipe for 32 cycles here, as long as plain FMAs would take, and m16n8k16 with
// bf16 operands for 9.)  The products of one step of sixteen elements (of one key tile) start from zero and are
// added to the running sums by the FMA units, which round to nearest: the tensor core truncates, and over thousands of keys that is a
// drift (2 to 3 e-6 of the result, against 3.5 e-7).
// Queries lie in shared memory in the order of the fragments; keys and values as they come, their rows padded so that the accesses of a
// fragment fall into different banks.
template <int TYPE>
struct Terms {
  static constexpr int N = TYPE == LBI_F32 ? 3 : TYPE == LBI_F16 ? 2 : 1;
};
template <int TYPE, bool E4M3, int DHP>
struct AnyTile {   // DHP: head_dim rounded up to 64, 128 or 256
  using Q = typename Elem<TYPE>::T;
  using C = typename Elem<E4M3 ? LBI_E4M3 : TYPE>::T;
  static constexpr int KEYS = 16, STAGES = DHP == 256 && sizeof(C) == 4 ? 1 : 2;
  static constexpr int NQ = Terms<TYPE>::N, NC = E4M3 ? 1 : Terms<TYPE>::N, NP = TYPE == LBI_F32 ? 3 : 2;
  static constexpr int LAST = TYPE == LBI_F32 ? 2 : 1;   // terms i and j are multiplied if i + j <= LAST
  static constexpr int Q_BYTES = DHP / 16 * 32 * 16 * NQ;
  __host__ __device__ static int k_pitch(int dim) { return dim * (int)sizeof(C) + (sizeof(C) == 4 ? 32 : 16); }
  __host__ __device__ static int v_pitch(int dim) { return dim * (int)sizeof(C) + 16; }
  __host__ __device__ static int stage(int dim) { return KEYS * (k_pitch(dim) + v_pitch(dim)) + 8 * KEYS + 16; }   // K, V, scales, which keys exist
  __host__ __device__ static int smem(int dim) {
    const int join = WARPS * ROW_TILE * (dim + 4) * 4 + WARPS * ROW_TILE * 8, ring = WARPS * STAGES * stage(dim);
    return Q_BYTES + (join > ring ? join : ring);
  }
};

// The bf16 terms of two values, as words of two.
template <int N>
__device__ __forceinline__ void split_bf16(float x0, float x1, uint32_t* w) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    w[i] = pack16<LBI_BF16>(x0, x1);
    x0 -= __uint_as_float(w[i] << 16);
    x1 -= __uint_as_float(w[i] & 0xffff0000u);
  }
}

template <int TYPE, bool E4M3, int DHP>
__global__ void __launch_bounds__(WARPS * 32) attn_any_kernel(const AttnArgs a) {
  using L = AnyTile<TYPE, E4M3, DHP>;
  using T = typename L::Q;
  using C = typename L::C;
  constexpr int KEYS = L::KEYS, STAGES = L::STAGES;
  extern __shared__ __align__(128) uint8_t smem[];
  const lbi_paged_batch& p = a.b;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, dim = p.head_dim;
  if (a.zero_tail && !a.part_o) zero_rows_of_nobody(p, (T*)a.out, a.heads * dim);
  const RowsUnit u = rows_unit(a, ROW_TILE);
  if (!u.any) return;

  constexpr int NQ = L::NQ, NC = L::NC, NP = L::NP, LAST = L::LAST;
  uint4* qs = reinterpret_cast<uint4*>(smem);   // [16 elements][term][lane]
  int limit[2];
  for (int ks = warp; ks < dim / 16; ks += WARPS) {
    uint32_t w[4][NQ];
#pragma unroll
    for (int e = 0; e < 4; ++e) {   // rows g and g + 8, elements 2 t, + 1 and 2 t + 8, + 9
      const int r = g + 8 * (e & 1), rr = u.local + r;
      const T* src = (const T*)a.q + (int64_t)(u.first_row + rr / a.group) * a.q_stride + (u.kh * a.group + rr % a.group) * dim + ks * 16 + 2 * t + 8 * (e >> 1);
      const bool live = r < u.n_rows;
      split_bf16<NQ>(live ? to_f<T>(src[0]) : 0.f, live ? to_f<T>(src[1]) : 0.f, w[e]);
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) qs[(ks * NQ + i) * 32 + lane] = make_uint4(w[0][i], w[1][i], w[2][i], w[3][i]);
  }
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) limit[hh] = g + 8 * hh < u.n_rows ? u.first_pos + (u.local + g + 8 * hh) / a.group : -1;
  __syncthreads();

  float o[DHP / 8][4];
#pragma unroll
  for (int i = 0; i < DHP / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  const int k_pitch = L::k_pitch(dim), v_pitch = L::v_pitch(dim), stage = L::stage(dim);
  uint8_t* ring = smem + L::Q_BYTES + warp * STAGES * stage;
  const int n_tiles = u.k1 > u.k0 ? (u.k1 - u.k0 + KEYS - 1) / KEYS : 0;
  const int mine = n_tiles > warp ? (n_tiles - warp + WARPS - 1) / WARPS : 0;
  const int* table = p.table + (int64_t)u.b * p.table_stride;
  auto load_page = [&](int i) {
    const int pos = u.k0 + (warp + i * WARPS) * KEYS + lane;
    return i < mine && lane < KEYS && pos < u.k1 ? __ldg(table + (pos >> a.page_shift)) : -1;
  };
  const int row_chunks = dim * (int)sizeof(C) / 16;
  auto copy_tile = [&](int i, int page) {
    const int pos = u.k0 + (warp + i * WARPS) * KEYS + lane;
    const int slot = key_slot(a, u, pos, lane < KEYS && pos < u.k1, page);
    uint8_t* k_dst = ring + (i % STAGES) * stage;
    uint8_t* v_dst = k_dst + KEYS * k_pitch;
    for (int j = 0; j < KEYS * row_chunks; j += 32) {   // KEYS * row_chunks is a multiple of 8, the last round may be partial
      const int row = min((j + lane) / row_chunks, KEYS - 1), c = (j + lane) - row * row_chunks;
      const int s = __shfl_sync(0xffffffffu, slot, row);
      if (c < row_chunks) {
        const int64_t off = (int64_t)max(s, 0) * dim * sizeof(C) + c * 16;
        cp_async16(smem_addr(k_dst + row * k_pitch + c * 16), (const uint8_t*)p.k + off, s >= 0);
        cp_async16(smem_addr(v_dst + row * v_pitch + c * 16), (const uint8_t*)p.v + off, s >= 0);
      }
    }
    uint8_t* extra = v_dst + KEYS * v_pitch;
    if (E4M3 && lane < KEYS) {
      cp_async4(smem_addr(extra + lane * 4), p.k_scale + max(slot, 0), slot >= 0);
      cp_async4(smem_addr(extra + (KEYS + lane) * 4), p.v_scale + max(slot, 0), slot >= 0);
    }
    const uint32_t there = __ballot_sync(0xffffffffu, slot >= 0);
    if (lane == 0) *reinterpret_cast<volatile uint32_t*>(extra + 8 * KEYS) = there;
  };

  int page = load_page(0);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    const int next = load_page(i + 1);
    if (i < mine) copy_tile(i, page);
    cp_async_commit();
    page = next;
  }
  for (int i = 0; i < mine; ++i) {
    if (STAGES > 1) {
      cp_async_wait<STAGES - 2>();
      __syncwarp();
    }
    const int next = load_page(i + STAGES);
    if (i + STAGES - 1 < mine) copy_tile(i + STAGES - 1, page);
    cp_async_commit();
    page = next;
    if (STAGES == 1) {   // no room for a tile ahead
      cp_async_wait<0>();
      __syncwarp();
    }
    const uint8_t* k_src = ring + (i % STAGES) * stage;
    const uint8_t* v_src = k_src + KEYS * k_pitch;
    const uint8_t* extra = v_src + KEYS * v_pitch;
    const int base = u.k0 + (warp + i * WARPS) * KEYS;

    float s[KEYS / 8][4];
#pragma unroll
    for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
    // products of one sum wait for each other, and the compiler keeps them in the order in which they stand here: term by term
    constexpr int KN = KEYS / 8;
#pragma unroll 2
    for (int ks = 0; ks < dim / 16; ++ks) {
      alignas(16) uint32_t q[NQ][4];
      uint32_t k[KN][2][NC];
      float c[KN][2][4];   // the leading products and the others
#pragma unroll
      for (int i = 0; i < NQ; ++i) *reinterpret_cast<uint4*>(q[i]) = qs[(ks * NQ + i) * 32 + lane];
#pragma unroll
      for (int n = 0; n < KN; ++n) {
        const C* row = reinterpret_cast<const C*>(k_src + (n * 8 + g) * k_pitch) + ks * 16 + 2 * t;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x[2];
          load_f<C, 2>(row + 8 * h, x);
          split_bf16<NC>(x[0], x[1], k[n][h]);
#pragma unroll
          for (int e = 0; e < 4; ++e) c[n][h][e] = 0.f;
        }
      }
#pragma unroll
      for (int j = NC - 1; j >= 0; --j)
#pragma unroll
        for (int i = NQ - 1; i >= 0; --i)
#pragma unroll
          for (int n = 0; n < KN; ++n)
            if (i + j <= LAST) mma16816<LBI_BF16>(c[n][i + j == 0 ? 0 : 1], q[i], k[n][0][j], k[n][1][j]);
#pragma unroll
      for (int n = 0; n < KN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] += c[n][0][e] + c[n][1][e];
    }

    const uint32_t there = *reinterpret_cast<const volatile uint32_t*>(extra + 8 * KEYS);
    float vs[KEYS / 8][2], top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < KEYS / 8; ++n) {
      float ks[2] = {a.scale_log2, a.scale_log2};
      if (E4M3) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          ks[e] *= reinterpret_cast<const float*>(extra)[n * 8 + 2 * t + e];
          vs[n][e] = reinterpret_cast<const float*>(extra)[KEYS + n * 8 + 2 * t + e];
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = n * 8 + 2 * t + (e & 1);
        const bool seen = base + key <= limit[e >> 1] && (there >> key & 1u);
        s[n][e] = seen ? s[n][e] * ks[e & 1] : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
      }
    }
    float keep[2], ref[2];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      top[hh] = fmaxf(top[hh], __shfl_xor_sync(0xffffffffu, top[hh], 1));
      top[hh] = fmaxf(top[hh], __shfl_xor_sync(0xffffffffu, top[hh], 2));
      const float mn = fmaxf(m[hh], top[hh]);
      ref[hh] = mn == -INFINITY ? 0.f : mn;
      keep[hh] = ex2(m[hh] - ref[hh]);
      m[hh] = mn;
      l[hh] *= keep[hh];
    }
    uint32_t pf[4][NP];   // rows g and g + 8, keys 2 t, + 1 and 8 + 2 t, + 1
#pragma unroll
    for (int n = 0; n < KN; ++n)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          w[e] = ex2(s[n][2 * hh + e] - ref[hh]);
          l[hh] += w[e];
          if (E4M3) w[e] *= vs[n][e];
        }
        split_bf16<NP>(w[0], w[1], pf[2 * n + hh]);
      }
    alignas(16) uint32_t pa[NP][4];
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) pa[i][e] = pf[e][i];
    constexpr int VN = 4;   // products of eight elements at a time
#pragma unroll
    for (int n0 = 0; n0 < DHP / 8; n0 += VN) {
      if (n0 * 8 >= dim) break;
      uint32_t v[VN][2][NC];
      float c[VN][4];
#pragma unroll
      for (int n = 0; n < VN; ++n) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const C* at = reinterpret_cast<const C*>(v_src + (8 * h + 2 * t) * v_pitch) + (n0 + n) * 8 + g;
          const C* below = reinterpret_cast<const C*>(reinterpret_cast<const uint8_t*>(at) + v_pitch);
          const bool live = (n0 + n) * 8 < dim;
          split_bf16<NC>(live ? to_f<C>(*at) : 0.f, live ? to_f<C>(*below) : 0.f, v[n][h]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) c[n][e] = 0.f;
      }
#pragma unroll
      for (int j = NC - 1; j >= 0; --j)
#pragma unroll
        for (int i = NP - 1; i >= 0; --i)
#pragma unroll
          for (int n = 0; n < VN; ++n)
            if (i + j <= LAST) mma16816<LBI_BF16>(c[n], pa[i], v[n][0][j], v[n][1][j]);
#pragma unroll
      for (int n = 0; n < VN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n0 + n][e] = fmaf(o[n0 + n][e], keep[e >> 1], c[n][e]);
    }
    __syncwarp();
  }
  cp_async_wait<0>();
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 1);
    l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 2);
  }
  __syncthreads();
  float* ml = reinterpret_cast<float*>(smem + L::Q_BYTES);
  float* os = ml + 2 * WARPS * ROW_TILE;
  if (t == 0) {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      ml[warp * ROW_TILE + g + 8 * hh] = m[hh];
      ml[(WARPS + warp) * ROW_TILE + g + 8 * hh] = l[hh];
    }
  }
#pragma unroll
  for (int n = 0; n < DHP / 8; ++n) {
    if (n * 8 >= dim) break;
#pragma unroll
    for (int e = 0; e < 4; ++e) os[(warp * ROW_TILE + g + 8 * (e >> 1)) * (dim + 4) + 8 * n + 2 * t + (e & 1)] = o[n][e];
  }
  __syncthreads();
  join_and_store<T, ROW_TILE>(a, u, ml, dim);
}

// ------------------------------------------------------------------------------------------------ host side
template <int TYPE, bool E4M3, int DH, int KEYS, int STAGES, int BLOCKS, int NT>
int launch_rows(const AttnArgs& a, cudaStream_t st) {
  using L = RowsTile<E4M3, DH, KEYS, STAGES, NT>;
  auto kernel = attn_rows_kernel<TYPE, E4M3, DH, KEYS, STAGES, BLOCKS, NT>;
  static lbi::PerDeviceOnce once;
  cudaError_t e = once.max_dynamic_smem(kernel, L::SMEM);
  if (e != cudaSuccess) return (int)e;
  const int64_t blocks = tile_bound(a.b, a.group, L::ROWS) * a.b.kv_heads * a.splits;
  if (blocks >= (1ll << 31)) return (int)cudaErrorInvalidValue;
  kernel<<<(unsigned)blocks, WARPS * 32, L::SMEM, st>>>(a);
  return (int)cudaGetLastError();
}

template <int TYPE, int NT>
int launch_rows(const AttnArgs& a, cudaStream_t st) {   // keys per tile, tiles in flight per warp, blocks per SM
  // Measured, 64 sequences of 8192 tokens: e4m3 head_dim 128 134 us (32, 3, 2: 138), head_dim 64 218 us (16, 4, 4: 256).
  if (a.b.cache_type == LBI_E4M3)
    return a.b.head_dim == 128 ? launch_rows<TYPE, true, 128, 16, 3, NT == 1 ? 4 : 3, NT>(a, st)
         : a.b.head_dim == 64  ? launch_rows<TYPE, true, 64, 32, 3, 4, NT>(a, st) : launch_rows<TYPE, true, 32, 32, 6, 3, NT>(a, st);
  return a.b.head_dim == 128 ? launch_rows<TYPE, false, 128, 16, 3, 2, NT>(a, st)
       : a.b.head_dim == 64  ? launch_rows<TYPE, false, 64, 16, 4, 3, NT>(a, st) : launch_rows<TYPE, false, 32, 32, 4, 3, NT>(a, st);
}

template <int TYPE, bool E4M3, int DHP>
int launch_any(const AttnArgs& a, cudaStream_t st) {
  using L = AnyTile<TYPE, E4M3, DHP>;
  auto kernel = attn_any_kernel<TYPE, E4M3, DHP>;
  static lbi::PerDeviceOnce once;
  cudaError_t e = once.max_dynamic_smem(kernel, L::smem(DHP));
  if (e != cudaSuccess) return (int)e;
  const int64_t blocks = tile_bound(a.b, a.group, ROW_TILE) * a.b.kv_heads * a.splits;
  if (blocks >= (1ll << 31)) return (int)cudaErrorInvalidValue;
  kernel<<<(unsigned)blocks, WARPS * 32, L::smem(a.b.head_dim), st>>>(a);
  return (int)cudaGetLastError();
}
template <int TYPE>
int launch_any(const AttnArgs& a, cudaStream_t st) {
  const int dim = a.b.head_dim;
  if (a.b.cache_type == LBI_E4M3)
    return dim <= 64 ? launch_any<TYPE, true, 64>(a, st) : dim <= 128 ? launch_any<TYPE, true, 128>(a, st) : launch_any<TYPE, true, 256>(a, st);
  return dim <= 64 ? launch_any<TYPE, false, 64>(a, st) : dim <= 128 ? launch_any<TYPE, false, 128>(a, st) : launch_any<TYPE, false, 256>(a, st);
}

}  // namespace paged
}  // namespace lbi

extern "C" lbi_attention_plan lbi_paged_attention_plan(const lbi_paged_batch* p, int type, int heads, float scale, int64_t max_context, int sm_count) {
  using namespace lbi::paged;
  lbi_attention_plan plan{0, ROW_TILE, 1, 1 << 30};
  if (p->rows == 0 || p->batch == 0) return plan;
  const int group = heads / p->kv_heads;
  const int64_t capacity = (int64_t)p->table_width * p->page_size;
  const int64_t longest = max_context > 0 ? std::min(max_context, capacity) : capacity;
  // Which tiles: by the rows (tokens x heads of a group) of an average sequence.  The 16-row tiles read the cache once per 16 rows, the
  // 256-row tiles cost the same up to 256.  Measured with 32 / 8 heads of 128, 8 sequences over 4000 keys (16 over 8000), 16-row / 256-row:
  // 16-bit pages 73 / 62 us (175 / 171) at 28 and 32 rows; e4m3 64 / 83 us (206 / 249) at 48 rows, 93 / 83 (259 / 249) at 64, 114 / 83
  // (363 / 249) at 92; e4m3 at head_dim 64 46 / 64 us (132 / 198) at 60 and 64, equal at 96.  The tcgen05 kernel takes its row maximum
  // before the scale, so it needs a positive one.
  const bool tiled = type != LBI_F32 && (p->head_dim == 32 || p->head_dim == 64 || p->head_dim == 128);
  const int64_t enough = p->cache_type != LBI_E4M3 ? 32 : p->head_dim == 128 ? 64 : 96;
  plan.kernel = !tiled ? 0 : p->head_dim >= 64 && (int64_t)p->rows * group >= enough * p->batch && scale > 0.f ? 2 : 1;
  if (plan.kernel == 2) {
    // Parts of a context pay where there are too few units (256 rows x key head) for the slots: one block per SM, or two (head_dim 64,
    // 16-bit pages), of which the second adds less than the first.  Units of more than one round are left whole: those of a causal or a
    // ragged batch are uneven, the longest start first, and the others fill in behind them.  A part costs as much as 600 keys (its start,
    // its partial result, the joining).  Over 174 batches of 1 to 32 sequences, 4 to 4096 new tokens behind 0 to 32000, 1 to 64 heads of 64
    // or 128, this choice takes 1.03 times the best number of parts (geometric mean; 1.53 at worst); filling whole rounds of equal
    // units took 1.085 (1.96) on half of them, e.g. 130 us in two parts against 66 us whole for 16 prompts of 1024 tokens, 4 heads of 128.
    // Tiles, where the row offsets are on the device: half a tile's room per sequence, and a tile for each
    const double mean_tiles = p->cu ? std::max((double)p->rows * group / 256 + 0.5 * p->batch, (double)std::min(p->batch, p->rows))
                                    : (double)p->batch * ((p->rows / p->batch * group + 255) / 256);
    const double units = mean_tiles * p->kv_heads;
    const bool two = p->head_dim == 64 && p->cache_type != LBI_E4M3;
    const double slots = sm_count * (two ? 2 : 1);
    double best = 0;
    for (int splits = 1; splits <= 16 && (splits == 1 || longest / splits >= 256); ++splits) {
      const double rounds = units * splits / slots;
      const double cost = (rounds >= 1 ? rounds : two ? 1 - std::min(0.3, 0.6 * (1 - rounds)) : 1) * ((double)longest / splits + 600);
      if (splits == 1 || cost < 0.95 * best) {
        best = cost;
        plan.splits = splits;
      }
    }
    plan.split_keys = (int)std::max<int64_t>(128, ((longest + plan.splits - 1) / plan.splits + 127) / 128 * 128);
  } else {
    // Parts of equal length, so that a batch of uneven contexts is balanced by the order in which blocks finish: of about 2048 keys
    // (the partial results are under 2 % of the bytes read), so many that the blocks fill whole rounds of two per SM.  Not below 256
    // keys, and 64, a tile per warp, for the kernel that splits its operands (2.6 us per tile; 7 sequences of up to 782 keys took 19.5 us
    // in parts of 256).  Not more parts than 64 MB hold the results of: with so many rows those are seven rounds of blocks and more.
    // Measured with and without this bound: 1024 new tokens, 16 heads of 256, over 16384 keys 7919 (3 parts) / 8118 us (8); 256 single
    // tokens of 32 heads on 8 of 128 over 32768 keys, e4m3, 2749 (15) / 2770 us (16).
    const int64_t least = plan.kernel == 0 ? 64 : 256;
    if (plan.kernel == 1 && (int64_t)p->rows * group <= 8ll * p->batch) plan.rows = 8;
    const int64_t units = tile_bound(*p, group, plan.rows) * p->kv_heads, slots = 2 * sm_count;
    const int64_t rounds = std::max<int64_t>(1, (longest * units + slots * 2048 - 1) / (slots * 2048));
    const int64_t room = (64ll << 20) / ((int64_t)p->rows * heads * (p->head_dim + 1) * 4);
    const int64_t parts = std::max<int64_t>(1, std::min(room, rounds * slots / units));
    const int64_t keys = std::max<int64_t>(least, ((longest + parts - 1) / parts + 63) / 64 * 64);
    plan.splits = (int)std::max<int64_t>(1, (longest + keys - 1) / keys);
    plan.split_keys = (int)keys;
  }
  return plan;
}

extern "C" int lbi_paged_attention(const lbi_paged_batch* p, const void* q, int64_t q_stride, void* out, float* part_o, float* part_lse,
                                   lbi_attention_plan plan, int type, int heads, float scale, int zero_tail, int sm_count, cudaStream_t st) {
  using namespace lbi::paged;
  if (p->head_dim % 16 != 0 || p->head_dim > 256 || type < 0 || type > LBI_F16 || heads % p->kv_heads != 0) return (int)cudaErrorInvalidValue;
  if (p->rows == 0 || p->batch == 0) return 0;
  if ((plan.splits > 1) != (part_o != nullptr)) return (int)cudaErrorInvalidValue;
  AttnArgs a{*p, q, q_stride, out, part_o, part_lse, heads, heads / p->kv_heads, zero_tail, shift_of(p->page_size), plan.splits, plan.split_keys,
             scale * 1.4426950408889634f};
  int rc;
  if (plan.kernel == 0) rc = type == LBI_F32 ? launch_any<LBI_F32>(a, st) : type == LBI_BF16 ? launch_any<LBI_BF16>(a, st) : launch_any<LBI_F16>(a, st);
  else if (plan.kernel == 1 && plan.rows == 8) rc = type == LBI_BF16 ? launch_rows<LBI_BF16, 1>(a, st) : launch_rows<LBI_F16, 1>(a, st);
  else if (plan.kernel == 1) rc = type == LBI_BF16 ? launch_rows<LBI_BF16, 2>(a, st) : launch_rows<LBI_F16, 2>(a, st);
  else rc = launch_attn_tiles(a, type, st);
  if (rc != 0 || plan.splits == 1) return rc;
  return type == LBI_F32 ? launch_combine<LBI_F32>(a, sm_count, st) : type == LBI_BF16 ? launch_combine<LBI_BF16>(a, sm_count, st) : launch_combine<LBI_F16>(a, sm_count, st);
}
