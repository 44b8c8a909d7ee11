// Causal attention of new tokens over a paged key / value cache.
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j   over the positions j <= context - new + i of the sequence; no position: o_i = 0.
//
// Three kernels:
//   attn_rows_kernel   16 query rows at a time (tokens x heads of a group) for 16-bit queries: decoding, a few new tokens.
//   attn_tiles_kernel  256 rows at a time on tcgen05 (paged_attn_tc.cu): chunks of a prompt.
//   attn_row_kernel    one warp per (token, head): fp32 queries and head sizes that the tiles do not cover.
//   combine_kernel     joins the parts of a long context.
#include <algorithm>

#include "paged.cuh"

namespace lbi {
namespace paged {

// ------------------------------------------------------------------------------------------------ 16-row tiles
// Bound by reading the cache once: 2 head_dim sizeof(code) bytes per key and kv head.  All query heads of a group (and several new
// tokens, if there are) share a tile of 16 rows, so that one read of a key serves them all, and mma.sync m16n8k16 does the products:
// with at most 16 rows the tensor work is a few per cent of the time, and the operands come straight from the copies below, which
// tcgen05 (128 rows, operands through descriptors) would only add steps to.  Every warp works alone on its own keys: a ring of
// cp.async tiles in shared memory (no block barrier in the loop), S = Q K^T, running maximum and sum, O += P V in registers; the
// four warps of a block are joined through shared memory at the end.  The page ids of a tile are loaded one tile ahead of its copies.
//
// e4m3 pages: codes become 16-bit values exactly.  With u_j = scale s_j k_scale_j + log2 v_scale_j the weights 2^(u_j - max u) carry
// the value's scale and stay in (0, 1] (fp16 has no range for p * v_scale); the sum of exponentials takes 2^(u_j - max u) / v_scale_j.
// P is rounded to the queries' 16-bit type before the second product (half a step of the result's type, as the result itself);
// maximum, sum and output stay in fp32.

constexpr int ROW_TILE = 16;
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

template <int TYPE, bool E4M3, int DH, int KEYS, int STAGES>
struct RowsTile {
  static constexpr int RB = DH * (E4M3 ? 1 : 2);
  static constexpr int TILE = KEYS * RB;
  static constexpr int STAGE = 2 * TILE + (E4M3 ? 8 * KEYS : 0) + 16;   // K, V, scales, which keys exist
  static constexpr int RING = STAGES * STAGE;
  static constexpr int JOIN = WARPS * ROW_TILE * (DH + 4) * 4 + WARPS * ROW_TILE * 8;
  static constexpr int SMEM = WARPS * RING > JOIN ? WARPS * RING : JOIN;
};

template <int TYPE, bool E4M3, int DH, int KEYS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32, 2) attn_rows_kernel(const AttnArgs a) {
  using T = typename Elem<TYPE>::T;
  using L = RowsTile<TYPE, E4M3, DH, KEYS, STAGES>;
  extern __shared__ __align__(128) uint8_t smem[];
  const lbi_paged_batch& p = a.b;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % a.splits;
  const int64_t unit = blockIdx.x / a.splits;
  const int kh = (int)(unit % p.kv_heads);
  const int64_t tile = unit / p.kv_heads;

  if (a.zero_tail && !a.part_o)
    for (int64_t row = (int64_t)last_row(p) + blockIdx.x; row < p.rows; row += gridDim.x)
      for (int i = threadIdx.x; i < a.heads * DH; i += WARPS * 32) ((T*)a.out)[row * a.heads * DH + i] = from_f<T>(0.f);

  const int b = seq_of_tile(p, tile, a.group, ROW_TILE);
  const int2 r = seq_rows(p, b);
  const int local = (int)(tile - first_tile(p, b, a.group, ROW_TILE)) * ROW_TILE;   // first row of the tile in the sequence's tile space
  const int rows_b = (r.y - r.x) * a.group;
  if (local < 0 || local >= rows_b) return;
  const int n_rows = min(ROW_TILE, rows_b - local);
  const int ctx = __ldg(p.context + b);
  const int first_pos = ctx - (r.y - r.x);                                          // position of the sequence's first new token
  const int64_t capacity = (int64_t)p.table_width << a.page_shift;
  const int keys = (int)min((int64_t)first_pos + (local + n_rows - 1) / a.group + 1, capacity);
  const int k0 = split * a.split_keys;
  const int k1 = split == a.splits - 1 ? keys : min(keys, k0 + a.split_keys);

  // query fragments: row g (and g + 8) of the tile; the order of the head's elements within a product of 16 is free as long as Q and
  // K agree: natural for 16-bit pages (ldmatrix), 4 neighbours per thread for codes (one 32-bit load)
  uint32_t qf[DH / 16][4];
  int limit[2];
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    const int rr = local + g + 8 * hh;
    const bool live = g + 8 * hh < n_rows;
    const int token = live ? rr / a.group : 0, head = kh * a.group + (live ? rr % a.group : 0);
    limit[hh] = live ? first_pos + token : -1;
    const uint32_t* src = reinterpret_cast<const uint32_t*>((const T*)a.q + (int64_t)(r.x + token) * a.q_stride + head * DH);
#pragma unroll
    for (int ks = 0; ks < DH / 16; ++ks) {
      qf[ks][hh] = live ? src[ks * 8 + (E4M3 ? 2 * t : t)] : 0u;
      qf[ks][2 + hh] = live ? src[ks * 8 + (E4M3 ? 2 * t + 1 : t + 4)] : 0u;
    }
  }
  float o[DH / 8][4];
#pragma unroll
  for (int i = 0; i < DH / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  const uint32_t ring = smem_addr(smem) + warp * L::RING;
  const int n_tiles = k1 > k0 ? (k1 - k0 + KEYS - 1) / KEYS : 0;
  const int mine = n_tiles > warp ? (n_tiles - warp + WARPS - 1) / WARPS : 0;      // tiles warp, warp + 4, ...
  const int* table = p.table + (int64_t)b * p.table_stride;
  auto load_page = [&](int i) {   // page id of key `lane` of this warp's i-th tile; -1: not there
    const int pos = k0 + (warp + i * WARPS) * KEYS + lane;
    return i < mine && lane < KEYS && pos < k1 ? __ldg(table + (pos >> a.page_shift)) : -1;
  };
  auto copy_tile = [&](int i, int page) {
    const int st = i % STAGES;
    const int pos = k0 + (warp + i * WARPS) * KEYS + lane;
    const bool wanted = lane < KEYS && pos < k1;
    int slot = -1;
    if (wanted) {
      if (page >= 0 && page < p.num_pages) slot = (page * p.kv_heads + kh) * p.page_size + (pos & (p.page_size - 1));
      else if (p.status) atomicCAS(p.status, 0, 84);
    }
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

    float s[KEYS / 8][4];
#pragma unroll
    for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
    if (!E4M3) {
      const int mi = lane >> 3, row = lane & 7;
#pragma unroll
      for (int ks = 0; ks < DH / 16; ++ks)
#pragma unroll
        for (int np = 0; np < KEYS / 16; ++np) {
          uint32_t f[4];
          ldsm4(kd + swz<L::RB>(np * 16 + (mi >> 1) * 8 + row, 2 * ks + (mi & 1)), f);
          mma16816<TYPE>(s[2 * np], qf[ks], f[0], f[1]);
          mma16816<TYPE>(s[2 * np + 1], qf[ks], f[2], f[3]);
        }
    } else {
#pragma unroll
      for (int ks = 0; ks < DH / 16; ++ks)
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n) {
          const uint32_t w = lds32(kd + swz<L::RB>(n * 8 + g, ks) + 4 * t);
          uint32_t f0, f1;
          codes_to_16<TYPE>(w, f0, f1);
          mma16816<TYPE>(s[n], qf[ks], f0, f1);
        }
    }

    const uint32_t there = lds32(kd + L::STAGE - 16);
    float inv_vs[KEYS / 8][2];
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < KEYS / 8; ++n) {
      float ks[2] = {a.scale_log2, a.scale_log2}, lv[2] = {0.f, 0.f};
      if (E4M3) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          ks[e] *= __uint_as_float(lds32(vd + L::TILE + (n * 8 + 2 * t + e) * 4));
          const float vs = positive_scale(__uint_as_float(lds32(vd + L::TILE + (KEYS + n * 8 + 2 * t + e) * 4)));
          lv[e] = lg2(vs);
          inv_vs[n][e] = __frcp_rn(vs);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = n * 8 + 2 * t + (e & 1);
        const bool seen = base + key <= limit[e >> 1] && (there >> key & 1u);
        s[n][e] = seen ? fmaf(s[n][e], ks[e & 1], lv[e & 1]) : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
      }
    }
    float keep[2], ref[2];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      top[hh] = fmaxf(top[hh], __shfl_xor_sync(0xffffffffu, top[hh], 1));
      top[hh] = fmaxf(top[hh], __shfl_xor_sync(0xffffffffu, top[hh], 2));
      const float mn = fmaxf(m[hh], top[hh]);
      ref[hh] = mn == -INFINITY ? 0.f : mn;      // a row that has seen no key yet
      keep[hh] = ex2(m[hh] - ref[hh]);
      m[hh] = mn;
      l[hh] *= keep[hh];
    }
    uint32_t pf[KEYS / 16][4];
#pragma unroll
    for (int n = 0; n < KEYS / 8; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = ex2(s[n][e] - ref[e >> 1]);
        l[e >> 1] += E4M3 ? s[n][e] * inv_vs[n][e & 1] : s[n][e];
      }
      pf[n >> 1][(n & 1) * 2] = pack16<TYPE>(s[n][0], s[n][1]);
      pf[n >> 1][(n & 1) * 2 + 1] = pack16<TYPE>(s[n][2], s[n][3]);
    }
#pragma unroll
    for (int n = 0; n < DH / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] *= keep[e >> 1];
    if (!E4M3) {
      const int mi = lane >> 3, row = lane & 7;
#pragma unroll
      for (int kk = 0; kk < KEYS / 16; ++kk)
#pragma unroll
        for (int n = 0; n < DH / 16; ++n) {
          uint32_t f[4];
          ldsm4_t(vd + swz<L::RB>(kk * 16 + (mi & 1) * 8 + row, 2 * n + (mi >> 1)), f);
          mma16816<TYPE>(o[2 * n], pf[kk], f[0], f[1]);
          mma16816<TYPE>(o[2 * n + 1], pf[kk], f[2], f[3]);
        }
    } else {
#pragma unroll
      for (int kk = 0; kk < KEYS / 16; ++kk)
#pragma unroll
        for (int c = 0; c < DH / 32; ++c) {   // elements 32 c + 4 g .. + 3 of four keys: column g of four products
          uint32_t w[4];
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4)
            w[q4] = lds32(vd + swz<L::RB>(kk * 16 + 2 * t + (q4 & 1) + (q4 >> 1) * 8, 2 * c + (g >> 2)) + 4 * (g & 3));
          uint32_t lo[4], hi[4];
          codes_to_16<TYPE>(__byte_perm(w[0], w[1], 0x5140), lo[0], lo[1]);
          codes_to_16<TYPE>(__byte_perm(w[0], w[1], 0x7362), lo[2], lo[3]);
          codes_to_16<TYPE>(__byte_perm(w[2], w[3], 0x5140), hi[0], hi[1]);
          codes_to_16<TYPE>(__byte_perm(w[2], w[3], 0x7362), hi[2], hi[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) mma16816<TYPE>(o[4 * c + e], pf[kk], lo[e], hi[e]);
        }
    }
    __syncwarp();   // the stage may be overwritten
  }
  cp_async_wait<0>();
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 1);
    l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 2);
  }

  // ------------------------------------------------------------------ join the warps
  __syncthreads();
  float* ml = reinterpret_cast<float*>(smem);                     // [warp][row] maximum, then sum
  float* os = ml + 2 * WARPS * ROW_TILE;                          // [warp][row][DH + 4]
  if (t == 0) {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      ml[warp * ROW_TILE + g + 8 * hh] = m[hh];
      ml[(WARPS + warp) * ROW_TILE + g + 8 * hh] = l[hh];
    }
  }
#pragma unroll
  for (int n = 0; n < DH / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int col = 2 * t + (e & 1);
      const int d = E4M3 ? 32 * (n >> 2) + 4 * col + (n & 3) : 8 * n + col;
      os[(warp * ROW_TILE + g + 8 * (e >> 1)) * (DH + 4) + d] = o[n][e];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < n_rows * (DH / 8); i += WARPS * 32) {
    const int rr = i / (DH / 8), d = i % (DH / 8) * 8;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, ml[w * ROW_TILE + rr]);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f, acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = ex2(ml[w * ROW_TILE + rr] - ref);
      sum += f * ml[(WARPS + w) * ROW_TILE + rr];
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += f * os[(w * ROW_TILE + rr) * (DH + 4) + d + e];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= inv;
    const int64_t at = (int64_t)(r.x + (local + rr) / a.group) * a.heads + kh * a.group + (local + rr) % a.group;
    if (a.part_o) {
      store_f<float, 8>(a.part_o + (at * a.splits + split) * DH + d, acc);
      if (d == 0) a.part_lse[at * a.splits + split] = sum == 0.f ? -INFINITY : top + log2f(sum);
    } else {
      store_f<T, 8>((T*)a.out + at * DH + d, acc);
    }
  }
}

// Joins the parts of a context: o = sum_s 2^(lse_s - max) o_s / sum_s 2^(lse_s - max).  A group of LANES threads owns a (token, head),
// four elements each; with SHARE > 1 so many groups share its parts (few rows, many parts), which are then added in their order.
constexpr int COMBINE_THREADS = 128;

template <int TYPE, int LANES, int SHARE>
__global__ void __launch_bounds__(COMBINE_THREADS) combine_kernel(const AttnArgs a) {
  using T = typename Elem<TYPE>::T;
  constexpr int GROUPS = COMBINE_THREADS / LANES, ROWS = GROUPS / SHARE;
  __shared__ float part[SHARE > 1 ? GROUPS : 1][LANES * 4 + 1];
  const lbi_paged_batch& p = a.b;
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, share = group % SHARE, dim = p.head_dim, d = lane * 4;
  const int64_t at = (int64_t)blockIdx.x * ROWS + group / SHARE;
  const bool exists = at < (int64_t)p.rows * a.heads;
  const bool owned = exists && at / a.heads < last_row(p);
  const float* lse = a.part_lse + at * a.splits;
  float top = -INFINITY;
  if (owned)
    for (int s = lane; s < a.splits; s += LANES) top = fmaxf(top, lse[s]);
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float ref = top == -INFINITY ? 0.f : top;
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
  if (owned) {
#pragma unroll 4
    for (int s = share; s < a.splits; s += SHARE) {
      const float w = ex2(__ldg(lse + s) - ref);
      const float4 x = d < dim ? __ldg(reinterpret_cast<const float4*>(a.part_o + (at * a.splits + s) * dim + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
      sum += w;
      acc[0] += w * x.x;
      acc[1] += w * x.y;
      acc[2] += w * x.z;
      acc[3] += w * x.w;
    }
  }
  if (SHARE > 1) {
#pragma unroll
    for (int e = 0; e < 4; ++e) part[group][d + e] = acc[e];
    if (lane == 0) part[group][LANES * 4] = sum;
    __syncthreads();
    if (share == 0) {
#pragma unroll
      for (int g = 1; g < SHARE; ++g) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += part[group + g][d + e];
        sum += part[group + g][LANES * 4];
      }
    }
  }
  if (share != 0 || !exists || d >= dim || (!owned && !a.zero_tail)) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] *= inv;
  store_f<T, 4>((T*)a.out + at * dim + d, acc);
}

template <int TYPE>
int launch_combine(const AttnArgs& a, int sm_count, cudaStream_t st) {
  // several groups per row where the rows alone give less than two blocks per SM
  const int64_t rows = (int64_t)a.b.rows * a.heads;
  const bool few = rows < 2ll * sm_count * 4 && a.splits >= 8;
  const int lanes = a.b.head_dim <= 32 ? 8 : a.b.head_dim <= 64 ? 16 : a.b.head_dim <= 128 ? 32 : 64;
  const int64_t per_block = COMBINE_THREADS / lanes / (few ? (lanes == 64 ? 2 : 4) : 1), blocks = (rows + per_block - 1) / per_block;
  if (blocks >= (1ll << 31)) return (int)cudaErrorInvalidValue;
#define LBI_COMBINE(L, S) combine_kernel<TYPE, L, S><<<(unsigned)blocks, COMBINE_THREADS, 0, st>>>(a)
  if (lanes == 8) { if (few) LBI_COMBINE(8, 4); else LBI_COMBINE(8, 1); }
  else if (lanes == 16) { if (few) LBI_COMBINE(16, 4); else LBI_COMBINE(16, 1); }
  else { if (few) LBI_COMBINE(32, 4); else LBI_COMBINE(32, 1); }
#undef LBI_COMBINE
  return (int)cudaGetLastError();
}

// ------------------------------------------------------------------------------------------------ one warp per row
// fp32 queries and head sizes without a tile: the lanes share the head's elements, the running maximum, sum and output stay in
// registers in fp32 and every key is read once.  e4m3 pages: the key's scale multiplies its score, the value's its probability.

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

// ------------------------------------------------------------------------------------------------ host side
template <int TYPE, bool E4M3, int DH, int KEYS, int STAGES>
int launch_rows(const AttnArgs& a, cudaStream_t st) {
  using L = RowsTile<TYPE, E4M3, DH, KEYS, STAGES>;
  auto kernel = attn_rows_kernel<TYPE, E4M3, DH, KEYS, STAGES>;
  static lbi::PerDeviceOnce once;
  cudaError_t e = once.max_dynamic_smem(kernel, L::SMEM);
  if (e != cudaSuccess) return (int)e;
  const int64_t blocks = tile_bound(a.b, a.group, ROW_TILE) * a.b.kv_heads * a.splits;
  if (blocks >= (1ll << 31)) return (int)cudaErrorInvalidValue;
  kernel<<<(unsigned)blocks, WARPS * 32, L::SMEM, st>>>(a);
  return (int)cudaGetLastError();
}

template <int TYPE>
int launch_rows(const AttnArgs& a, cudaStream_t st) {   // about 8 KB of keys and values per stage
  if (a.b.cache_type == LBI_E4M3)
    return a.b.head_dim == 128 ? launch_rows<TYPE, true, 128, 32, 3>(a, st)
         : a.b.head_dim == 64  ? launch_rows<TYPE, true, 64, 32, 5>(a, st) : launch_rows<TYPE, true, 32, 32, 6>(a, st);
  return a.b.head_dim == 128 ? launch_rows<TYPE, false, 128, 16, 3>(a, st)
       : a.b.head_dim == 64  ? launch_rows<TYPE, false, 64, 32, 3>(a, st) : launch_rows<TYPE, false, 32, 32, 5>(a, st);
}

template <int TYPE>
int launch_row(const AttnArgs& a, cudaStream_t st) {
  const int64_t blocks = ((int64_t)a.b.rows * a.heads + 3) / 4;
  if (blocks >= (1ll << 31)) return (int)cudaErrorInvalidValue;
  if (a.b.cache_type == LBI_E4M3) attn_row_kernel<TYPE, true><<<(unsigned)blocks, 128, 0, st>>>(a);
  else attn_row_kernel<TYPE, false><<<(unsigned)blocks, 128, 0, st>>>(a);
  return (int)cudaGetLastError();
}

}  // namespace paged
}  // namespace lbi

extern "C" lbi_attention_plan lbi_paged_attention_plan(const lbi_paged_batch* p, int type, int heads, float scale, int64_t max_context, int sm_count) {
  using namespace lbi::paged;
  lbi_attention_plan plan{0, 1, 1 << 30};
  if (type == LBI_F32 || p->rows == 0 || p->batch == 0 || !(p->head_dim == 32 || p->head_dim == 64 || p->head_dim == 128)) return plan;
  const int group = heads / p->kv_heads;
  const int64_t capacity = (int64_t)p->table_width * p->page_size;
  const int64_t longest = max_context > 0 ? std::min(max_context, capacity) : capacity;
  // the tcgen05 kernel takes its row maximum before the scale, so it needs a positive one
  plan.kernel = p->head_dim >= 64 && (int64_t)p->rows * group >= 64ll * p->batch && scale > 0.f ? 2 : 1;
  if (plan.kernel == 2) {
    // One block per SM, or two (head_dim 64, 16-bit pages).  Parts of a context pay where whole units leave the last round of blocks half empty: the
    // number of parts (of 512 keys at least) with the fewest key tiles per SM, 4 % added per part for the partial results and the
    // block's own start.
    const int64_t units = tile_bound(*p, group, 256) * p->kv_heads;
    sm_count *= p->head_dim == 64 && p->cache_type != LBI_E4M3 ? 2 : 1;
    double best = 0;
    for (int splits = 1; splits <= 16 && (splits == 1 || longest / splits >= 512); ++splits) {
      const double cost = (double)((units * splits + sm_count - 1) / sm_count) / splits * (1 + 0.04 * (splits - 1));
      if (splits == 1 || cost < 0.95 * best) {
        best = cost;
        plan.splits = splits;
      }
    }
    plan.split_keys = (int)std::max<int64_t>(128, ((longest + plan.splits - 1) / plan.splits + 127) / 128 * 128);
  } else {
    // Parts of equal length, so that a batch of uneven contexts is balanced by the order in which blocks finish: of about 2048 keys
    // (the partial results are under 2 % of the bytes read), so many that the blocks fill whole rounds of two per SM, and not below
    // 256 keys.
    const int64_t units = tile_bound(*p, group, ROW_TILE) * p->kv_heads, slots = 2 * sm_count;
    const int64_t rounds = std::max<int64_t>(1, (longest * units + slots * 2048 - 1) / (slots * 2048));
    const int64_t parts = std::max<int64_t>(1, rounds * slots / units);
    const int64_t keys = std::max<int64_t>(256, ((longest + parts - 1) / parts + 63) / 64 * 64);
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
  if (plan.kernel == 0)
    return type == LBI_F32 ? launch_row<LBI_F32>(a, st) : type == LBI_BF16 ? launch_row<LBI_BF16>(a, st) : launch_row<LBI_F16>(a, st);
  const int rc = plan.kernel == 2 ? launch_attn_tiles(a, type, st) : type == LBI_BF16 ? launch_rows<LBI_BF16>(a, st) : launch_rows<LBI_F16>(a, st);
  if (rc != 0 || plan.splits == 1) return rc;
  return type == LBI_BF16 ? launch_combine<LBI_BF16>(a, sm_count, st) : launch_combine<LBI_F16>(a, sm_count, st);
}
