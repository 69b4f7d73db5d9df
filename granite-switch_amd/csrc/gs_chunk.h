// What the chunk forms of attention over a paged cache share: the order of their parts, a
// part's query rows, the softmax of a tile of 64 keys with the product of its values, the
// results, and the launch (gs_chunk.hip: a bf16 cache, gs_chunk_e4m3.hip: a quantised one).
#pragma once

#include "gs_paged_rows.h"

namespace gs {
namespace {

constexpr int kCWaves = 4;
constexpr int kCKeys = 64;
constexpr int kCStages = 2;

// V rows that no query of a tile sees are zero in LDS: the cache may hold
// anything there, and 0 * NaN is not 0.
__device__ const u32x4 g_zero16 = {0, 0, 0, 0};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// 4 x 16 elements, transposed: lane i of 16 gives the address of 4 elements of
// row i / 4 and gets column i of the 4 rows.
__device__ __forceinline__ uint64_t read_tr(const char* p) {
  return __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p)));
}

// As dma16, with the wait state that M0 needs.
__device__ __forceinline__ void dma16_row(const char* src, uint32_t lds_dst) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds_dst) : "memory", "m0");
}
// As above from a uniform base and the lane's byte offset.
__device__ __forceinline__ void dma16_off(const char* base, uint32_t off, uint32_t lds_dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds_dst) : "memory", "m0");
}
constexpr int wait_vm_lds0(int n) { return (n & 15) | (7 << 4) | ((n >> 4) << 14); }

struct ChunkItem {
  int s, j, part, nparts, slot;      // slot: of the tile's first partial result, or -1
  int order;                         // of the tile among the split ones
  addr::PagedSeq sq;
};
// The chunk form's parts (a tile of a sequence, or one of those it is split into) for
// one head: the sequences with the longest parts first, in eight classes, a
// sequence's tiles and parts from the last.
struct ChunkOrder {
  Batch4 q;
  int tiles;                         // key tiles that a part of a split tile has
  uint32_t magic;
  int longest;                       // key tiles of the longest part
  ClassOrder order;
  uint64_t split;                    // before the lane's: partial results, split tiles << 32
  int total;

  struct Count {
    int nt, np, longest;             // tiles, parts of each, key tiles of the longest part
  };
  __device__ __forceinline__ Count count(const PagedArgs& a, const addr::PagedSeq& sq) const {
    Count c;
    c.nt = addr::chunk_tiles(sq, a.tq);
    c.longest = addr::chunk_key_tiles(addr::chunk_tile(sq, a.tq.tq, a.window, c.nt - 1));
    c.np = addr::chunk_parts(sq, a.tq, a.window, tiles, magic);
    if (c.np > 1) c.longest = min(c.longest, 2 * tiles);
    return c;
  }
  __device__ __forceinline__ int class_of(int x) const {   // x <= longest, only the order matters
    return min(7, static_cast<int>(8.f * static_cast<float>(longest - x) * __builtin_amdgcn_rcpf(static_cast<float>(longest) + 1.f)));
  }
  __device__ __forceinline__ void plan(const PagedArgs& a) {
    load_batch(a, q, 0);
    uint64_t work = 0;
    each_seq<true>(a, q, [&](int, const addr::PagedSeq& sq) { work += addr::chunk_work2(sq, a.tq, a.window); });
    tiles = addr::chunk_part_tiles(static_cast<int64_t>(of_lane(lane_sums(work), 63)), a.chunk_share, kChunkLeast);
    magic = addr::div_magic(tiles);
    int most = 0;
    split = 0;
    each_seq<true>(a, q, [&](int, const addr::PagedSeq& sq) {
      const Count c = count(a, sq);
      most = max(most, c.longest);
      if (c.np > 1) split += static_cast<uint64_t>(c.nt) << 32 | static_cast<uint32_t>(c.nt * c.np);
    });
    longest = lanes_most(most);
    order = ClassOrder{0, 0, a.chunk_parts >= 65536};
    each_seq<true>(a, q, [&](int, const addr::PagedSeq& sq) {
      const Count c = count(a, sq);
      order.add(class_of(c.longest), c.nt * c.np);
    });
    total = order.place();
    const uint64_t to = lane_sums(split);
    // for the join, with the entries that the tiles' first parts write
    if (threadIdx.x == 0 && blockIdx.x == 0) a.chunk_list[0].x = static_cast<int>(of_lane(to, 63) >> 32);
    split = to - split;
  }
  // The r-th part (0 <= r < total).
  __device__ __forceinline__ ChunkItem part(const PagedArgs& a, int r) {
    ChunkItem it{-1, 0, 0, 1, 0, 0, {0, 0, 0}};
    uint64_t sp = split;
    each_seq<true>(a, q, [&](int s, const addr::PagedSeq& sq) {
      const Count c = count(a, sq);
      const int x = r - order.next(class_of(c.longest), c.nt * c.np);
      if (x >= 0 && x < c.nt * c.np) {
        it.s = s;
        it.j = c.nt * c.np - 1 - x;                  // a sequence's last tiles, the longest, first
        it.nparts = c.np;
        it.slot = static_cast<int>(static_cast<uint32_t>(sp));
        it.order = static_cast<int>(sp >> 32);
        it.sq = sq;
      }
      if (c.np > 1) sp += static_cast<uint64_t>(c.nt) << 32 | static_cast<uint32_t>(c.nt * c.np);
    });
    const int from = __builtin_ctzll(__ballot(it.s >= 0));
    const auto u = [&](int x) { return __builtin_amdgcn_readlane(x, from); };   // uniform, and known to be
    const int np = u(it.nparts), x = u(it.j), j = np > 1 ? x / np : x;
    return ChunkItem{u(it.s), j, x - j * np, np, np > 1 ? u(it.slot) + j * np : -1, u(it.order) + j, {u(it.sq.q0), u(it.sq.n), u(it.sq.len)}};
  }
};

// The maximum, or the sum, over a lane and the one 32 lanes away.
__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A part's query rows, as a lane has them: wave w rows 32 w .. 32 w + 31 of the tile's.
struct ChunkRow {
  addr::PagedTile tile;
  int kt0, kt1;                      // the part's key tiles
  int nrow, r;                       // rows of the tile; the lane's
  bool live, wave_live;
  int qh, hi, lo;                    // head; the lane's row sees [lo, hi)
  int64_t tok;
  int any_lo, any_hi, all_lo, all_hi;   // what the wave's rows see between them, and all of them
};
__device__ __forceinline__ ChunkRow chunk_row(const PagedArgs& a, const ChunkItem& it, int h) {
  const int tid = threadIdx.x, wave = tid >> 6, lq = tid & 31;
  const addr::PagedSeq& sq = it.sq;
  ChunkRow w;
  w.tile = addr::chunk_tile(sq, a.tq.tq, a.window, it.j);
  const int nkt = addr::chunk_key_tiles(w.tile);
  w.kt0 = 0;
  w.kt1 = nkt;
  if (it.nparts > 1) addr::chunk_part_range(nkt, it.part, it.nparts, w.kt0, w.kt1);
  w.nrow = (w.tile.i1 - w.tile.i0 + 1) * a.G;
  w.r = wave * 32 + lq;
  w.live = w.r < w.nrow;
  uint32_t r_q, r_h;
  addr::div_by(w.live ? w.r : 0, a.G, a.g_magic, r_q, r_h);
  const int qi = w.tile.i0 + static_cast<int>(r_q);
  w.qh = h * a.G + static_cast<int>(r_h);
  w.hi = w.live ? sq.len - sq.n + qi + 1 : 0;
  w.lo = a.window > 0 ? w.hi - a.window : 0;
  w.tok = sq.q0 + qi;
  const int w0 = wave * 32, w1 = min(w0 + 31, w.nrow - 1);
  w.wave_live = w0 < w.nrow;
  const int base_pos = sq.len - sq.n + w.tile.i0 + 1;
  w.all_hi = __builtin_amdgcn_readfirstlane(base_pos + w0 / a.G);
  w.any_hi = __builtin_amdgcn_readfirstlane(w.wave_live ? base_pos + w1 / a.G : 0);
  w.any_lo = a.window > 0 ? w.all_hi - a.window : 0;
  w.all_lo = a.window > 0 ? w.any_hi - a.window : 0;
  return w;
}

// The lane's query row: columns 16 st + 8 (l / 32) .. + 7 for every step.
template <int DT>
__device__ __forceinline__ void chunk_queries(const PagedArgs& a, const ChunkRow& w, u32x4 (&qf)[DT / 16]) {
  const int hl = (threadIdx.x >> 5) & 1;
  const char* qp = static_cast<const char*>(a.q) + (w.tok * a.q_ts + static_cast<int64_t>(w.qh) * a.q_hs) * 2;
#pragma unroll
  for (int st = 0; st < DT / 16; ++st) {
    const int d = 16 * st + 8 * hl;
    const u32x4 x = *reinterpret_cast<const u32x4*>(qp + (d < a.D ? d : 0) * 2);
    qf[st] = w.live && d < a.D ? x : u32x4{0, 0, 0, 0};
  }
}

// Running sums of the lane's row.
template <int DT>
struct ChunkSums {
  f32x16 o[DT / 32];                 // O^T tiles of 32 columns
  float m, lsum;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int d = 0; d < DT / 32; ++d)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[d][v] = 0.f;
    m = -INFINITY;
    lsum = 0.f;
  }
};

// Scores of the 64 keys of a tile: keys 32 u + mfma32_row(v, l), unscaled (`k0`: the lane's
// address of its keys in the tile).
template <int DT>
__device__ __forceinline__ void chunk_scores(const u32x4 (&qf)[DT / 16], const char* lds, uint32_t k0, f32x16 (&sc)[2]) {
  u32x4 kf[DT / 16][2];
#pragma unroll
  for (int st = 0; st < DT / 16; ++st)
#pragma unroll
    for (int u = 0; u < 2; ++u) kf[st][u] = ld16(lds + (k0 ^ (st * 32)) + u * 32 * DT * 2);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int v = 0; v < 16; ++v) sc[u][v] = 0.f;
#pragma unroll
  for (int st = 0; st < DT / 16; ++st)
#pragma unroll
    for (int u = 0; u < 2; ++u) sc[u] = mfma32_bf16(kf[st][u], qf[st], sc[u]);
}

// LDS address of the lane's values in a tile of 64 rows of DT bf16: the permutation is an
// exclusive or, so a column tile is one more on it.
template <int DT>
__device__ __forceinline__ uint32_t chunk_v_at() {
  const int l = threadIdx.x & 63, v_row = 4 * (l >> 5) + ((l & 15) >> 2);
  return v_row * DT * 2 + addr::chunk_v_pos(DT, v_row, 2 * ((l >> 4) & 1) + ((l & 3) >> 1)) * 16 + (l & 1) * 8;
}

// The scores of the 64 keys from tb on: softmax, and their values (`v0`: the lane's address
// in the tile) into the sums.
template <int DT>
__device__ __forceinline__ void chunk_values(const PagedArgs& a, const ChunkRow& w, int tb, f32x16 (&sc)[2], const char* lds,
                                             uint32_t v0, ChunkSums<DT>& sum) {
  constexpr int kRowB = DT * 2, kDT = DT / 32;
  const int l = threadIdx.x & 63;
  // the first half of V under the softmax
  uint64_t vf[kDT][4][2];
  const auto read_v = [&](int d) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int x = 0; x < 2; ++x) vf[d][g][x] = read_tr(lds + (v0 ^ (d * 64)) + (g * 16 + 8 * x) * kRowB);
  };
#pragma unroll
  for (int d = 0; d < kDT / 2; ++d) read_v(d);
  __builtin_amdgcn_sched_barrier(0);
  if (tb + kCKeys > w.all_hi || tb < w.all_lo) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int t = tb + 32 * u + mfma32_row(v, l);
        if (t >= w.hi || t < w.lo) sc[u][v] = -INFINITY;
      }
  }
  float mx = sc[0][0];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int v = 0; v < 16; ++v) mx = fmaxf(mx, sc[u][v]);
  mx = max_halves(mx) * a.scale_log2;
  // the reference point follows the maximum once it has grown by 2^8: the sums
  // stay far from their limits, and o is rarely scaled
  if (__any(mx > sum.m + 8.f)) {
    const float mn = fmaxf(sum.m, mx);
    const float f = sum.m == mn ? 1.f : __builtin_amdgcn_exp2f(sum.m - mn);
    sum.m = mn;
    sum.lsum *= f;
#pragma unroll
    for (int d = 0; d < kDT; ++d)
#pragma unroll
      for (int v = 0; v < 16; ++v) sum.o[d][v] *= f;
  }
  const float ms = sum.m == -INFINITY ? 0.f : sum.m;
  u32x4 pf[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = __builtin_amdgcn_exp2f(fmaf(sc[g >> 1][8 * (g & 1) + i], a.scale_log2, -ms));
      sum.lsum += p[i];
    }
    // Probabilities are rounded to bf16, each off by up to 2^-8 of itself; their total stays in
    // fp32.  Two bf16 numbers for each, off by 2^-16, are half as many products again, where
    // instructions bound: over a quantised cache 121 -> 143 us for 8192 rows of prompts, 90 -> 106
    // for a step of 48 decode rows and 16 chunks, 58 -> 67 for 8 chunks of 3 .. 64 rows.
#pragma unroll
    for (int i = 0; i < 4; ++i) pf[g][i] = pack_bf16x2(p[2 * i], p[2 * i + 1]);
  }
#pragma unroll
  for (int d = kDT / 2; d < kDT; ++d) read_v(d);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int d = 0; d < kDT; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const u32x4 x = {static_cast<uint32_t>(vf[d][g][0]), static_cast<uint32_t>(vf[d][g][0] >> 32),
                       static_cast<uint32_t>(vf[d][g][1]), static_cast<uint32_t>(vf[d][g][1] >> 32)};
      sum.o[d] = mfma32_bf16(x, pf[g], sum.o[d]);
    }
}

// A whole tile's rows, or a part's partial result.
template <int DT>
__device__ __forceinline__ void chunk_results(const PagedArgs& a, const ChunkItem& it, int h, const ChunkRow& w, ChunkSums<DT>& sum) {
  constexpr int kDT = DT / 32;
  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63, hl = l >> 5;
  const addr::PagedSeq& sq = it.sq;
  f32x16 (&o)[kDT] = sum.o;
  const float m = sum.m, lsum = sum_halves(sum.lsum);
  if (it.slot < 0) {
    const float inv = lsum == 0.f ? 0.f : 1.0f / lsum;
    uint16_t* out = static_cast<uint16_t*>(a.out) + w.tok * a.o_ts + static_cast<int64_t>(w.qh) * a.o_hs;
    // A lane has columns 8 k + 4 hl .. + 3 of its row for every k: swapped between the
    // two halves of the wave, 8 consecutive ones of every other k.
#pragma unroll
    for (int d = 0; d < kDT; ++d)
#pragma unroll
      for (int v = 0; v < 16; v += 8) {
        uint32_t x4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = lsum == 0.f ? 0.f : o[d][v + 2 * i] * inv, y = lsum == 0.f ? 0.f : o[d][v + 2 * i + 1] * inv;
          x4[i] = pack_bf16x2(x, y);
        }
        const auto p0 = __builtin_amdgcn_permlane32_swap(x4[0], x4[2], false, false);
        const auto p1 = __builtin_amdgcn_permlane32_swap(x4[1], x4[3], false, false);
        const int col = 32 * d + 2 * v + 8 * hl;
        if (w.live && col < a.D) *reinterpret_cast<u32x4*>(out + col) = u32x4{p0[0], p1[0], p0[1], p1[1]};
      }
    if (a.lse != nullptr && hl == 0 && w.live) a.lse[w.tok * a.H + w.qh] = lsum == 0.f ? -INFINITY : (m + log2f(lsum)) * 0.6931471805599453f;
    return;
  }
  float* p = a.chunk_ws + (static_cast<int64_t>(h) * addr::chunk_slots_per_head(a.HK, a.chunk_slots) + it.slot + it.part) *
                              addr::chunk_partial_floats(kChunkRows, DT);
  if (w.wave_live) {                                   // in the order of the registers: whole lines
#pragma unroll
    for (int d = 0; d < kDT; ++d)
#pragma unroll
      for (int v = 0; v < 16; v += 4)
        *reinterpret_cast<f32x4*>(p + ((((wave * kDT + d) * 4 + (v >> 2)) * 64 + l) << 2)) =
            f32x4{o[d][v], o[d][v + 1], o[d][v + 2], o[d][v + 3]};
    if (hl == 0 && w.live) {
      p[kChunkRows * DT + w.r] = m;
      p[kChunkRows * (DT + 1) + w.r] = lsum;
    }
  }
  if (it.part == 0 && h == 0 && tid == 0) a.chunk_list[1 + it.order] = make_int4(sq.q0 + w.tile.i0, w.nrow, it.nparts, it.slot);
}

// The split tiles' parts, joined in the order of their keys: workgroups take (tile,
// an eighth of it, head) in turn, a thread 4 columns of a row, 8 parts' loads in
// flight.  (A workgroup that joined its tile at the end of the launch above would read
// all its parts alone: 14 parts of 128 rows took it 50 us.)
template <int DT>
__global__ __launch_bounds__(256) void chunk_join_kernel(PagedArgs a) {
  constexpr int kBatch = 8;
  constexpr int kGroups = 8, kDT = DT / 32;
  const int64_t size = addr::chunk_partial_floats(kChunkRows, DT);
  const int total = a.chunk_list[0].x * kGroups * a.HK;
  for (int w = blockIdx.x; w < total; w += gridDim.x) {
    const int h = w % a.HK, g = (w / a.HK) % kGroups;
    const int4 e = a.chunk_list[1 + w / (a.HK * kGroups)];
    const float* first = a.chunk_ws + (static_cast<int64_t>(h) * addr::chunk_slots_per_head(a.HK, a.chunk_slots) + e.w) * size;
    for (int y = threadIdx.x; y < 128 * kDT; y += 256) {
      const int x = g * 128 * kDT + y, l = x & 63;   // the x-th four floats: chunk_part's order
      const int jr = x / (256 * kDT) * 32 + (l & 31), d = (x / 256 % kDT) * 32 + ((x >> 6) & 3) * 8 + (l >> 5) * 4;
      if (jr >= e.y) continue;
      float M = -INFINITY, L = 0.f;
      f32x4 acc = {0, 0, 0, 0};
      for (int p0 = 0; p0 < e.z; p0 += kBatch) {
        f32x4 px[kBatch];
        float pm[kBatch], pl[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const float* p = first + min(p0 + k, e.z - 1) * size;
          px[k] = *reinterpret_cast<const f32x4*>(p + 4 * x);
          pm[k] = p[kChunkRows * DT + jr];
          pl[k] = p[kChunkRows * (DT + 1) + jr];
        }
        float Mn = M;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) Mn = fmaxf(Mn, pm[k]);
        const float ms = Mn == -INFINITY ? 0.f : Mn;
        const float f0 = __builtin_amdgcn_exp2f(M - ms);           // M = -inf: nothing summed yet
        L *= f0;
        acc *= f0;
        M = Mn;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const float f = p0 + k < e.z ? __builtin_amdgcn_exp2f(pm[k] - ms) : 0.f;
          L += f * pl[k];
          acc += f * px[k];
        }
      }
      uint32_t jq, jh;
      addr::div_by(jr, a.G, a.g_magic, jq, jh);
      row_store<true>(a, e.x + static_cast<int>(jq), h * a.G + static_cast<int>(jh), d, acc, M, L);
    }
  }
  zero_outside<true>(a);
}

// A workgroup of a ragged launch (grid: addr::ragged_role): its part of the row form, or
// of the chunk form by `chunk`.
template <int DT, bool E4M3, class F>
__device__ __forceinline__ void ragged_work(char* lds, const F& chunk) {
  int i;
  if (addr::ragged_role(blockIdx.x, fresh_args().ragged_block, fresh_args().row_blocks, i)) {
    const PagedArgs& a = fresh_args();
    const int r = i / a.HK, h = i - r * a.HK;
    RowOrder<true, DT> order;
    order.plan(a);
    if (r < order.total) row_part<true, DT, E4M3>(fresh_args(), order.part(a, r), h, *reinterpret_cast<RowShared<DT>*>(lds));
  } else {
    const PagedArgs& a = fresh_args();
    ChunkOrder order;
    order.plan(a);
    const int r = i / a.HK, h = i - r * a.HK;        // 8 heads: a head's parts on one XCD
    if (r < order.total) chunk(fresh_args(), order.part(a, r), h);
  }
}

}  // namespace
}  // namespace gs
