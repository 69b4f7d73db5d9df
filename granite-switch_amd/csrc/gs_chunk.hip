// Attention of a ragged bf16 batch over a paged cache (head widths up to 128, a scale
// above zero): one launch in which sequences of many rows take the chunk form here and
// those of few (a decode row among prompts) the row form (gs_paged_rows.h).
//
// Two workgroups share a compute unit: parts of the row form, which stream the cache,
// and of the chunk form, which multiply, are launched in turn.
//
// The chunk form.
// A workgroup of 4 waves takes 128 (query, head) rows of one sequence and
// key/value head -- 32 queries where 4 query heads share it, so the group's
// heads read K and V once -- and walks the keys in tiles of 64.  Keys and values
// go from the pages straight into LDS (two stages), 16 bytes a lane, permuted so
// that every operand read falls on different banks.  Two workgroups share a
// compute unit: one multiplies while the other is in its softmax, its start or
// its end.
//
// Per wave, 32 rows: S^T = K Q^T with 32 x 32 x 16 products, the keys as rows.  A
// lane then has one query row: the running maximum and total are its own, and its
// 16 scores of 32 keys are, packed in order, the operand that O^T = V^T P^T takes
// (its keys permuted alike: V^T is read transposed from LDS, 4 keys at a time).
//
// 4 D operations a score, and on the vector units its exponential, maximum, total and
// packing: these take 54% of the SIMDs' cycles and the products 30% (prompts), with two waves a
// SIMD to overlap them.  8192 rows of 16 prompts (32 query, 8 key/value heads of 128):
// 105 us, 620 TFLOP/s of the products that the mask leaves, where a large library product
// reaches 1586.  A step of 48 decode rows and 16 chunks of 256 over up to 3839 keys: 90 us.
#include <algorithm>

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

// One part: 128 rows of a sequence and head h over its key tiles.
template <int DT>
__device__ __forceinline__ void chunk_part(const PagedArgs& a, const ChunkItem& it, int h, char* lds) {
  constexpr int kRowB = DT * 2;                     // bytes of a key row in LDS
  constexpr int kTileB = kCKeys * kRowB;            // of a stage's keys, and of its values
  constexpr int kStageB = 2 * kTileB;
  constexpr int kRowsPer = 1024 / kRowB;            // rows a wave transfer moves
  constexpr int kMoves = 8 / kRowsPer;              // transfers for 8 keys (as many for the values); a wave moves 16 keys
  constexpr int kSteps = DT / 16;
  constexpr int kDT = DT / 32;                      // O^T tiles of 32 columns

  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63;
  const int lq = l & 31, hl = l >> 5;
  const int s = it.s;
  const addr::PagedSeq& sq = it.sq;
  const addr::PagedTile tile = addr::chunk_tile(sq, a.tq.tq, a.window, it.j);
  const int nkt = addr::chunk_key_tiles(tile);
  int kt0 = 0, kt1 = nkt;
  if (it.nparts > 1) addr::chunk_part_range(nkt, it.part, it.nparts, kt0, kt1);

  // ---- the lane's query row ---------------------------------------------------
  const int nrow = (tile.i1 - tile.i0 + 1) * a.G;
  const int r = wave * 32 + lq;
  const bool live = r < nrow;
  uint32_t r_q, r_h;
  addr::div_by(live ? r : 0, a.G, a.g_magic, r_q, r_h);
  const int qi = tile.i0 + static_cast<int>(r_q);
  const int qh = h * a.G + static_cast<int>(r_h);
  const int hi = live ? sq.len - sq.n + qi + 1 : 0;                // sees [lo, hi)
  const int lo = a.window > 0 ? hi - a.window : 0;
  const int64_t tok = sq.q0 + qi;
  u32x4 qf[kSteps];
  {
    const char* qp = static_cast<const char*>(a.q) + (tok * a.q_ts + static_cast<int64_t>(qh) * a.q_hs) * 2;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const int d = 16 * st + 8 * hl;
      const u32x4 x = *reinterpret_cast<const u32x4*>(qp + (d < a.D ? d : 0) * 2);
      qf[st] = live && d < a.D ? x : u32x4{0, 0, 0, 0};
    }
  }
  // what the wave's rows see between them: [any_lo, any_hi); all of them: [all_lo, all_hi)
  const int w0 = wave * 32, w1 = min(w0 + 31, nrow - 1);
  const bool wave_live = w0 < nrow;
  const int base_pos = sq.len - sq.n + tile.i0 + 1;
  const int all_hi = __builtin_amdgcn_readfirstlane(base_pos + w0 / a.G);
  const int any_hi = __builtin_amdgcn_readfirstlane(wave_live ? base_pos + w1 / a.G : 0);
  const int any_lo = a.window > 0 ? all_hi - a.window : 0, all_lo = a.window > 0 ? any_hi - a.window : 0;

  // ---- transfers ------------------------------------------------------------------
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr_t)(lds)));
  const int32_t* trow = a.table + static_cast<int64_t>(s) * a.ld_table;
  const int t_row = l / (64 / kRowsPer), t_pos = l % (64 / kRowsPer);   // the lane's row and LDS position in a transfer
  // Where the wave's keys are: lanes 2 i and 2 i + 1 hold the byte offsets of the
  // wave's 16 keys in tile i of 32 (its first 8 and its last 8), one load of page
  // ids and one division for 32 tiles.
  const int wave_u = __builtin_amdgcn_readfirstlane(wave);
  const char* k_head = static_cast<const char*>(a.k) + static_cast<int64_t>(h) * a.k_hs * 2;
  const char* v_head = static_cast<const char*>(a.v) + static_cast<int64_t>(h) * a.v_hs * 2;
  int64_t k_from = 0, v_from = 0;
  const auto load_ids = [&](int kt) {
    uint32_t pg, row8;
    const int oct = addr::paged_octet(tile.first + (kt + (l >> 1)) * kCKeys + 16 * wave + 8 * (l & 1), tile.ve);
    addr::div_by(static_cast<uint32_t>(oct) >> 3, a.page_octets, a.page_magic, pg, row8);
    const int64_t page = addr::paged_page(trow[pg], a.num_pages);
    k_from = (page * a.k_ps + static_cast<int64_t>(row8 * 8) * a.k_rs) * 2;
    v_from = (page * a.v_ps + static_cast<int64_t>(row8 * 8) * a.v_rs) * 2;
  };
  const auto lane64 = [](int64_t x, int i) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(x), i);
    const uint32_t up = __builtin_amdgcn_readlane(static_cast<uint32_t>(static_cast<uint64_t>(x) >> 32), i);
    return static_cast<int64_t>(lo | (static_cast<uint64_t>(up) << 32));
  };
  // Whole rows within 32-bit offsets: a transfer is a uniform base and these.
  const bool plain = a.D == DT && a.k_rs < (1 << 26) && a.v_rs < (1 << 26);
  uint32_t k_off[kMoves], v_off[kMoves];
#pragma unroll
  for (int x = 0; x < kMoves; ++x) {
    const int row = x * kRowsPer + t_row;              // of 8: the permutation is the same for each 8 rows or repeats in 16
    k_off[x] = static_cast<uint32_t>(row * a.k_rs) * 2;
    v_off[x] = static_cast<uint32_t>(row * a.v_rs + addr::chunk_v_pos(DT, row, t_pos) * 8) * 2;
  }
  uint32_t k_pos[2][kMoves];
#pragma unroll
  for (int oc = 0; oc < 2; ++oc)
#pragma unroll
    for (int x = 0; x < kMoves; ++x) k_pos[oc][x] = k_off[x] + addr::chunk_k_pos(DT, 8 * oc + x * kRowsPer + t_row, t_pos) * 16;
  const auto issue = [&](int kt, int stage) {
    const int i32 = (kt - kt0) & 31;
    if (i32 == 0) load_ids(kt);
#pragma unroll
    for (int oc = 0; oc < 2; ++oc) {
      const char* kbase = k_head + lane64(k_from, 2 * i32 + oc);
      const char* vbase = v_head + lane64(v_from, 2 * i32 + oc);
      const uint32_t dst = lds0 + stage * kStageB + (16 * wave_u + 8 * oc) * kRowB;
      const int t0 = tile.first + kt * kCKeys + 16 * wave_u + 8 * oc;
      if (plain && t0 >= tile.vs && t0 + 8 <= tile.ve) {
#pragma unroll
        for (int x = 0; x < kMoves; ++x) {
          dma16_off(kbase, k_pos[oc][x], dst + x * 1024);
          dma16_off(vbase, v_off[x], dst + x * 1024 + kTileB);
        }
      } else {
        const char* zero = reinterpret_cast<const char*>(&g_zero16);
#pragma unroll
        for (int x = 0; x < kMoves; ++x) {
          const int row = x * kRowsPer + t_row;
          const int kp = addr::chunk_k_pos(DT, 8 * oc + row, t_pos), vp = addr::chunk_v_pos(DT, row, t_pos);
          const bool seen = t0 + row >= tile.vs && t0 + row < tile.ve;
          dma16_row(kp * 8 < a.D ? kbase + (row * a.k_rs + kp * 8) * 2 : zero, dst + x * 1024);
          dma16_row(seen && vp * 8 < a.D ? vbase + (row * a.v_rs + vp * 8) * 2 : zero, dst + x * 1024 + kTileB);
        }
      }
    }
  };

  f32x16 o[kDT];
#pragma unroll
  for (int d = 0; d < kDT; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = 0.f;
  float m = -INFINITY, lsum = 0.f;

  // LDS addresses of the lane's operand rows: the permutations are exclusive ors, so
  // a K step or a column tile is one more on the address of the first.
  const uint32_t k_at = lq * kRowB + addr::chunk_k_pos(DT, lq, hl) * 16;
  const int v_row = 4 * hl + ((l & 15) >> 2);
  const uint32_t v_at = kTileB + v_row * kRowB + addr::chunk_v_pos(DT, v_row, 2 * ((l >> 4) & 1) + ((l & 3) >> 1)) * 16 + (l & 1) * 8;

  // Tile kt, in `stage`; `next` tells whether tile kt + 1 is moved to the other one.
  const auto compute = [&](int kt, int stage, bool next) {
    const int tb = tile.first + kt * kCKeys;
    const bool active = wave_live && tb < any_hi && tb + kCKeys > any_lo;
    // every read of K on its way before the first product, the transfers' addresses made meanwhile
    u32x4 kf[kSteps][2];
    if (active) {
#pragma unroll
      for (int st = 0; st < kSteps; ++st)
#pragma unroll
        for (int u = 0; u < 2; ++u) kf[st][u] = ld16(lds + ((k_at + stage * kStageB) ^ (st * 32)) + u * 32 * kRowB);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (next) issue(kt + 1, stage ^ 1);              // the stage of tile kt - 1, which every wave is past
    if (!active) return;
    f32x16 sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) sc[u][v] = 0.f;
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int u = 0; u < 2; ++u) sc[u] = mfma32_bf16(kf[st][u], qf[st], sc[u]);
    // the first half of V under the softmax
    uint64_t vf[kDT][4][2];
    const auto read_v = [&](int d) {
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int x = 0; x < 2; ++x) vf[d][g][x] = read_tr(lds + ((v_at + stage * kStageB) ^ (d * 64)) + (g * 16 + 8 * x) * kRowB);
    };
#pragma unroll
    for (int d = 0; d < kDT / 2; ++d) read_v(d);
    __builtin_amdgcn_sched_barrier(0);
    if (tb + kCKeys > all_hi || tb < all_lo) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int t = tb + 32 * u + mfma32_row(v, l);
          if (t >= hi || t < lo) sc[u][v] = -INFINITY;
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
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx);
      const float f = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      lsum *= f;
#pragma unroll
      for (int d = 0; d < kDT; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] *= f;
    }
    const float ms = m == -INFINITY ? 0.f : m;
    u32x4 pf[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = __builtin_amdgcn_exp2f(fmaf(sc[g >> 1][8 * (g & 1) + i], a.scale_log2, -ms));
        lsum += p[i];
      }
      // bf16 probabilities with the error they have in the row form; two bf16 numbers for each
      // are half as many products again, where instructions bound.  The total stays in fp32.
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
        o[d] = mfma32_bf16(x, pf[g], o[d]);
      }
  };

  // ---- the walk over the keys ---------------------------------------------------
  const int n = kt1 - kt0;
  if (n > 0) {
    issue(kt0, 0);
    int stage = 0;
    for (int i = 0; i < n; ++i) {
      mem_fence_compiler();
      __builtin_amdgcn_s_waitcnt(wait_vm_lds0(0));                 // own transfers landed, own reads done
      __builtin_amdgcn_s_barrier();
      mem_fence_compiler();
      compute(kt0 + i, stage, i + 1 < n);
      stage ^= 1;
    }
  }

  // ---- results --------------------------------------------------------------------
  lsum = sum_halves(lsum);
  if (it.slot < 0) {
    const float inv = lsum == 0.f ? 0.f : 1.0f / lsum;
    uint16_t* out = static_cast<uint16_t*>(a.out) + tok * a.o_ts + static_cast<int64_t>(qh) * a.o_hs;
    // A lane has columns 8 k + 4 hl .. + 3 of its row for every k: swapped between the
    // two halves of the wave, 8 consecutive ones of every other k.
#pragma unroll
    for (int d = 0; d < kDT; ++d)
#pragma unroll
      for (int v = 0; v < 16; v += 8) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = lsum == 0.f ? 0.f : o[d][v + 2 * i] * inv, y = lsum == 0.f ? 0.f : o[d][v + 2 * i + 1] * inv;
          w[i] = pack_bf16x2(x, y);
        }
        const auto p0 = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
        const auto p1 = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
        const int col = 32 * d + 2 * v + 8 * hl;
        if (live && col < a.D) *reinterpret_cast<u32x4*>(out + col) = u32x4{p0[0], p1[0], p0[1], p1[1]};
      }
    if (a.lse != nullptr && hl == 0 && live) a.lse[tok * a.H + qh] = lsum == 0.f ? -INFINITY : (m + log2f(lsum)) * 0.6931471805599453f;
    return;
  }
  float* p = a.chunk_ws + (static_cast<int64_t>(h) * addr::chunk_slots_per_head(a.HK, a.chunk_slots) + it.slot + it.part) *
                              addr::chunk_partial_floats(kChunkRows, DT);
  if (wave_live) {                                   // in the order of the registers: whole lines
#pragma unroll
    for (int d = 0; d < kDT; ++d)
#pragma unroll
      for (int v = 0; v < 16; v += 4)
        *reinterpret_cast<f32x4*>(p + ((((wave * kDT + d) * 4 + (v >> 2)) * 64 + l) << 2)) =
            f32x4{o[d][v], o[d][v + 1], o[d][v + 2], o[d][v + 3]};
    if (hl == 0 && live) {
      p[kChunkRows * DT + r] = m;
      p[kChunkRows * (DT + 1) + r] = lsum;
    }
  }
  if (it.part == 0 && h == 0 && tid == 0) a.chunk_list[1 + it.order] = make_int4(sq.q0 + tile.i0, nrow, it.nparts, it.slot);
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

// Grid: addr::ragged_role.
template <int DT>
__global__ __launch_bounds__(64 * kCWaves, 2) void ragged_attention_kernel(PagedArgs) {
  __shared__ __attribute__((aligned(1024))) char lds[addr::cmax(kCStages * 2 * kCKeys * DT * 2, static_cast<int>(sizeof(RowShared<DT>)))];
  int i;
  if (addr::ragged_role(blockIdx.x, fresh_args().ragged_block, fresh_args().row_blocks, i)) {
    const PagedArgs& a = fresh_args();
    const int r = i / a.HK, h = i - r * a.HK;
    RowOrder<true, DT> order;
    order.plan(a);
    if (r < order.total) row_part<true, DT>(fresh_args(), order.part(a, r), h, *reinterpret_cast<RowShared<DT>*>(lds));
  } else {
    const PagedArgs& a = fresh_args();
    ChunkOrder order;
    order.plan(a);
    const int r = i / a.HK, h = i - r * a.HK;        // 8 heads: a head's parts on one XCD
    if (r < order.total) chunk_part<DT>(fresh_args(), order.part(a, r), h, lds);
  }
}

}  // namespace

int chunk_slots_for(int cus) { return 2 * cus; }

int64_t chunk_list_floats(int HK, int cus) { return 4 * (1 + static_cast<int64_t>(addr::chunk_slots_per_head(HK, chunk_slots_for(cus))) / 2); }

int64_t chunk_workspace_bytes(int HK, int DT, int cus) {
  return static_cast<int64_t>(HK) * addr::chunk_slots_per_head(HK, chunk_slots_for(cus)) * addr::chunk_partial_floats(kChunkRows, DT) * 4;
}

// Tiles of a head at most: each sequence may end with a partial one.
static int64_t chunk_most_tiles(const PagedArgs& a) {
  return a.T / a.tq.tq + std::min(a.B, a.T / (a.row_limit / a.G + 1));   // a tile more for each sequence of more rows than row_limit
}

// Parts at most: tiles, and the split tiles' parts.
int64_t chunk_most_parts(const PagedArgs& a) {
  return chunk_most_tiles(a) + addr::chunk_slots_per_head(a.HK, a.chunk_slots);
}

int64_t ragged_grid(const PagedArgs& a) {
  return static_cast<int64_t>(a.row_blocks) * a.ragged_block +
         std::max<int64_t>(static_cast<int64_t>(a.row_blocks) * a.ragged_block, (a.chunk_parts * a.HK + 7) & ~int64_t(7));
}

void launch_ragged(const PagedArgs& a, int DT, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(ragged_grid(a)));
  const dim3 join(static_cast<unsigned>(a.chunk_slots));
  if (DT == 64) {
    hipLaunchKernelGGL((ragged_attention_kernel<64>), grid, dim3(64 * kCWaves), 0, st, a);
    hipLaunchKernelGGL((chunk_join_kernel<64>), join, dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((ragged_attention_kernel<128>), grid, dim3(64 * kCWaves), 0, st, a);
    hipLaunchKernelGGL((chunk_join_kernel<128>), join, dim3(256), 0, st, a);
  }
}

}  // namespace gs
