// Attention of query chunks over a paged cache (bf16, head widths up to 128):
// the form of gs_paged_attention for sequences of many rows.
//
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
#include <algorithm>

#include "gs_paged.h"

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
  int s, j, part, nparts, slot;      // slot: its partial result's, or -1
  addr::PagedSeq sq;
};
struct ChunkShared {
  int64_t work[4];
  int items[4], split[4];
  int found[8];
};

__device__ __forceinline__ int wave_scan(int v) {
  const int l = lane_id();
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(v, d, 64);
    if (l >= d) v += u;
  }
  return v;
}

// The r-th part (JOIN: the r-th tile that was split) of the batch's tiles for one
// head, in order of sequences, tiles and parts.  by_xcd: r is a workgroup of
// (part, head) pairs.  Every thread of a workgroup of 256 calls it.
template <bool JOIN>
__device__ __forceinline__ ChunkItem find_chunk(const PagedArgs& a, int r, bool by_xcd, int& h, ChunkShared& sh) {
  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63;
  const int run = (a.B + 255) >> 8;
  const int s0 = min(tid * run, a.B), s1 = min(s0 + run, a.B);
  addr::PagedSeq first{0, 0, 0};                     // the thread's first sequence: its only one up to 256
  if (s0 < s1) first = seq_of_form<true>(a, s0);
  int64_t work = addr::chunk_work2(first, a.tq, a.window);
  for (int s = s0 + 1; s < s1; ++s) work += addr::chunk_work2(seq_of_form<true>(a, s), a.tq, a.window);
#pragma unroll
  for (int d = 32; d; d >>= 1) work += __shfl_xor(work, d, 64);
  if (l == 0) sh.work[wave] = work;
  if (tid == 0) sh.found[0] = -1;
  __syncthreads();
  const int pt = addr::chunk_part_tiles(sh.work[0] + sh.work[1] + sh.work[2] + sh.work[3], a.chunk_share, kChunkLeast);
  const uint32_t pm = addr::div_magic(pt);
  struct Count {
    int nt, np, items, split;                        // items: parts (JOIN: split tiles); split: partial results
  };
  const auto count = [&](const addr::PagedSeq& sq) {
    Count c;
    c.nt = addr::chunk_tiles(sq, a.tq);
    c.np = addr::chunk_parts(sq, a.tq, a.window, pt, pm);
    c.split = c.np > 1 ? c.nt * c.np : 0;
    c.items = JOIN ? (c.np > 1 ? c.nt : 0) : c.nt * c.np;
    return c;
  };
  const Count c0 = count(first);
  int items = c0.items, split = c0.split;
  for (int s = s0 + 1; s < s1; ++s) {
    const Count c = count(seq_of_form<true>(a, s));
    items += c.items;
    split += c.split;
  }
  int at = wave_scan(items), sl = wave_scan(split);
  if (l == 63) {
    sh.items[wave] = at;
    sh.split[wave] = sl;
  }
  __syncthreads();
  int n = 0;
  at -= items;
  sl -= split;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) {
      at += sh.items[w];
      sl += sh.split[w];
    }
    n += sh.items[w];
  }
  if (by_xcd) {
    // consecutive workgroups go to the XCDs in turn: each XCD takes a contiguous
    // range of (head, part), so a sequence's tiles share one L2's keys
    const int total = n * a.HK, per = (total + 7) >> 3;
    const int t = (r & 7) * per + (r >> 3);
    if ((r >> 3) >= per || t >= total) {
      r = -1;
    } else {
      h = t / n;
      r = n - 1 - (t - h * n);                       // a sequence's last tiles, the longest, first
    }
  }
  if (r >= at && r < at + items) {
    addr::PagedSeq sq = first;
    for (int s = s0;; ++s) {
      if (s > s0) sq = seq_of_form<true>(a, s);
      const Count c = count(sq);
      if (r < at + c.items) {
        const int k = r - at;
        sh.found[0] = s;
        sh.found[1] = JOIN ? k : k / c.np;
        sh.found[2] = JOIN ? 0 : k % c.np;
        sh.found[3] = c.np;
        sh.found[4] = c.np > 1 ? sl + (JOIN ? k * c.np : k) : -1;
        sh.found[5] = sq.q0;
        sh.found[6] = sq.n;
        sh.found[7] = sq.len;
        break;
      }
      at += c.items;
      sl += c.split;
    }
  }
  __syncthreads();
  const int* f = sh.found;
  const auto u = [](int x) { return __builtin_amdgcn_readfirstlane(x); };   // uniform, and known to be
  h = u(h);
  return ChunkItem{u(f[0]), u(f[1]), u(f[2]), u(f[3]), u(f[4]), {u(f[5]), u(f[6]), u(f[7])}};
}

__device__ __forceinline__ void store4(const PagedArgs& a, int64_t e, f32x4 x) {
  uint32_t* p = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + e);
  const uint64_t w = pack_bf16x2(x[0], x[1]) | (static_cast<uint64_t>(pack_bf16x2(x[2], x[3])) << 32);
  *reinterpret_cast<uint64_t*>(p) = w;
}

template <int DT>
__global__ __launch_bounds__(64 * kCWaves, 2) void chunk_attention_kernel(PagedArgs a) {
  constexpr int kRowB = DT * 2;                     // bytes of a key row in LDS
  constexpr int kTileB = kCKeys * kRowB;            // of a stage's keys, and of its values
  constexpr int kStageB = 2 * kTileB;
  constexpr int kRowsPer = 1024 / kRowB;            // rows a wave transfer moves
  constexpr int kMoves = 8 / kRowsPer;              // transfers for 8 keys (as many for the values); a wave moves 16 keys
  constexpr int kSteps = DT / 16;
  constexpr int kDT = DT / 32;                      // O^T tiles of 32 columns
  __shared__ __attribute__((aligned(1024))) char lds[kCStages * kStageB];
  __shared__ ChunkShared sh;

  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63;
  const int lq = l & 31, hl = l >> 5;
  int h = 0;
  const ChunkItem it = find_chunk<false>(a, blockIdx.x, true, h, sh);
  if (it.s < 0) return;
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

  // LDS addresses of the lane's operand rows, per K step and per column tile
  uint32_t k_at[kSteps], v_at[kDT];
#pragma unroll
  for (int st = 0; st < kSteps; ++st) k_at[st] = lq * kRowB + addr::chunk_k_pos(DT, lq, 2 * st + hl) * 16;
  const int v_row = 4 * hl + ((l & 15) >> 2);
#pragma unroll
  for (int d = 0; d < kDT; ++d)
    v_at[d] = kTileB + v_row * kRowB + addr::chunk_v_pos(DT, v_row, 4 * d + 2 * ((l >> 4) & 1) + ((l & 3) >> 1)) * 16 + (l & 1) * 8;

  // Tile kt, in `stage`; `next` tells whether tile kt + 1 is moved to the other one.
  const auto compute = [&](int kt, int stage, bool next) {
    const int tb = tile.first + kt * kCKeys;
    const char* base = lds + stage * kStageB;
    const bool active = wave_live && tb < any_hi && tb + kCKeys > any_lo;
    // every read of K on its way before the first product, the transfers' addresses made meanwhile
    u32x4 kf[kSteps][2];
    if (active) {
#pragma unroll
      for (int st = 0; st < kSteps; ++st)
#pragma unroll
        for (int u = 0; u < 2; ++u) kf[st][u] = ld16(base + k_at[st] + u * 32 * kRowB);
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
        for (int x = 0; x < 2; ++x) vf[d][g][x] = read_tr(base + v_at[d] + (g * 16 + 8 * x) * kRowB);
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
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * a.scale_log2;
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
      // bf16 probabilities (relative error 2^-8, as the values and the result have); the total stays in fp32
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
  lsum += __shfl_xor(lsum, 32, 64);
  if (!live) return;
  if (it.slot < 0) {
    const float inv = lsum == 0.f ? 0.f : 1.0f / lsum;
    const int64_t e = tok * a.o_ts + static_cast<int64_t>(qh) * a.o_hs;
#pragma unroll
    for (int d = 0; d < kDT; ++d)
#pragma unroll
      for (int v = 0; v < 16; v += 4) {
        const int col = 32 * d + mfma32_row(v, l);
        f32x4 x = {o[d][v], o[d][v + 1], o[d][v + 2], o[d][v + 3]};
        x = lsum == 0.f ? f32x4{0, 0, 0, 0} : x * inv;
        if (col < a.D) store4(a, e + col, x);
      }
    if (a.lse != nullptr && hl == 0) a.lse[tok * a.H + qh] = lsum == 0.f ? -INFINITY : (m + log2f(lsum)) * 0.6931471805599453f;
  } else {
    float* p = a.chunk_ws + (static_cast<int64_t>(h) * addr::chunk_slots_per_head(a.HK, a.chunk_slots) + it.slot) * addr::chunk_partial_floats(kChunkRows, DT);
#pragma unroll
    for (int d = 0; d < kDT; ++d)
#pragma unroll
      for (int v = 0; v < 16; v += 4)
        *reinterpret_cast<f32x4*>(p + r * DT + 32 * d + mfma32_row(v, l)) = f32x4{o[d][v], o[d][v + 1], o[d][v + 2], o[d][v + 3]};
    if (hl == 0) {
      p[kChunkRows * DT + r] = m;
      p[kChunkRows * (DT + 1) + r] = lsum;
    }
  }
}

// The parts of a tile joined, in the order of their keys: grid (split tiles x row groups, heads).
constexpr int kJoinRows = 32;
template <int DT>
__global__ __launch_bounds__(256) void chunk_join_kernel(PagedArgs a) {
  __shared__ ChunkShared sh;
  int h = blockIdx.y;
  const ChunkItem it = find_chunk<true>(a, blockIdx.x / (kChunkRows / kJoinRows), false, h, sh);
  if (it.s < 0) return;
  const addr::PagedSeq& sq = it.sq;
  const addr::PagedTile tile = addr::chunk_tile(sq, a.tq.tq, a.window, it.j);
  const int nrow = (tile.i1 - tile.i0 + 1) * a.G;
  const int64_t size = addr::chunk_partial_floats(kChunkRows, DT);
  const float* first = a.chunk_ws + (static_cast<int64_t>(h) * addr::chunk_slots_per_head(a.HK, a.chunk_slots) + it.slot) * size;
  const int r0 = (blockIdx.x % (kChunkRows / kJoinRows)) * kJoinRows;
  for (int x = threadIdx.x; x < kJoinRows * (DT / 4); x += 256) {
    const int r = r0 + x / (DT / 4), d = (x % (DT / 4)) * 4;
    if (r >= nrow) break;
    float M = -INFINITY;
    for (int p = 0; p < it.nparts; ++p) M = fmaxf(M, first[p * size + kChunkRows * DT + r]);
    const float ms = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    f32x4 acc = {0, 0, 0, 0};
    for (int p = 0; p < it.nparts; ++p) {
      const float f = exp2f(first[p * size + kChunkRows * DT + r] - ms);
      L += f * first[p * size + kChunkRows * (DT + 1) + r];
      acc += f * *reinterpret_cast<const f32x4*>(first + p * size + r * DT + d);
    }
    if (d >= a.D) continue;
    const int64_t tok = sq.q0 + tile.i0 + r / a.G;
    const int head = h * a.G + r % a.G;
    store4(a, tok * a.o_ts + static_cast<int64_t>(head) * a.o_hs + d, L == 0.f ? f32x4{0, 0, 0, 0} : acc * (1.0f / L));
    if (a.lse != nullptr && d == 0) a.lse[tok * a.H + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
  }
}

}  // namespace

int chunk_slots_for(int cus) { return 2 * cus; }

int64_t chunk_workspace_bytes(int HK, int DT, int cus) {
  return static_cast<int64_t>(HK) * addr::chunk_slots_per_head(HK, chunk_slots_for(cus)) * addr::chunk_partial_floats(kChunkRows, DT) * 4;
}

// Tiles of a head at most: each sequence may end with a partial one.
static int64_t chunk_most_tiles(const PagedArgs& a) {
  const int tq = addr::chunk_tq(kChunkRows, a.G);
  return a.T / tq + std::min(a.B, a.T);
}

// Parts at most: tiles, and the split tiles' parts.
int64_t chunk_grid(const PagedArgs& a) {
  const int64_t per_head = chunk_most_tiles(a) + addr::chunk_slots_per_head(a.HK, a.chunk_slots);
  return 8 * ((per_head * a.HK + 7) / 8);
}

void launch_chunk(const PagedArgs& a, int DT, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(chunk_grid(a)));
  // split tiles at most: half the partial results, as each has two or more
  const int64_t split = std::min<int64_t>(chunk_most_tiles(a), addr::chunk_slots_per_head(a.HK, a.chunk_slots) / 2);
  const dim3 join(static_cast<unsigned>(split * (kChunkRows / kJoinRows)), static_cast<unsigned>(a.HK));
  if (DT == 64) {
    hipLaunchKernelGGL((chunk_attention_kernel<64>), grid, dim3(64 * kCWaves), 0, st, a);
    hipLaunchKernelGGL((chunk_join_kernel<64>), join, dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((chunk_attention_kernel<128>), grid, dim3(64 * kCWaves), 0, st, a);
    hipLaunchKernelGGL((chunk_join_kernel<128>), join, dim3(256), 0, st, a);
  }
}

}  // namespace gs
