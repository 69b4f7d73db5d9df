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

#include "gs_chunk.h"

namespace gs {
namespace {

// One part: 128 rows of a sequence and head h over its key tiles.
template <int DT>
__device__ __forceinline__ void chunk_part(const PagedArgs& a, const ChunkItem& it, int h, char* lds) {
  constexpr int kRowB = DT * 2;                     // bytes of a key row in LDS
  constexpr int kTileB = kCKeys * kRowB;            // of a stage's keys, and of its values
  constexpr int kStageB = 2 * kTileB;
  constexpr int kRowsPer = 1024 / kRowB;            // rows a wave transfer moves
  constexpr int kMoves = 8 / kRowsPer;              // transfers for 8 keys (as many for the values); a wave moves 16 keys
  constexpr int kSteps = DT / 16;

  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63;
  const int lq = l & 31, hl = l >> 5;
  const int s = it.s;
  const ChunkRow w = chunk_row(a, it, h);
  const addr::PagedTile& tile = w.tile;
  u32x4 qf[kSteps];
  chunk_queries<DT>(a, w, qf);

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
    const int i32 = (kt - w.kt0) & 31;
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

  ChunkSums<DT> sum;
  sum.clear();

  // LDS address of the lane's operand rows of K, as chunk_v_at.
  const uint32_t k_at = lq * kRowB + addr::chunk_k_pos(DT, lq, hl) * 16, v_at = kTileB + chunk_v_at<DT>();

  // Tile kt, in `stage`; `next` tells whether tile kt + 1 is moved to the other one.
  const auto compute = [&](int kt, int stage, bool next) {
    const int tb = tile.first + kt * kCKeys;
    const bool active = w.wave_live && tb < w.any_hi && tb + kCKeys > w.any_lo;
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
    chunk_values<DT>(a, w, tb, sc, lds, v_at + stage * kStageB, sum);
  };

  // ---- the walk over the keys ---------------------------------------------------
  const int n = w.kt1 - w.kt0;
  if (n > 0) {
    issue(w.kt0, 0);
    int stage = 0;
    for (int i = 0; i < n; ++i) {
      mem_fence_compiler();
      __builtin_amdgcn_s_waitcnt(wait_vm_lds0(0));                 // own transfers landed, own reads done
      __builtin_amdgcn_s_barrier();
      mem_fence_compiler();
      compute(w.kt0 + i, stage, i + 1 < n);
      stage ^= 1;
    }
  }
  chunk_results<DT>(a, it, h, w, sum);
}

template <int DT>
__global__ __launch_bounds__(64 * kCWaves, 2) void ragged_attention_kernel(PagedArgs) {
  __shared__ __attribute__((aligned(1024))) char lds[addr::cmax(kCStages * 2 * kCKeys * DT * 2, static_cast<int>(sizeof(RowShared<DT>)))];
  ragged_work<DT, false>(lds, [&](const PagedArgs& a, const ChunkItem& it, int h) { chunk_part<DT>(a, it, h, lds); });
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
