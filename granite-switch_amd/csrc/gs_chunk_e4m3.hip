// Attention of a ragged bf16 batch over a quantised paged cache: gs_chunk.hip's form with
// keys and values that become bf16, exactly, on their way to LDS.
//
// Each wave loads its 16 keys and values of the next tile into registers before the products
// of this one, and after them makes them bf16 with their rows' scales and stores them: 32
// conversions a tile of 64 x 128 in each of the four waves, where every wave's own would be
// 128.  Scores are not summed by e4m3 products of the cache as it is, which would need none
// for the keys: the matrix units hold those sums to 2^-11 of the largest product (measured,
// 64 terms), bf16 ones to 2^-21.
//
// 8192 rows of 16 prompts (32 query, 8 key/value heads of 128): 119 .. 122 us, 540 TFLOP/s of
// the products that the mask leaves, 103 over a bf16 cache; vector instructions take 54% of the
// SIMDs' cycles and the products 25%.  A step of 48 decode rows and 16 chunks of 256 over up to
// 3839 keys: 92 us.  8 chunks of 3 .. 64 rows over up to 16384 keys: 58 us, where a part's
// start (its schedule, its first tile) is a sixth of its time and the join 7.
#include "gs_chunk.h"

namespace gs {
namespace {

// One part: 128 rows of a sequence and head h over its key tiles.
template <int DT>
__device__ __forceinline__ void chunk_part_e4m3(const PagedArgs& a, const ChunkItem& it, int h, char* lds) {
  constexpr int kRowB = DT * 2;                     // bytes of a key row in LDS
  constexpr int kTileB = kCKeys * kRowB;            // of a stage's keys, and of its values
  constexpr int kStageB = 2 * kTileB;
  constexpr int kRowsPer = 1024 / DT;               // rows of the cache that 16 bytes a lane are
  constexpr int kMoves = 16 / kRowsPer;             // loads for the wave's 16 keys (as many for the values)
  constexpr int kSteps = DT / 16;

  const int tid = threadIdx.x, l = tid & 63;
  const int lq = l & 31, hl = l >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const ChunkRow w = chunk_row(a, it, h);
  const addr::PagedTile& tile = w.tile;
  u32x4 qf[kSteps];
  chunk_queries<DT>(a, w, qf);

  // ---- transfers ------------------------------------------------------------------
  const int32_t* trow = a.table + static_cast<int64_t>(it.s) * a.ld_table;
  const int t_row = l / (64 / kRowsPer), t_pos = l % (64 / kRowsPer);   // the lane's row and 16 columns in a load
  const char* k_head = static_cast<const char*>(a.k) + static_cast<int64_t>(h) * a.k_hs;
  const char* v_head = static_cast<const char*>(a.v) + static_cast<int64_t>(h) * a.v_hs;
  const uint8_t* ks_head = a.ks + static_cast<int64_t>(h) * a.ks_hs;
  const uint8_t* vs_head = a.vs + static_cast<int64_t>(h) * a.vs_hs;
  // Lanes 2 i and 2 i + 1 hold where the wave's 16 keys of tile i of 32 are (its first 8 and
  // its last 8): page and first row.
  int id_page = 0, id_row = 0;
  const auto load_ids = [&](int kt) {
    uint32_t pg, row8;
    const int oct = addr::paged_octet(tile.first + (kt + (l >> 1)) * kCKeys + 16 * wave + 8 * (l & 1), tile.ve);
    addr::div_by(static_cast<uint32_t>(oct) >> 3, a.page_octets, a.page_magic, pg, row8);
    id_page = addr::paged_page(trow[pg], a.num_pages);
    id_row = static_cast<int>(row8 * 8);
  };
  // a lane's places in the 8 rows of a page that it loads from
  const int in8 = t_row & 7, col = t_pos * 16 < a.D ? t_pos * 16 : 0;
  const int64_t k_lane = in8 * a.k_rs + col, v_lane = in8 * a.v_rs + col;
  u32x4 k_raw[kMoves], v_raw[kMoves];
  uint32_t k_scale[kMoves], v_scale[kMoves];
  const auto issue = [&](int kt) {
    const int i32 = (kt - w.kt0) & 31;
    if (i32 == 0) load_ids(kt);
    const char* kb[2];
    const char* vb[2];
    const uint8_t* ksb[2];
    const uint8_t* vsb[2];
#pragma unroll
    for (int oc = 0; oc < 2; ++oc) {                   // uniform: the first row of 8
      const int64_t page = __builtin_amdgcn_readlane(id_page, 2 * i32 + oc);
      const int row = __builtin_amdgcn_readlane(id_row, 2 * i32 + oc);
      kb[oc] = k_head + page * a.k_ps + row * a.k_rs;
      vb[oc] = v_head + page * a.v_ps + row * a.v_rs;
      ksb[oc] = ks_head + page * a.ks_ps + row;
      vsb[oc] = vs_head + page * a.vs_ps + row;
    }
#pragma unroll
    for (int x = 0; x < kMoves; ++x) {
      const bool second = kMoves == 2 ? x == 1 : t_row >= 8;
      k_raw[x] = ld16((second ? kb[1] : kb[0]) + k_lane);
      v_raw[x] = ld16((second ? vb[1] : vb[0]) + v_lane);
      k_scale[x] = (second ? ksb[1] : ksb[0])[in8];
      v_scale[x] = (second ? vsb[1] : vsb[0])[in8];
    }
  };
  // What `issue` loaded into LDS.  Values that no query of the tile sees are zero: the cache
  // may hold anything there, and 0 * NaN is not 0.
  const auto land = [&](int kt, int stage) {
#pragma unroll
    for (int x = 0; x < kMoves; ++x) {
      const int row = x * kRowsPer + t_row;          // of the wave's 16
      const int t = tile.first + kt * kCKeys + 16 * wave + row;
      const bool seen = t >= tile.vs && t < tile.ve, cols = t_pos * 16 < a.D;
      char* to = lds + stage * kStageB + (16 * wave + row) * kRowB;
      const auto put = [&](u32x4 raw, float f, char* to0, char* to1) {
        u32x4 y[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i >> 1][2 * (i & 1)] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[i], f, false));
          y[i >> 1][2 * (i & 1) + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[i], f, true));
        }
        st16(to0, y[0]);
        st16(to1, y[1]);
      };
      put(sel16(cols, k_raw[x]), cols ? __uint_as_float(k_scale[x] << 23) : 1.f, to + addr::chunk_k_pos(DT, row, 2 * t_pos) * 16,
          to + addr::chunk_k_pos(DT, row, 2 * t_pos + 1) * 16);
      // odd rows store their second piece first: neighbours' rows are on different banks
      const u32x4 vr = v_raw[x];
      const bool odd = (row & 1) != 0;
      put(sel16(seen && cols, odd ? u32x4{vr[2], vr[3], vr[0], vr[1]} : vr), seen ? __uint_as_float(v_scale[x] << 23) : 1.f,
          to + kTileB + addr::chunk_v_pos(DT, row, 2 * t_pos + (row & 1)) * 16,
          to + kTileB + addr::chunk_v_pos(DT, row, 2 * t_pos + 1 - (row & 1)) * 16);
    }
  };

  ChunkSums<DT> sum;
  sum.clear();

  // LDS address of the lane's operand rows of K, as chunk_v_at.
  const uint32_t k_at = lq * kRowB + addr::chunk_k_pos(DT, lq, hl) * 16, v_at = kTileB + chunk_v_at<DT>();

  // Tile kt, in `stage`; `next` tells whether tile kt + 1 goes to the other one.
  const auto compute = [&](int kt, int stage, bool next) {
    const int tb = tile.first + kt * kCKeys;
    const bool active = w.wave_live && tb < w.any_hi && tb + kCKeys > w.any_lo;
    if (next) issue(kt + 1);
    if (active) {
      f32x16 sc[2];
      chunk_scores<DT>(qf, lds, k_at + stage * kStageB, sc);
      chunk_values<DT>(a, w, tb, sc, lds, v_at + stage * kStageB, sum);
    }
    if (next) land(kt + 1, stage ^ 1);               // the stage of tile kt - 1, which every wave is past
  };

  // ---- the walk over the keys ---------------------------------------------------
  const int n = w.kt1 - w.kt0;
  if (n > 0) {
    issue(w.kt0);
    land(w.kt0, 0);
    int stage = 0;
    for (int i = 0; i < n; ++i) {
      lds_barrier();                                 // the tile is stored, and the other stage read
      compute(w.kt0 + i, stage, i + 1 < n);
      stage ^= 1;
    }
  }
  chunk_results<DT>(a, it, h, w, sum);
}

template <int DT>
__global__ __launch_bounds__(64 * kCWaves, 2) void ragged_attention_e4m3_kernel(PagedArgs) {
  __shared__ __attribute__((aligned(1024))) char lds[addr::cmax(kCStages * 2 * kCKeys * DT * 2, static_cast<int>(sizeof(RowShared<DT>)))];
  ragged_work<DT, true>(lds, [&](const PagedArgs& a, const ChunkItem& it, int h) { chunk_part_e4m3<DT>(a, it, h, lds); });
}

}  // namespace

void launch_ragged_e4m3(const PagedArgs& a, int DT, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(ragged_grid(a)));
  // a workgroup for an eighth of a tile up to 2 chunk_slots of them: with one chunk_slots the
  // invocation chunks' join took some workgroups two turns (59.7 us for the call, 57.7 so; the
  // bf16 cache's calls show no difference)
  const dim3 join(static_cast<unsigned>(2 * a.chunk_slots));
  if (DT == 64) {
    hipLaunchKernelGGL((ragged_attention_e4m3_kernel<64>), grid, dim3(64 * kCWaves), 0, st, a);
    hipLaunchKernelGGL((chunk_join_kernel<64>), join, dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((ragged_attention_e4m3_kernel<128>), grid, dim3(64 * kCWaves), 0, st, a);
    hipLaunchKernelGGL((chunk_join_kernel<128>), join, dim3(256), 0, st, a);
  }
}

}  // namespace gs
