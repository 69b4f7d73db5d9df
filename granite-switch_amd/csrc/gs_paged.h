// What the kernels over a paged cache share (gs_paged.hip, gs_chunk.hip).
#pragma once

#include <algorithm>
#include <vector>

#include "gs_addr.h"
#include "gs_common.h"

namespace gs {

struct PagedArgs {
  const void* q;
  int64_t q_ts, q_hs;               // token and head strides, elements
  void* out;
  int64_t o_ts, o_hs;
  const void* k;
  int64_t k_ps, k_hs, k_rs;         // page, head and row strides
  const void* v;
  int64_t v_ps, v_hs, v_rs;
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lens;
  const int32_t* cu;
  float* lse;                       // [T, H] or NULL
  float* ws;                        // row form: partial results
  float* chunk_ws;                  // chunk form: partial results
  int4* chunk_list;                 // the split tiles: their number, then first query, rows, parts and first partial result of each
  int* row_count;                   // by an item's first partial result: its workgroups that are done; zero between calls
  int64_t max_len;
  uint32_t page_octets, page_magic;
  int num_pages;
  int B, T, H, HK, G, D;
  int window;
  int row_wgs;                      // workgroups that the row form fills
  int64_t row_parts;                // its parts for each head, at most
  int row_slots;                    // its partial results for each head
  int row_limit;                    // sequences of at most so many rows take the row form, others the chunk form
  int64_t chunk_parts;              // chunk form: parts for each head, at most
  int chunk_slots;                  // workgroups that the chunk form fills
  int ragged_block, row_blocks;     // a ragged launch's order (addr::ragged_role)
  double chunk_share;               // HK / (2 chunk_slots)
  addr::ChunkTq tq;                 // queries of a chunk tile
  uint32_t g_magic;                 // div_magic(G)
  float scale_log2;
  const uint8_t* ks;                // scales of a quantised cache, page and head strides
  const uint8_t* vs;
  int64_t ks_ps, ks_hs, vs_ps, vs_hs;
};

__device__ __host__ __forceinline__ addr::PagedSeq any_seq(const PagedArgs& a, int s) {
  return a.cu != nullptr ? addr::paged_seq(a.cu[s], a.cu[s + 1], a.lens[s], a.T, a.max_len)
                         : addr::paged_seq(s, s + 1, a.lens[s], a.T, a.max_len);
}
// A sequence as a form sees it: the row form has those of at most row_limit rows,
// the chunk form the others.
template <bool CHUNK>
__device__ __host__ __forceinline__ addr::PagedSeq only_form(const PagedArgs& a, addr::PagedSeq q) {
  const bool few = static_cast<int64_t>(q.n) * a.G <= a.row_limit;
  if (few == CHUNK) q.n = 0;
  return q;
}
template <bool CHUNK>
__device__ __host__ __forceinline__ addr::PagedSeq seq_of_form(const PagedArgs& a, int s) {
  return only_form<CHUNK>(a, any_seq(a, s));
}

// The kernel's only argument, to be loaded where it is used: a kernel of several
// forms would keep all its fields in registers throughout.
__device__ __forceinline__ const PagedArgs& fresh_args() {
  typedef const __attribute__((address_space(4))) PagedArgs* Ptr;
  Ptr p = (Ptr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const PagedArgs*)(p);
}

// Ragged bf16 batches, head widths up to 128 (gs_chunk.hip).
constexpr int kChunkRows = 128;
constexpr int kChunkLeast = 4;      // key tiles of a part, at least
int chunk_slots_for(int cus);
int64_t chunk_list_floats(int HK, int cus);
int64_t chunk_workspace_bytes(int HK, int DT, int cus);
int64_t chunk_most_parts(const PagedArgs& a);
int64_t ragged_grid(const PagedArgs& a);
void launch_ragged(const PagedArgs& a, int DT, hipStream_t st);
void launch_ragged_e4m3(const PagedArgs& a, int DT, hipStream_t st);   // over a quantised cache (gs_chunk_e4m3.hip)
// The row form over a quantised cache (gs_paged_e4m3.hip), on that many workgroups.
void launch_rows_e4m3(const PagedArgs& a, bool bf16, int DT, int64_t workgroups, hipStream_t st);

// Strides that keep rows on 16-byte boundaries.
inline bool strides_ok(int64_t a, int64_t b, int n) { return a >= 0 && b >= 0 && a % n == 0 && b % n == 0; }

// ---------------------------------------------------------------------------
// Address model: the kernels' global accesses for given tables, replayed with
// the kernels' own arithmetic.
// ---------------------------------------------------------------------------
struct PagedModel {
  int64_t bad = 0, checked = 0, chunk_parts = 0;
  int window = 0;                                   // as the caller gave it
  std::vector<char> rows;                           // output rows written
  char msg[256] = "";
  void fail(const char* what, int64_t at, int64_t n, int64_t cap) {
    if (bad++ == 0) snprintf(msg, sizeof(msg), "%s: elements [%lld, %lld) of %lld", what, (long long)at, (long long)(at + n), (long long)cap);
  }
  void in(const char* what, int64_t at, int64_t n, int64_t cap) {
    ++checked;
    if (at < 0 || at + n > cap) fail(what, at, n, cap);
  }
};
// What the rows of a tile see, from the definition in 64 bits, against what the kernels take
// it for: every key that a row sees is among the tile's, none from before or past those.
inline void model_seen(PagedModel& m, const addr::PagedSeq& sq, const addr::PagedTile& t) {
  int64_t vs = INT64_MAX, ve = 0;
  for (int qi = t.i0; qi <= t.i1; ++qi) {
    const int64_t hi = static_cast<int64_t>(sq.len) - sq.n + qi + 1, lo = std::max<int64_t>(0, m.window > 0 ? hi - m.window : 0);
    if (hi <= lo) continue;
    vs = std::min(vs, lo);
    ve = hi;
  }
  if (ve == 0 ? t.ve != t.vs : t.vs != vs || t.ve != ve) m.fail("keys that a tile's rows see", t.vs, t.ve - t.vs, ve);
}
inline int64_t extent3(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t cols) {
  return (n0 - 1) * s0 + (n1 - 1) * s1 + (n2 - 1) * s2 + cols;
}

}  // namespace gs
