// Attention over a paged key/value cache.
//
// A cache is [pages, kv heads, page rows, head dim] with any page, head and row
// stride, token t of a sequence in row t % page of page table[t / page].  Pages
// hold a multiple of 8 rows: the 8 tokens from a multiple of 8 on share a page,
// which is the granule every address is computed for.
//
// Per query row one pass over the keys it sees with the running maximum and
// total of its softmax.  Two forms: 16 rows at a time with the cache read
// straight into registers (gs_paged_rows.h), for one new token of a sequence and
// for fp32; and 128 rows at a time through LDS (gs_chunk.hip), for the sequences
// of a ragged bf16 batch that have many.
#include <algorithm>

#include "gs_paged_rows.h"

namespace gs {
namespace {

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
int paged_width(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

// Workgroups of the row form that run at a time: two to a compute unit, one at
// widths past 128.
int row_wgs_for(int D, int cus) { return paged_width(D) == 256 ? cus : 2 * cus; }

// The workspace: counters that are zero between calls, at the same place for
// every call whatever its sizes, then the partial results.
constexpr int64_t kHeadInts = GS_PAGED_HEAD_BYTES / 4;

int64_t row_partial_floats(int HK, int D, int cus) {
  return static_cast<int64_t>(HK) * addr::row_slots_per_head(HK, 2 * cus) * addr::paged_partial_floats(paged_width(D));
}

// Whether ragged calls of these sizes have a chunk form, and the rows up to
// which a sequence stays with the row form.
bool chunk_form(bool bf16, int G, int D) { return bf16 && D <= 128 && G <= kChunkRows; }
constexpr int kRowFormRows = 16;

int64_t attention_ws_bytes(bool bf16, bool ragged, int G, int HK, int D, int cus) {
  return (kHeadInts + row_partial_floats(HK, D, cus)) * 4 +
         (ragged && chunk_form(bf16, G, D) ? chunk_list_floats(HK, cus) * 4 + chunk_workspace_bytes(HK, paged_width(D), cus) : 0);
}

// Parts of the row form for each head, at most.
int64_t row_most_parts(const PagedArgs& a) {
  // one tile to a sequence where sequences of more take the chunk form
  const int64_t items = a.row_limit != INT32_MAX ? std::min(a.B, a.T)
                                                 : std::min<int64_t>(a.B, a.T) + static_cast<int64_t>(a.T) * a.G / 16;
  return addr::row_most_parts(items, a.HK, a.row_wgs);
}

// The longest sequence that a page table addresses.
int64_t paged_reach(int max_pages, int page_size) {
  return std::min<int64_t>(static_cast<int64_t>(max_pages) * page_size, (int64_t(1) << 31) - (1 << 16));
}
// The window that the kernels get: none where no sequence is longer.  They subtract it from
// positions, which are negative for rows without one: num_tokens + window fits 32 bits.
int paged_window(int window, int64_t reach) { return window < reach ? window : 0; }

// What follows from the sizes alone.
void plan_paged(PagedArgs& a, bool bf16, int cus, int max_pages, int page_size, float scale) {
  a.max_len = paged_reach(max_pages, page_size);
  a.window = paged_window(a.window, a.max_len);
  a.page_octets = static_cast<uint32_t>(page_size / 8);
  a.page_magic = addr::div_magic(a.page_octets);
  // The chunk form hides keys and takes the maximum before it scales, which is right for a
  // scale above zero only; the row form scales first.
  a.row_limit = a.cu != nullptr && chunk_form(bf16, a.G, a.D) && scale > 0.f ? kRowFormRows : INT32_MAX;
  a.chunk_slots = chunk_slots_for(cus);
  a.row_slots = addr::row_slots_per_head(a.HK, 2 * cus);
  a.row_wgs = row_wgs_for(a.D, cus);
  a.ragged_block = (cus + 7) & ~7;
  a.row_blocks = 0;
  if (a.row_limit != INT32_MAX) a.row_wgs = cus;     // beside the chunk form: half the workgroups
  a.row_parts = row_most_parts(a);
  if (a.row_limit != INT32_MAX) a.row_blocks = static_cast<int>((a.row_parts * a.HK + a.ragged_block - 1) / a.ragged_block);
  a.chunk_share = static_cast<double>(a.HK) / (2.0 * a.chunk_slots);
  a.tq.tq = std::max(1, addr::chunk_tq(kChunkRows, a.G));
  a.tq.magic = addr::div_magic(a.tq.tq);
  a.chunk_parts = a.row_limit != INT32_MAX ? chunk_most_parts(a) : 0;
  a.g_magic = addr::div_magic(a.G);
  a.scale_log2 = scale * 1.44269504088896340736f;
}

// Workgroups of the row form for each head.  Rows of a ragged batch: a sequence's tiles
// see more keys one after the other, a workgroup for each part evens that out (6 chunks of
// 151 .. 1001 rows, fp32: 133 us, 160 else).
int64_t row_grid(const PagedArgs& a) {
  return a.cu != nullptr ? a.row_parts : std::min<int64_t>(a.row_parts, std::max(1, a.row_wgs / a.HK));
}

template <bool BF16, int DT>
void launch_paged(const PagedArgs& a, int64_t n, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(n * a.HK));
  hipLaunchKernelGGL((paged_attention_kernel<BF16, DT>), grid, dim3(256), 0, st, a);
}


// The attention kernels for one width and element type.
template <bool BF16, int DT, bool E4M3>
void model_attention(PagedModel& m, const PagedArgs& a) {
  using F = PagedForm<BF16, DT, E4M3>;
  constexpr int kUnit = F::kBlock * kPWaves;
  constexpr int kVec = 16 / F::kES, kKVec = 16 / F::kCS;
  const int max_pages = static_cast<int>(a.max_len / (8 * a.page_octets));
  const int64_t page_rows = 8 * a.page_octets;
  const int64_t k_elems = extent3(a.num_pages, a.k_ps, a.HK, a.k_hs, page_rows, a.k_rs, a.D);
  const int64_t v_elems = extent3(a.num_pages, a.v_ps, a.HK, a.v_hs, page_rows, a.v_rs, a.D);
  const int64_t q_elems = extent3(a.T, a.q_ts, a.H, a.q_hs, 1, 0, a.D);
  const int64_t o_elems = extent3(a.T, a.o_ts, a.H, a.o_hs, 1, 0, a.D);
  const int64_t ks_elems = extent3(a.num_pages, a.ks_ps, a.HK, a.ks_hs, page_rows, 1, 1);
  const int64_t vs_elems = extent3(a.num_pages, a.vs_ps, a.HK, a.vs_hs, page_rows, 1, 1);
  std::vector<char> slots(static_cast<size_t>(a.row_slots), 0);
  std::vector<char>& rows = m.rows;
  int64_t U = 0;
  for (int s = 0; s < a.B; ++s) U += addr::paged_seq_units(seq_of_form<false>(a, s), a.G, a.window, kUnit);
  bool chunks = false;
  for (int s = 0; s < a.B; ++s) chunks |= seq_of_form<true>(a, s).n > 0;
  const int most = std::max(addr::row_part_units(U, a.HK, a.row_wgs), addr::row_part_least(a.row_limit != INT32_MAX, E4M3, chunks));
  const uint32_t magic = addr::div_magic(most);
  int64_t parts = 0, slot = 0;
  for (int s = 0; s < a.B && !m.bad; ++s) {
    const addr::PagedSeq sq = seq_of_form<false>(a, s);
    const int nu = addr::paged_tile_units(sq, a.G, a.window, kUnit);
    const int np = addr::row_parts(nu, most, magic);
    const int64_t nrows = static_cast<int64_t>(sq.n) * a.G;
    for (int j = 0; j < addr::paged_tiles(sq, a.G) && !m.bad; ++j) {
      const addr::PagedTile t = addr::paged_tile(sq, a.G, a.window, j);
      model_seen(m, sq, t);
      const int nblk = (t.ve - t.first + F::kBlock - 1) / F::kBlock;
      if (nblk > nu * kPWaves) m.fail("blocks past the item's units", nblk, 0, nu * kPWaves);
      const int nrow = static_cast<int>(std::min<int64_t>(16, nrows - static_cast<int64_t>(j) * 16));
      parts += np;
      if (np > 1) {
        m.in("partial results", slot, np, a.row_slots);
        m.in("counters", (a.HK - 1) * static_cast<int64_t>(a.row_slots) + slot, 1, kHeadInts);
        m.in("parts of an item", 0, np, addr::kMostParts);
        slot += np;
      }
      int covered = 0;
      for (int p = 0; p < np; ++p) {
        int w0 = 0, w1 = nu;
        if (np > 1) addr::chunk_part_range(nu, p, np, w0, w1);
        if (w0 != covered) m.fail("a unit taken other than once", w0, 1, nu);
        covered = w1;
      }
      if (covered != nu) m.fail("a unit taken other than once", covered, 1, nu);
      for (int h = 0; h < a.HK && !m.bad; ++h) {
        for (int q = 0; q < nrow; ++q) {
          const int64_t rr = static_cast<int64_t>(j) * 16 + q;
          const int64_t tok = sq.q0 + rr / a.G, head = h * a.G + rr % a.G;
          m.in("output row", tok * a.H + head, 1, static_cast<int64_t>(a.T) * a.H);
          if (m.bad) return;
          if (rows[tok * a.H + head]++) m.fail("output row written twice", tok * a.H + head, 1, static_cast<int64_t>(a.T) * a.H);
          m.in("out", tok * a.o_ts + head * a.o_hs, a.D, o_elems);
        }
        for (int l = 0; l < 64; ++l) {
          const int lq = l & 15, lg = l >> 4;
          const int64_t r = static_cast<int64_t>(j) * 16 + lq;
          const bool live = r < nrows;
          const int qi = live ? static_cast<int>(r / a.G) : t.i0;
          const int64_t qh = h * a.G + (live ? r - static_cast<int64_t>(qi) * a.G : 0);
          for (int st = 0; st < F::kSteps; ++st) {
            const int d = row_q_col<BF16, DT, E4M3>(st, lg);
            m.in("q", (sq.q0 + qi) * a.q_ts + qh * a.q_hs + (d < a.D ? d : 0), kVec, q_elems);
          }
          const int k_oct = BF16 ? 8 * (lq >> 2) : 8 * (lq >> 3), v_oct = BF16 ? 8 * lg : 8 * (lg >> 1);
          const int k_in = BF16 ? (lq & 3) : (lq & 7), v_in = BF16 ? 0 : 4 * (lg & 1);
          for (int b = 0; b < nblk + 2 * kPWaves && nblk > 0; ++b) {            // ids are read up to two rounds ahead
            const int tb = t.first + b * F::kBlock;
            uint32_t kp, kr, vp, vr;
            const int kt = addr::paged_octet(tb + k_oct, t.ve), vt = addr::paged_octet(tb + v_oct, t.ve);
            addr::div_by(static_cast<uint32_t>(kt) >> 3, a.page_octets, a.page_magic, kp, kr);
            addr::div_by(static_cast<uint32_t>(vt) >> 3, a.page_octets, a.page_magic, vp, vr);
            if (kp != static_cast<uint32_t>(kt / page_rows) || kr * 8 != static_cast<uint32_t>(kt % page_rows)) m.fail("division", kt, 0, page_rows);
            m.in("page table row", kp, 1, max_pages);
            m.in("page table row", vp, 1, max_pages);
            if (m.bad) return;
            const int64_t k_page = addr::paged_page(a.table[s * a.ld_table + kp], a.num_pages);
            const int64_t v_page = addr::paged_page(a.table[s * a.ld_table + vp], a.num_pages);
            const int64_t kb = k_page * a.k_ps + h * a.k_hs + (kr * 8 + k_in) * a.k_rs;
            const int64_t vb = v_page * a.v_ps + h * a.v_hs + (vr * 8 + v_in) * a.v_rs;
            if (E4M3) {
              m.in("k scales", k_page * a.ks_ps + h * a.ks_hs + kr * 8, 8, ks_elems);
              m.in("v scales", v_page * a.vs_ps + h * a.vs_hs + vr * 8, 8, vs_elems);
            }
            m.in("page row", kr * 8 + k_in + 4 * (F::kKT - 1), 1, page_rows);
            m.in("page row", vr * 8 + v_in + F::kKeys - 1, 1, page_rows);
            for (int u2 = 0; u2 < F::kKT; ++u2)
              for (int p = 0; p < F::kKP; ++p) {
                const int d = row_k_col<BF16, DT, E4M3>(p, lg);
                m.in("k cache", kb + 4 * u2 * a.k_rs + (d < a.D ? d : 0), kKVec, k_elems);
              }
            for (int tt = 0; tt < F::kKeys; ++tt)
              for (int n = 0; n < F::kVN; ++n) {
                const int d = n * 16 * F::kVW + F::kVW * lq;
                m.in("v cache", vb + tt * a.v_rs + (d < a.D ? d : 0), F::kVW, v_elems);
              }
          }
        }
      }
    }
  }
  const int64_t grid = a.row_parts;
  m.in("parts", 0, parts, grid);
  if (a.row_limit == INT32_MAX) return;
  // a ragged launch: every part of either form has one workgroup
  std::vector<char> row(static_cast<size_t>(parts) * a.HK, 0), pair(static_cast<size_t>(m.chunk_parts) * a.HK, 0);
  for (int64_t w = 0; w < ragged_grid(a); ++w) {
    int i;
    if (addr::ragged_role(static_cast<int>(w), a.ragged_block, a.row_blocks, i)) {
      if (i < static_cast<int64_t>(row.size())) ++row[i];
    } else {
      if (i < static_cast<int64_t>(pair.size())) ++pair[i];
    }
  }
  for (char c : row)
    if (c != 1 && !m.bad) m.fail("a row part taken other than once", 0, 1, parts);
  for (char c : pair)
    if (c != 1 && !m.bad) m.fail("a chunk part taken other than once", 0, 1, m.chunk_parts);
}

// What the chunk form's transfers leave in LDS, and what the operand reads take from it.
template <int DT, bool E4M3>
void model_chunk_lds(PagedModel& m) {
  constexpr int kWaves = 4, kRowB = DT * 2, kTileB = 64 * kRowB;
  std::vector<int> k_lds(kTileB / 16, -1), v_lds(kTileB / 16, -1);
  const auto put = [&](std::vector<int>& lds, int at, int piece) {
    m.in("stored (LDS)", at, 16, kTileB);
    if (m.bad) return;
    if (lds[at / 16] != -1) m.fail("a place stored twice", at, 16, kTileB);
    lds[at / 16] = piece;
  };
  for (int w = 0; w < kWaves; ++w)
    for (int l = 0; l < 64; ++l) {
      constexpr int kRowsPer = E4M3 ? 1024 / DT : 1024 / kRowB, kLanes = 64 / kRowsPer;
      for (int x = 0; x < 16 / kRowsPer; ++x) {
        const int in = x * kRowsPer + l / kLanes, pos = l % kLanes, row = 16 * w + in;
        if (E4M3) {                                  // 16 columns of the cache, stored as two pieces
          for (int e = 0; e < 2; ++e) {
            put(k_lds, row * kRowB + addr::chunk_k_pos(DT, in, 2 * pos + e) * 16, row * 64 + 2 * pos + e);
            put(v_lds, row * kRowB + addr::chunk_v_pos(DT, in, 2 * pos + e) * 16, row * 64 + 2 * pos + e);
          }
        } else {                                     // a transfer moves to consecutive places
          const int at = (16 * w + x * kRowsPer) * kRowB + l * 16;
          put(k_lds, at, row * 64 + addr::chunk_k_pos(DT, row, pos));
          put(v_lds, at, row * 64 + addr::chunk_v_pos(DT, row, pos));
        }
      }
    }
  for (int l = 0; l < 64; ++l) {
    const int lq = l & 31, hl = l >> 5, v_row = 4 * hl + ((l & 15) >> 2);
    for (int u = 0; u < 2; ++u)
      for (int st = 0; st < DT / 16; ++st) {
        const int at = ((lq * kRowB + addr::chunk_k_pos(DT, lq, hl) * 16) ^ (st * 32)) + u * 32 * kRowB;
        m.in("K operand (LDS)", at, 16, kTileB);
        if (k_lds[at / 16] != (32 * u + lq) * 64 + 2 * st + hl) m.fail("K operand of another piece", at, 16, kTileB);
      }
    for (int d = 0; d < DT / 32; ++d)
      for (int g = 0; g < 4; ++g)
        for (int x = 0; x < 2; ++x) {
          const int piece = 4 * d + 2 * ((l >> 4) & 1) + ((l & 3) >> 1);
          const int at = ((v_row * kRowB + addr::chunk_v_pos(DT, v_row, piece - 4 * d) * 16 + (l & 1) * 8) ^ (d * 64)) + (g * 16 + 8 * x) * kRowB;
          m.in("V operand (LDS)", at, 8, kTileB);
          if (v_lds[at / 16] != (g * 16 + 8 * x + v_row) * 64 + piece) m.fail("V operand of another piece", at, 8, kTileB);
        }
  }
}
// The chunk form.
void model_chunk(PagedModel& m, const PagedArgs& a, bool e4m3) {
  const bool wide = paged_width(a.D) == 128;
  if (e4m3) wide ? model_chunk_lds<128, true>(m) : model_chunk_lds<64, true>(m);
  else wide ? model_chunk_lds<128, false>(m) : model_chunk_lds<64, false>(m);
  const int max_pages = static_cast<int>(a.max_len / (8 * a.page_octets));
  const int64_t page_rows = 8 * a.page_octets;
  const int64_t k_elems = extent3(a.num_pages, a.k_ps, a.HK, a.k_hs, page_rows, a.k_rs, a.D);
  const int64_t v_elems = extent3(a.num_pages, a.v_ps, a.HK, a.v_hs, page_rows, a.v_rs, a.D);
  const int64_t ks_elems = extent3(a.num_pages, a.ks_ps, a.HK, a.ks_hs, page_rows, 1, 1);
  const int64_t vs_elems = extent3(a.num_pages, a.vs_ps, a.HK, a.vs_hs, page_rows, 1, 1);
  const int64_t q_elems = extent3(a.T, a.q_ts, a.H, a.q_hs, 1, 0, a.D), o_elems = extent3(a.T, a.o_ts, a.H, a.o_hs, 1, 0, a.D);
  const addr::ChunkTq& tq = a.tq;
  int64_t U2 = 0, n = 0, slots = 0, split = 0;
  for (int s = 0; s < a.B; ++s) U2 += addr::chunk_work2(seq_of_form<true>(a, s), tq, a.window);
  const int pt = addr::chunk_part_tiles(U2, a.chunk_share, kChunkLeast);
  for (int s = 0; s < a.B && !m.bad; ++s) {
    const addr::PagedSeq sq = seq_of_form<true>(a, s);
    const int nt = addr::chunk_tiles(sq, tq), np = addr::chunk_parts(sq, tq, a.window, pt, addr::div_magic(pt));
    n += static_cast<int64_t>(nt) * np;
    if (np > 1) {
      slots += static_cast<int64_t>(nt) * np;
      split += nt;
    }
    for (int j = 0; j < nt && !m.bad; ++j) {
      const addr::PagedTile t = addr::chunk_tile(sq, tq.tq, a.window, j);
      const int nkt = addr::chunk_key_tiles(t);
      model_seen(m, sq, t);
      const int nrow = (t.i1 - t.i0 + 1) * a.G;
      if (nrow < 1 || nrow > kChunkRows) m.fail("rows of a tile", 0, nrow, kChunkRows);
      for (int h = 0; h < a.HK && !m.bad; ++h) {
        for (int r = 0; r < nrow; ++r) {
          const int64_t tok = sq.q0 + t.i0 + r / a.G, head = h * a.G + r % a.G;
          m.in("output row", tok * a.H + head, 1, static_cast<int64_t>(a.T) * a.H);
          if (m.bad) return;
          if (m.rows[tok * a.H + head]++) m.fail("output row written twice", tok, 1, a.T);
          m.in("q", tok * a.q_ts + head * a.q_hs, a.D, q_elems);
          m.in("out", tok * a.o_ts + head * a.o_hs, a.D, o_elems);
        }
        for (int kt = 0; kt < nkt + 2 && nkt > 0; ++kt)       // ids are read past the last tile, too
          for (int w = 0; w < 8; ++w) {
            uint32_t pg, row;
            addr::div_by(static_cast<uint32_t>(addr::paged_octet(t.first + kt * 64 + 8 * w, t.ve)) >> 3, a.page_octets, a.page_magic, pg, row);
            m.in("page table row", pg, 1, max_pages);
            if (m.bad) return;
            if (kt >= nkt) continue;
            const int64_t page = addr::paged_page(a.table[s * a.ld_table + pg], a.num_pages);
            for (int rr = 0; rr < 8; ++rr) {
              m.in("page row", row * 8 + rr, 1, page_rows);
              m.in("k cache", page * a.k_ps + h * a.k_hs + (row * 8 + rr) * a.k_rs, a.D, k_elems);
              m.in("v cache", page * a.v_ps + h * a.v_hs + (row * 8 + rr) * a.v_rs, a.D, v_elems);
              if (e4m3) m.in("k scales", page * a.ks_ps + h * a.ks_hs + row * 8 + rr, 1, ks_elems);
              if (e4m3) m.in("v scales", page * a.vs_ps + h * a.vs_hs + row * 8 + rr, 1, vs_elems);
            }
          }
      }
    }
  }
  m.in("list of split tiles", 4, 4 * split, chunk_list_floats(a.HK, a.chunk_slots / 2));
  m.in("partial results", 0, slots, addr::chunk_slots_per_head(a.HK, a.chunk_slots));
  m.in("split tiles", 0, 2 * split, addr::chunk_slots_per_head(a.HK, a.chunk_slots));
  m.in("parts", 0, n, a.chunk_parts);
  m.chunk_parts = n;
}

// Every row of a sequence is written; the others are left to zero_outside.
void model_rows(PagedModel& m, const PagedArgs& a) {
  if (a.cu != nullptr) {
    int first, last;
    addr::paged_outside(a.cu[0], a.cu[a.B], a.T, first, last);
    for (int t = 0; t < a.T; ++t)
      for (int h = 0; h < a.H && (t < first || t >= last); ++h) {
        if (m.rows[static_cast<int64_t>(t) * a.H + h]++) m.fail("output row of no sequence written by a part", t, 1, a.T);
        m.in("out", t * a.o_ts + h * a.o_hs, a.D, extent3(a.T, a.o_ts, a.H, a.o_hs, 1, 0, a.D));
      }
    for (char c : m.rows)
      if (c != 1 && !m.bad) m.fail("output row written other than once", 0, c, 1);
  }
  for (int s = 0; s < a.B && !m.bad; ++s) {
    const addr::PagedSeq sq = a.cu != nullptr ? addr::paged_seq(a.cu[s], a.cu[s + 1], 0, a.T, 0) : addr::PagedSeq{s, 1, 0};
    for (int i = 0; i < sq.n; ++i)
      for (int h = 0; h < a.H; ++h)
        if (!m.rows[static_cast<int64_t>(sq.q0 + i) * a.H + h] && !m.bad) m.fail("output row never written", sq.q0 + i, 1, a.T);
  }
}

// Scales of a quantised cache (k NULL: it is not).
struct Scales {
  const uint8_t* k;
  int64_t k_ps, k_hs;
  const uint8_t* v;
  int64_t v_ps, v_hs;
};

int paged_attention(const char* who, bool e4m3, Scales sc, int32_t dtype, const void* q, int64_t q_ts, int64_t q_hs, const void* k_cache, int64_t k_ps,
                    int64_t k_hs, int64_t k_rs, const void* v_cache, int64_t v_ps, int64_t v_hs, int64_t v_rs,
                    int64_t num_pages, int32_t page_size, const int32_t* page_table, int64_t ld_table,
                    int32_t max_pages, const int32_t* kv_lens, const int32_t* cu_seqlens, int32_t num_seqs,
                    int64_t num_tokens, int32_t max_q, int32_t heads, int32_t kv_heads, int32_t head_dim,
                    float scale, int32_t window, void* out, int64_t o_ts, int64_t o_hs, float* lse,
                    void* workspace, int64_t workspace_bytes, void* stream) {
  GS_CHECK_ARG(dtype == GS_DTYPE_BF16 || dtype == GS_DTYPE_FP32, "%s: dtype=%d", who, dtype);
  GS_CHECK_ARG(num_tokens >= 0 && num_tokens < (int64_t(1) << 31) && num_seqs >= 0, "%s: num_tokens=%lld num_seqs=%d", who,
               (long long)num_tokens, num_seqs);
  GS_CHECK_ARG(cu_seqlens != nullptr || num_tokens == num_seqs, "%s: num_tokens=%lld of num_seqs=%d without cu_seqlens", who,
               (long long)num_tokens, num_seqs);
  GS_CHECK_ARG(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads <= 65536 && kv_heads <= 4096, "%s: heads=%d kv_heads=%d", who, heads, kv_heads);
  const bool bf16 = dtype == GS_DTYPE_BF16;
  const int ve = bf16 ? 8 : 4;
  const int de = e4m3 ? 16 : ve;                     // elements of 16 bytes of a cache row
  GS_CHECK_ARG(head_dim > 0 && head_dim <= 256 && head_dim % de == 0, "%s: head_dim=%d must be a multiple of %d up to 256", who,
               head_dim, de);
  GS_CHECK_ARG(page_size > 0 && page_size % 8 == 0, "%s: page_size=%d must be a multiple of 8", who, page_size);
  GS_CHECK_ARG(num_pages > 0 && num_pages < (int64_t(1) << 31) && max_pages >= 0 && ld_table >= max_pages,
               "%s: num_pages=%lld max_pages=%d ld_table=%lld", who, (long long)num_pages, max_pages, (long long)ld_table);
  GS_CHECK_ARG(window >= 0 && max_q >= 0, "%s: window=%d max_q=%d", who, window, max_q);
  GS_CHECK_ARG(num_tokens + paged_window(window, paged_reach(max_pages, page_size)) < (int64_t(1) << 31),
               "%s: num_tokens=%lld with window=%d past 32 bits", who, (long long)num_tokens, window);
  if (num_tokens == 0) return GS_OK;
  // the stride of a dimension of one is never used, and may be anything
  if (num_tokens == 1) q_ts = o_ts = 0;
  if (heads == 1) q_hs = o_hs = 0;
  if (kv_heads == 1) k_hs = v_hs = sc.k_hs = sc.v_hs = 0;
  if (num_pages == 1) k_ps = v_ps = sc.k_ps = sc.v_ps = 0;
  GS_CHECK_ARG(q != nullptr && k_cache != nullptr && v_cache != nullptr && out != nullptr &&
                   (num_seqs == 0 || (kv_lens != nullptr && (page_table != nullptr || max_pages == 0))) &&
                   (!e4m3 || (sc.k != nullptr && sc.v != nullptr)), "%s: null tensor", who);
  GS_CHECK_ARG(aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out) && strides_ok(q_ts, q_hs, ve) &&
                   strides_ok(k_ps, k_hs, de) && strides_ok(v_ps, v_hs, de) && strides_ok(k_rs, v_rs, de) &&
                   strides_ok(o_ts, o_hs, ve),
               "%s: q, the caches and out must be 16-byte aligned with strides that are multiples of 16 bytes", who);
  GS_CHECK_ARG(!e4m3 || (reinterpret_cast<uintptr_t>(sc.k) % 8 == 0 && reinterpret_cast<uintptr_t>(sc.v) % 8 == 0 &&
                         strides_ok(sc.k_ps, sc.k_hs, 8) && strides_ok(sc.v_ps, sc.v_hs, 8)),
               "%s: the scales must be 8-byte aligned with strides that are multiples of 8", who);
  const int cus = device_cus();
  const int64_t need = attention_ws_bytes(bf16, cu_seqlens != nullptr, heads / kv_heads, kv_heads, head_dim, cus);
  if (workspace == nullptr || workspace_bytes < need) {
    set_error("%s: workspace of %lld bytes needed (got %lld)", who, (long long)need, (long long)(workspace ? workspace_bytes : 0));
    return GS_ERR_WORKSPACE;
  }
  GS_CHECK_ARG(aligned16(workspace), "%s: workspace must be 16-byte aligned", who);
  PagedArgs a{};
  a.q = q; a.q_ts = q_ts; a.q_hs = q_hs;
  a.out = out; a.o_ts = o_ts; a.o_hs = o_hs;
  a.k = k_cache; a.k_ps = k_ps; a.k_hs = k_hs; a.k_rs = k_rs;
  a.v = v_cache; a.v_ps = v_ps; a.v_hs = v_hs; a.v_rs = v_rs;
  a.table = page_table; a.ld_table = ld_table;
  a.lens = kv_lens; a.cu = cu_seqlens; a.lse = lse;
  a.num_pages = static_cast<int>(num_pages);
  a.B = num_seqs; a.T = static_cast<int>(num_tokens);
  a.H = heads; a.HK = kv_heads; a.G = heads / kv_heads; a.D = head_dim;
  a.window = window;
  a.ks = sc.k; a.ks_ps = sc.k_ps; a.ks_hs = sc.k_hs;
  a.vs = sc.v; a.vs_ps = sc.v_ps; a.vs_hs = sc.v_hs;
  plan_paged(a, bf16, cus, max_pages, page_size, scale);
  const int DT = paged_width(head_dim);
  int* head = static_cast<int*>(workspace);
  a.row_count = head;
  a.ws = reinterpret_cast<float*>(head + kHeadInts);
  a.chunk_list = reinterpret_cast<int4*>(a.ws + row_partial_floats(kv_heads, head_dim, cus));
  a.chunk_ws = reinterpret_cast<float*>(a.chunk_list) + chunk_list_floats(kv_heads, cus);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t n = row_grid(a);
  if (a.row_limit != INT32_MAX && (max_q == 0 || static_cast<int64_t>(max_q) * a.G > a.row_limit)) {
    GS_CHECK_ARG(ragged_grid(a) < (int64_t(1) << 31), "%s: too many tiles", who);
    e4m3 ? launch_ragged_e4m3(a, DT, st) : launch_ragged(a, DT, st);
    GS_CHECK_LAUNCH(who);
    return GS_OK;
  }
  // max_q says that no sequence is the chunk form's: workgroups for such a batch, which take
  // whatever parts the lengths turn out to make
  a.row_limit = INT32_MAX;
  a.row_parts = row_most_parts(a);
  GS_CHECK_ARG(n * a.HK < (int64_t(1) << 31) && a.row_parts < (int64_t(1) << 31), "%s: too many tiles", who);
  if (e4m3) {
    launch_rows_e4m3(a, bf16, DT, n * a.HK, st);
    GS_CHECK_LAUNCH(who);
    return GS_OK;
  }
  switch (DT) {
    case 64: bf16 ? launch_paged<true, 64>(a, n, st) : launch_paged<false, 64>(a, n, st); break;
    case 128: bf16 ? launch_paged<true, 128>(a, n, st) : launch_paged<false, 128>(a, n, st); break;
    default: bf16 ? launch_paged<true, 256>(a, n, st) : launch_paged<false, 256>(a, n, st); break;
  }
  GS_CHECK_LAUNCH(who);
  return GS_OK;
}

template <int DT>
void model_width(PagedModel& m, const PagedArgs& a, bool bf16, bool e4m3) {
  if (bf16) e4m3 ? model_attention<true, DT, true>(m, a) : model_attention<true, DT, false>(m, a);
  else e4m3 ? model_attention<false, DT, true>(m, a) : model_attention<false, DT, false>(m, a);
}

int64_t check_addresses(const char* who, bool e4m3, int64_t s_ps, int64_t s_hs, int32_t dtype, int64_t q_ts, int64_t q_hs, int64_t k_ps, int64_t k_hs, int64_t k_rs,
                        int64_t v_ps, int64_t v_hs, int64_t v_rs, int64_t num_pages, int32_t page_size,
                        const int32_t* page_table, int64_t ld_table, int32_t max_pages,
                        const int32_t* kv_lens, const int32_t* cu_seqlens, int32_t num_seqs,
                        int64_t num_tokens, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t window,
                        int64_t o_ts, int64_t o_hs, int32_t cus, char* msg, int64_t msg_len,
                        int64_t* checked) {
  const bool bf16 = dtype == GS_DTYPE_BF16;
  GS_CHECK_ARG((bf16 || dtype == GS_DTYPE_FP32) && num_tokens > 0 && num_seqs >= 0 && num_tokens < (int64_t(1) << 31) &&
                   heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && head_dim > 0 && head_dim <= 256 &&
                   head_dim % (e4m3 ? 16 : bf16 ? 8 : 4) == 0 && page_size > 0 && page_size % 8 == 0 && num_pages > 0 &&
                   max_pages >= 0 && ld_table >= max_pages && (num_seqs == 0 || kv_lens != nullptr) && window >= 0 && cus > 0 &&
                   (cu_seqlens != nullptr || num_tokens == num_seqs), "%s: sizes", who);
  PagedArgs a{};
  a.q_ts = q_ts; a.q_hs = q_hs; a.o_ts = o_ts; a.o_hs = o_hs;
  a.k_ps = k_ps; a.k_hs = k_hs; a.k_rs = k_rs;
  a.v_ps = v_ps; a.v_hs = v_hs; a.v_rs = v_rs;
  a.table = page_table; a.ld_table = ld_table; a.lens = kv_lens; a.cu = cu_seqlens;
  a.num_pages = static_cast<int>(num_pages);
  a.B = num_seqs; a.T = static_cast<int>(num_tokens);
  a.H = heads; a.HK = kv_heads; a.G = heads / kv_heads; a.D = head_dim;
  a.window = window;
  static const uint8_t held = 0;
  if (e4m3) a.ks = a.vs = &held;                     // only whether there are scales
  a.ks_ps = a.vs_ps = s_ps; a.ks_hs = a.vs_hs = s_hs;
  plan_paged(a, bf16, cus, max_pages, page_size, 1.f);
  PagedModel m;
  m.window = window;
  m.rows.assign(static_cast<size_t>(a.T) * a.H, 0);
  if (a.row_limit != INT32_MAX) model_chunk(m, a, e4m3);
  switch (paged_width(head_dim)) {
    case 64: model_width<64>(m, a, bf16, e4m3); break;
    case 128: model_width<128>(m, a, bf16, e4m3); break;
    default: model_width<256>(m, a, bf16, e4m3); break;
  }
  model_rows(m, a);
  if (checked) *checked = m.checked;
  if (msg && msg_len > 0) snprintf(msg, static_cast<size_t>(msg_len), "%s", m.msg);
  return m.bad;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" {

int64_t gs_paged_attention_workspace_bytes(int32_t dtype, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t ragged) {
  if ((dtype != GS_DTYPE_BF16 && dtype != GS_DTYPE_FP32) || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 ||
      head_dim <= 0 || head_dim > 256) {
    set_error("gs_paged_attention_workspace_bytes: dtype=%d heads=%d kv_heads=%d head_dim=%d", dtype, heads, kv_heads, head_dim);
    return -GS_ERR_INVALID;
  }
  return attention_ws_bytes(dtype == GS_DTYPE_BF16, ragged != 0, heads / kv_heads, kv_heads, head_dim, device_cus());
}

int gs_paged_attention(int32_t dtype, const void* q, int64_t q_ts, int64_t q_hs, const void* k_cache, int64_t k_ps,
                       int64_t k_hs, int64_t k_rs, const void* v_cache, int64_t v_ps, int64_t v_hs, int64_t v_rs,
                       int64_t num_pages, int32_t page_size, const int32_t* page_table, int64_t ld_table,
                       int32_t max_pages, const int32_t* kv_lens, const int32_t* cu_seqlens, int32_t num_seqs,
                       int64_t num_tokens, int32_t max_q, int32_t heads, int32_t kv_heads, int32_t head_dim,
                       float scale, int32_t window, void* out, int64_t o_ts, int64_t o_hs, float* lse,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  return paged_attention("gs_paged_attention", false, Scales{}, dtype, q, q_ts, q_hs, k_cache, k_ps, k_hs, k_rs,
                         v_cache, v_ps, v_hs, v_rs, num_pages, page_size, page_table, ld_table, max_pages, kv_lens,
                         cu_seqlens, num_seqs, num_tokens, max_q, heads, kv_heads, head_dim, scale, window, out, o_ts,
                         o_hs, lse, workspace, workspace_bytes, stream);
}

int gs_paged_attention_e4m3(int32_t dtype, const void* q, int64_t q_ts, int64_t q_hs, const void* k_cache, int64_t k_ps,
                            int64_t k_hs, int64_t k_rs, const void* v_cache, int64_t v_ps, int64_t v_hs, int64_t v_rs,
                            const uint8_t* k_scales, int64_t ks_ps, int64_t ks_hs, const uint8_t* v_scales, int64_t vs_ps,
                            int64_t vs_hs,
                            int64_t num_pages, int32_t page_size, const int32_t* page_table, int64_t ld_table,
                            int32_t max_pages, const int32_t* kv_lens, const int32_t* cu_seqlens, int32_t num_seqs,
                            int64_t num_tokens, int32_t max_q, int32_t heads, int32_t kv_heads, int32_t head_dim,
                            float scale, int32_t window, void* out, int64_t o_ts, int64_t o_hs, float* lse,
                            void* workspace, int64_t workspace_bytes, void* stream) {
  return paged_attention("gs_paged_attention_e4m3", true, Scales{k_scales, ks_ps, ks_hs, v_scales, vs_ps, vs_hs},
                         dtype, q, q_ts, q_hs, k_cache, k_ps, k_hs, k_rs, v_cache, v_ps, v_hs, v_rs, num_pages,
                         page_size, page_table, ld_table, max_pages, kv_lens, cu_seqlens, num_seqs, num_tokens, max_q,
                         heads, kv_heads, head_dim, scale, window, out, o_ts, o_hs, lse, workspace, workspace_bytes,
                         stream);
}

int gs_capture_id(void* stream, int64_t* id) {
  GS_CHECK_ARG(id != nullptr, "gs_capture_id: id is null");
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long found = 0;
  const hipError_t e = hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream), &status, &found);
  if (e != hipSuccess) {
    set_error("gs_capture_id: %s", hipGetErrorString(e));
    return GS_ERR_HIP;
  }
  *id = status == hipStreamCaptureStatusActive ? static_cast<int64_t>(found) : 0;
  return GS_OK;
}

int64_t gs_check_paged_addresses(int32_t dtype, int64_t q_ts, int64_t q_hs, int64_t k_ps, int64_t k_hs, int64_t k_rs,
                                 int64_t v_ps, int64_t v_hs, int64_t v_rs, int64_t num_pages, int32_t page_size,
                                 const int32_t* page_table, int64_t ld_table, int32_t max_pages,
                                 const int32_t* kv_lens, const int32_t* cu_seqlens, int32_t num_seqs,
                                 int64_t num_tokens, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t window,
                                 int64_t o_ts, int64_t o_hs, int32_t cus, char* msg, int64_t msg_len,
                                 int64_t* checked) {
  return check_addresses("gs_check_paged_addresses", false, 0, 0, dtype, q_ts, q_hs, k_ps, k_hs, k_rs, v_ps, v_hs,
                         v_rs, num_pages, page_size, page_table, ld_table, max_pages, kv_lens, cu_seqlens, num_seqs,
                         num_tokens, heads, kv_heads, head_dim, window, o_ts, o_hs, cus, msg, msg_len, checked);
}

int64_t gs_check_paged_e4m3_addresses(int32_t dtype, int64_t q_ts, int64_t q_hs, int64_t k_ps, int64_t k_hs, int64_t k_rs,
                                      int64_t v_ps, int64_t v_hs, int64_t v_rs, int64_t s_ps, int64_t s_hs, int64_t num_pages, int32_t page_size,
                                      const int32_t* page_table, int64_t ld_table, int32_t max_pages,
                                      const int32_t* kv_lens, const int32_t* cu_seqlens, int32_t num_seqs,
                                      int64_t num_tokens, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t window,
                                      int64_t o_ts, int64_t o_hs, int32_t cus, char* msg, int64_t msg_len,
                                      int64_t* checked) {
  return check_addresses("gs_check_paged_e4m3_addresses", true, s_ps, s_hs, dtype, q_ts, q_hs, k_ps, k_hs, k_rs, v_ps,
                         v_hs, v_rs, num_pages, page_size, page_table, ld_table, max_pages, kv_lens, cu_seqlens,
                         num_seqs, num_tokens, heads, kv_heads, head_dim, window, o_ts, o_hs, cus, msg, msg_len,
                         checked);
}

}  // extern "C"
