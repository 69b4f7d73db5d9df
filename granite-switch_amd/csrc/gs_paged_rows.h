// The row form of attention over a paged cache: 16 (query, head) rows at a time,
// keys and values from the pages straight into registers.  Shared by the decode
// kernel (gs_paged.hip) and the kernel for ragged batches (gs_chunk.hip).
//
// An item is a tile of 16 rows of a sequence for one key/value head, a run of units
// of 128 keys (fp32: 64).  An item of more units than a workgroup's equal share is cut
// into parts.  A part leaves a partial result; the last of an item's workgroups to be
// done joins them, in the order of the keys.
//
// The memory rate bounds it: 2 G operations a byte of the cache (G query heads to a
// key/value head).  256 sequences of 16 .. 2047 keys, 8 key/value heads of 128, bf16:
// 109 us, 4.8 TB/s; one of 131071 keys: 105 us, 5.1 TB/s; a bare read reaches 6.8.  The
// longest parts start first: 112 us against 118 for the 256 sequences.  Equal runs of the
// batch's units, cut wherever they end, cost two joins a workgroup and took 114.
#pragma once

#include <type_traits>

#include "gs_paged.h"

namespace gs {
namespace {

// What the two element types differ in.  Both use 16 x 16 products: S^T = K Q^T
// with the keys as rows, so a lane has one query row's scores of consecutive
// keys, which is the operand that O^T = V^T P^T takes them as.  A quantised cache's
// rows (E4M3) become bf16 or fp32 operands in registers: a lane's 16 bytes of a key are
// 16 columns, so its query columns are the same ones.
template <bool BF16, int DT, bool E4M3 = false>
struct PagedForm;
template <int DT, bool E4M3>
struct PagedForm<true, DT, E4M3> {
  static constexpr int kBlock = 32;                 // keys of a wave's block
  static constexpr int kSteps = DT / 32;            // query pieces of 16 bytes per row and lane
  static constexpr int kKP = E4M3 ? DT / 64 : kSteps;   // K pieces of 16 bytes per key row and lane
  static constexpr int kKT = 2;                     // 16-key tiles of S^T in a block
  static constexpr int kVW = E4M3 && DT == 256 ? 16 : DT >= 128 ? 8 : 4;   // columns of a V vector
  static constexpr int kVN = DT / (16 * kVW);       // V vectors of a lane and key
  static constexpr int kKeys = 8;                   // keys of a lane: 8 g .. 8 g + 7
  static constexpr int kES = 2;
  static constexpr int kCS = E4M3 ? 1 : 2;          // bytes of a cache's element
};
template <int DT, bool E4M3>
struct PagedForm<false, DT, E4M3> {
  static constexpr int kBlock = 16;
  static constexpr int kSteps = DT / 16;
  static constexpr int kKP = E4M3 ? DT / 64 : kSteps;
  static constexpr int kKT = 1;
  static constexpr int kVW = E4M3 && DT >= 128 ? 8 : 4;
  static constexpr int kVN = DT / (16 * kVW);
  static constexpr int kKeys = 4;                   // keys 4 g .. 4 g + 3
  static constexpr int kES = 4;
  static constexpr int kCS = E4M3 ? 1 : 4;
};
// First column of query piece st of lane group lg, and of its K piece kp.
template <bool BF16, int DT, bool E4M3>
__device__ __host__ __forceinline__ int row_q_col(int st, int lg) {
  constexpr int kVec = BF16 ? 8 : 4;
  constexpr int kPer = E4M3 ? 16 / kVec : 1;        // query pieces of a K piece
  return kVec * (kPer * (4 * (st / kPer) + lg) + st % kPer);
}
template <bool BF16, int DT, bool E4M3>
__device__ __host__ __forceinline__ int row_k_col(int kp, int lg) {
  return (E4M3 ? 16 : BF16 ? 8 : 4) * (4 * kp + lg);
}

__device__ __forceinline__ f32x4 mfma16_bf16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16_f32(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
// Half h (0 low, 1 high) of two dwords, side by side.
__device__ __forceinline__ uint32_t pair16(uint32_t lo, uint32_t hi, int h) {
  return __builtin_amdgcn_perm(hi, lo, h ? 0x07060302u : 0x05040100u);
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int BYTES>
struct VVec;
template <>
struct VVec<16> {
  typedef u32x4 T;
};
template <>
struct VVec<8> {
  typedef u32x2 T;
};
template <>
struct VVec<4> {
  typedef uint32_t T __attribute__((ext_vector_type(1)));
};

// The power of two of byte `at` of a word of scales; for code 0 a float without exponent, which
// conversions take for 2^-127 and products for 0.
__device__ __forceinline__ float scale_of(uint32_t w, int at) { return __uint_as_float(((w >> (8 * at)) & 255u) << 23); }
// The bytes of four scales that are less than 2^-63, as ones: those below 64.
__device__ __forceinline__ uint32_t tiny_bytes(uint32_t w) {
  const uint32_t t = ~(w | (w << 1)) & 0x80808080u;  // neither of a byte's upper two bits
  return (t - (t >> 7)) | t;
}

// One 32-key (16-key, fp32) block's keys and values in a wave's registers.
struct NoScales {};
struct BlockScales {
  u32x2 k, v;                                       // of the 8 keys of the lane's K rows; of its V rows
};
template <bool BF16, int DT, bool E4M3 = false>
struct PagedBlock {
  using F = PagedForm<BF16, DT, E4M3>;
  u32x4 k[F::kKT][F::kKP];
  typename VVec<F::kVW * F::kCS>::T v[F::kKeys][F::kVN];
  std::conditional_t<E4M3, BlockScales, NoScales> s;
};

constexpr int kPWaves = 4;

template <int DT>
struct RowShared {
  float o[kPWaves][16][DT + 4];
  float m[kPWaves][16], l[kPWaves][16];
  float red[256][5];
  int last;
};

// ---------------------------------------------------------------------------
// Which part is whose: every wave works the batch's schedule out for itself, a lane
// per sequence, without LDS or a barrier (through them it took 4 us of a workgroup's
// start).
// ---------------------------------------------------------------------------
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_from(uint64_t x) {
  const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(x)), CTRL, ROWS, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(x >> 32)), CTRL, ROWS, 0xf, false);
  return static_cast<uint32_t>(lo) | (static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32);
}
// Sums over the lanes up to each: within rows of 16 from 1, 2, 4 and 8 lanes before,
// then from the last lanes of the rows before.
__device__ __forceinline__ uint64_t lane_sums(uint64_t x) {
  x += dpp_from<0x111, 0xf>(x);
  x += dpp_from<0x112, 0xf>(x);
  x += dpp_from<0x114, 0xf>(x);
  x += dpp_from<0x118, 0xf>(x);
  x += dpp_from<0x142, 0xa>(x);
  x += dpp_from<0x143, 0xc>(x);
  return x;
}
// The largest of the lanes' values, none below zero.
__device__ __forceinline__ int lanes_most(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ uint64_t of_lane(uint64_t x, int l) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(x), l);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(x >> 32), l);
  return lo | (static_cast<uint64_t>(hi) << 32);
}

// The batch's sequences, 256 at a time: lane l has s = base + 64 i + l.
struct Batch4 {
  int base;
  addr::PagedSeq sq[4];
};
__device__ __forceinline__ void load_batch(const PagedArgs& a, Batch4& q, int base) {
  q.base = base;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int s = base + 64 * i + lane_id();
    q.sq[i] = addr::PagedSeq{0, 0, 0};
    if (s < a.B) q.sq[i] = any_seq(a, s);
  }
}
// f(s, sequence) for each of the lane's sequences that a form has rows of, in order.
template <bool CHUNK, class F>
__device__ __forceinline__ void each_seq(const PagedArgs& a, Batch4& q, const F& f) {
  for (int base = 0; base < a.B; base += 256) {
    if (base != q.base) load_batch(a, q, base);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (base + 64 * i >= a.B) break;
      const addr::PagedSeq sq = only_form<CHUNK>(a, q.sq[i]);
      if (sq.n > 0) f(base + 64 * i + lane_id(), sq);
    }
  }
}

// Places of the parts in the order of their classes (0 first), within a class by lane:
// eight 16-bit counts in two words, or one class where there are more parts.
struct ClassOrder {
  uint64_t lo, hi;                   // counts of the lane's parts; then their places
  bool one;
  __device__ __forceinline__ void add(int cls, int parts) {
    const uint64_t x = static_cast<uint64_t>(parts) << (one ? 0 : 16 * (cls & 3));
    if (one || cls < 4) {
      lo += x;
    } else {
      hi += x;
    }
  }
  // counts to places; the number of parts
  __device__ __forceinline__ int place() {
    const uint64_t lo_to = lane_sums(lo), hi_to = lane_sums(hi);
    const uint64_t lo_all = of_lane(lo_to, 63), hi_all = of_lane(hi_to, 63);
    if (one) {
      lo = lo_to - lo;
      return static_cast<int>(lo_all);
    }
    constexpr uint64_t kOnes = 0x0001000100010001;   // times it: the fields up to each, added
    const uint64_t lo_cls = lo_all * kOnes, hi_cls = hi_all * kOnes + (lo_cls >> 48) * kOnes;
    lo = lo_cls - lo_all + lo_to - lo;
    hi = hi_cls - hi_all + hi_to - hi;
    return static_cast<int>(hi_cls >> 48);
  }
  // the place of the lane's next parts of a class
  __device__ __forceinline__ int next(int cls, int parts) {
    const int sh = 16 * (cls & 3);
    const int at = one ? static_cast<int>(lo) : static_cast<int>(((cls < 4 ? lo : hi) >> sh) & 65535);
    add(cls, parts);
    return at;
  }
};

// One part of the row form's work.
struct RowItem {
  int s, j, part, nparts, slot;      // slot: of the item's first partial result, or -1
  int units;                         // of the item
  addr::PagedSeq sq;
};

// A part as list_parts leaves it: its place among its sequence's from the last, and that
// sequence's parts to a tile, first partial result and units to a tile.
struct RowEntry {
  int s, x, np, slot, units, q0, n, len;
};
__device__ __forceinline__ RowItem row_item(const RowEntry& e) {
  const auto u = [](int x) { return __builtin_amdgcn_readfirstlane(x); };   // uniform, and known to be
  const int np = u(e.np), x = u(e.x), j = np > 1 ? x / np : x;
  return RowItem{u(e.s), j, x - j * np, np, np > 1 ? u(e.slot) + j * np : -1, u(e.units), {u(e.q0), u(e.n), u(e.len)}};
}

// The row form's parts for one head, in eight classes of length, the longest first;
// within one by lane.
template <bool BF16, int DT>
struct RowOrder {
  static constexpr int kUnit = PagedForm<BF16, DT>::kBlock * kPWaves;
  Batch4 q;
  int most;                          // units of a part
  uint32_t magic;
  ClassOrder order;
  int slots;                         // partial results before the lane's
  int total;

  struct Count {
    int nt, nu, np, cls;
  };
  __device__ __forceinline__ Count count(const PagedArgs& a, const addr::PagedSeq& sq) const {
    Count c;
    c.nt = addr::paged_tiles(sq, a.G);
    c.nu = addr::paged_tile_units(sq, a.G, a.window, kUnit);
    c.np = addr::row_parts(c.nu, most, magic);
    uint32_t x, rest;
    addr::div_by(static_cast<uint32_t>(8 * (most - (c.np > 1 ? most : c.nu))), static_cast<uint32_t>(most), magic, x, rest);
    c.cls = min(static_cast<int>(x), 7);
    return c;
  }
  __device__ __forceinline__ void plan(const PagedArgs& a) {
    load_batch(a, q, 0);
    uint64_t U = 0;
    each_seq<false>(a, q, [&](int, const addr::PagedSeq& sq) { U += addr::paged_seq_units(sq, a.G, a.window, kUnit); });
    most = addr::row_part_units(static_cast<int64_t>(of_lane(lane_sums(U), 63)), a.HK, a.row_wgs);
    const bool ragged = a.row_limit != INT32_MAX;
    bool chunks = false;
    if (ragged && a.ks != nullptr) each_seq<true>(a, q, [&](int, const addr::PagedSeq&) { chunks = true; });
    most = max(most, addr::row_part_least(ragged, a.ks != nullptr, __any(chunks)));
    magic = addr::div_magic(most);
    order = ClassOrder{0, 0, a.row_parts >= 65536};
    uint64_t sl = 0;
    each_seq<false>(a, q, [&](int, const addr::PagedSeq& sq) {
      const Count c = count(a, sq);
      order.add(c.cls, c.nt * c.np);
      sl += c.np > 1 ? c.nt * c.np : 0;
    });
    slots = static_cast<int>(lane_sums(sl) - sl);
    total = order.place();
  }
  // Parts k n + i (k even) or k n + n - 1 - i (k odd) for k in [k0, k1), into list[k - k0],
  // in one pass over the batch.
  __device__ __forceinline__ void list_parts(const PagedArgs& a, int i, int n, int k0, int k1, RowEntry* list) const {
    ClassOrder o = order;
    int sl = slots;
    Batch4 seqs = q;
    const uint32_t n_magic = addr::div_magic(n);
    each_seq<false>(a, seqs, [&](int s, const addr::PagedSeq& sq) {
      const Count c = count(a, sq);
      const int m = c.nt * c.np, at = o.next(c.cls, m);
      uint32_t k, rest;
      addr::div_by(static_cast<uint32_t>(at), static_cast<uint32_t>(n), n_magic, k, rest);
      for (int kk = max(static_cast<int>(k), k0); kk < k1 && kk * n < at + m; ++kk) {
        const int x = kk * n + ((kk & 1) != 0 ? n - 1 - i : i) - at;
        if (x >= 0 && x < m) list[kk - k0] = RowEntry{s, m - 1 - x, c.np, sl, c.nu, sq.q0, sq.n, sq.len};   // the last tiles first
      }
      sl += c.np > 1 ? m : 0;
    });
  }
  // The r-th part (0 <= r < total).
  __device__ __forceinline__ RowItem part(const PagedArgs& a, int r) {
    ClassOrder o = order;
    int sl = slots, at = 0;
    RowItem it{-1, 0, 0, 1, -1, 0, {0, 0, 0}};
    each_seq<false>(a, q, [&](int s, const addr::PagedSeq& sq) {
      const Count c = count(a, sq);
      const int x = r - o.next(c.cls, c.nt * c.np);
      if (x >= 0 && x < c.nt * c.np) {
        it.s = s;
        at = c.nt * c.np - 1 - x;                    // a sequence's last tiles, the longest, first
        it.nparts = c.np;
        it.slot = sl;
        it.units = c.nu;
        it.sq = sq;
      }
      sl += c.np > 1 ? c.nt * c.np : 0;
    });
    const int from = __builtin_ctzll(__ballot(it.s >= 0));
    const auto u = [&](int x) { return __builtin_amdgcn_readlane(x, from); };   // uniform, and known to be
    const int np = u(it.nparts), x = u(at), j = np > 1 ? x / np : x;
    return RowItem{u(it.s), j, x - j * np, np, np > 1 ? u(it.slot) + j * np : -1, u(it.units), {u(it.sq.q0), u(it.sq.n), u(it.sq.len)}};
  }
};

// A row of the result from its sums.
template <bool BF16>
__device__ __forceinline__ void row_store(const PagedArgs& a, int64_t tok, int head, int d, f32x4 acc, float M, float L) {
  if (d >= a.D) return;
  const f32x4 x = L == 0.f ? f32x4{0, 0, 0, 0} : acc * (1.0f / L);
  const int64_t e = tok * a.o_ts + static_cast<int64_t>(head) * a.o_hs + d;
  if constexpr (BF16) {
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + e) = u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
  } else {
    *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + e) = x;
  }
  if (a.lse != nullptr && d == 0)
    a.lse[tok * a.H + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

// Rows of a ragged batch that are in no sequence get zeros, 16 bytes a thread, dealt out
// over a launch's workgroups.
template <bool BF16>
__device__ __forceinline__ void zero_outside(const PagedArgs& a) {
  if (a.cu == nullptr) return;
  int first, last;
  addr::paged_outside(a.cu[0], a.cu[a.B], a.T, first, last);
  constexpr int kVec = BF16 ? 8 : 4;
  const int pieces = a.D / kVec;
  const int64_t row = static_cast<int64_t>(a.H) * pieces, n = (first + static_cast<int64_t>(a.T - last)) * row;
  for (int64_t x = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; x < n; x += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t i = x / row, t = i < first ? i : i - first + last;
    const int in = static_cast<int>(x - i * row), head = in / pieces, d = (in - head * pieces) * kVec;
    const int64_t e = t * a.o_ts + static_cast<int64_t>(head) * a.o_hs + d;
    *reinterpret_cast<u32x4*>(static_cast<char*>(a.out) + e * (BF16 ? 2 : 4)) = u32x4{0, 0, 0, 0};
    if (a.lse != nullptr && d == 0) a.lse[t * a.H + head] = -INFINITY;
  }
}

// Partial results are written and read by workgroups of different XCDs, whose L2s
// do not see each other's lines: agent-scope accesses, which go through to memory
// (writing an L2 back at a release instead took 30 us of a decode call's 114).
__device__ __forceinline__ void put_partial(float* p, f32x4 x) {
  uint64_t* w = reinterpret_cast<uint64_t*>(p);
  const u32x4 b = __builtin_bit_cast(u32x4, x);
  __hip_atomic_store(w, b[0] | (static_cast<uint64_t>(b[1]) << 32), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store(w + 1, b[2] | (static_cast<uint64_t>(b[3]) << 32), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void put_partial(float* p, float x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x4 get_partial4(const float* p) {
  const uint64_t* w = reinterpret_cast<const uint64_t*>(p);
  const uint64_t x = __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const uint64_t y = __hip_atomic_load(w + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return __builtin_bit_cast(f32x4, u32x4{static_cast<uint32_t>(x), static_cast<uint32_t>(x >> 32), static_cast<uint32_t>(y),
                                         static_cast<uint32_t>(y >> 32)});
}
__device__ __forceinline__ float get_partial(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Counts one of an item's workgroups that is done; true in every thread of the
// last one.  Every thread's partial results have reached memory when the counter
// moves (stores that were waited for), so the last one reads all of them.  The
// counter ends at zero.
__device__ __forceinline__ bool last_to_arrive(int* count, int of, int& shared) {
  mem_fence_compiler();
  __builtin_amdgcn_s_waitcnt(wait_vm(0));
  __syncthreads();
  if (threadIdx.x == 0) {
    const int n = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    shared = n == of - 1;
    if (n == of - 1) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  mem_fence_compiler();
  return shared != 0;
}

// Joins an item's np partial results: the maxima of 8 rows at a time through LDS, then
// each thread 4 columns of a row of every groups-th part.
template <bool BF16, int DT>
__device__ __forceinline__ void row_join(const PagedArgs& a, const addr::PagedSeq& sq, int j, int nrow, int h,
                                         const float* first, int np, RowShared<DT>& sh) {
  constexpr int kRows = 8;                           // kRows * np maxima fit into sh.o: np <= addr::kMostParts
  const int tid = threadIdx.x;
  float* sm = &sh.o[0][0][0];                        // [np][8]
  const auto slot_of = [&](int p) { return first + p * addr::paged_partial_floats(DT); };
  for (int r0 = 0; r0 < nrow; r0 += kRows) {
    const int nr = min(kRows, nrow - r0);
    const int items = nr * (DT / 4);                 // (row, 4 columns)
    const int groups = max(1, 256 / items);
    for (int base = 0; base < items; base += 256) {
      const int x = base + (groups > 1 ? tid % items : tid);
      const int g = groups > 1 ? tid / items : 0;
      const bool in = x < items && g < groups;
      const int q = in ? x / (DT / 4) : 0, d = in ? (x - q * (DT / 4)) * 4 : 0;
      float M = -INFINITY, L = 0.f;
      f32x4 acc = {0, 0, 0, 0};
      // 16 parts' loads in flight at a time; past the last they repeat it with weight 0
      f32x4 px[16];
      float lx[16];
      const auto load = [&](int p0) {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float* sl = slot_of(min(p0 + k * groups, np - 1));
          px[k] = get_partial4(sl + (r0 + q) * DT + d);
          lx[k] = get_partial(sl + 16 * DT + 16 + r0 + q);
        }
      };
      if (in) load(g);
      if (base == 0) {                               // the maxima meanwhile
        __syncthreads();
        for (int x = tid; x < np * kRows; x += 256) {
          const int q = x & (kRows - 1);
          sm[x] = q < nr ? get_partial(slot_of(x / kRows) + 16 * DT + r0 + q) : -INFINITY;
        }
        __syncthreads();
      }
      if (in) {
#pragma unroll 8
        for (int p = 0; p < np; ++p) M = fmaxf(M, sm[p * kRows + q]);
        const float ms = M == -INFINITY ? 0.f : M;
        for (int p0 = g; p0 < np; p0 += 16 * groups) {
          if (p0 != g) load(p0);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int p = p0 + k * groups;
            const float f = p < np ? __builtin_amdgcn_exp2f(sm[min(p, np - 1) * kRows + q] - ms) : 0.f;
            L += f * lx[k];
            acc += f * px[k];
          }
        }
      }
      if (groups > 1) {
        sh.red[tid][0] = L;
#pragma unroll
        for (int i = 0; i < 4; ++i) sh.red[tid][1 + i] = acc[i];
        __syncthreads();
        if (in && g == 0)
          for (int k = 1; k < groups; ++k) {
            L += sh.red[k * items + tid][0];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] += sh.red[k * items + tid][1 + i];
          }
      }
      if (in && g == 0) {
        const int64_t rr = static_cast<int64_t>(j) * 16 + r0 + q;
        const int qi = static_cast<int>(rr / a.G);
        row_store<BF16>(a, sq.q0 + qi, h * a.G + static_cast<int>(rr - static_cast<int64_t>(qi) * a.G), d, acc, M, L);
      }
    }
  }
}

// One part of an item, for key/value head h.
template <bool BF16, int DT, bool E4M3 = false>
__device__ __forceinline__ void row_part(const PagedArgs& a, const RowItem& it, int h, RowShared<DT>& sh) {
  using F = PagedForm<BF16, DT, E4M3>;
  constexpr int kOC = F::kVN * F::kVW;               // O^T tiles of 16 columns
  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63;
  const int lq = l & 15, lg = l >> 4;
  const int s = it.s, j = it.j;
  const addr::PagedSeq& sq = it.sq;
  const addr::PagedTile tile = addr::paged_tile(sq, a.G, a.window, j);
  int w0 = 0, w1 = it.units;
  if (it.nparts > 1) addr::chunk_part_range(it.units, it.part, it.nparts, w0, w1);

  // ---- the lane's query row ---------------------------------------------------------
  const int64_t rows = static_cast<int64_t>(sq.n) * a.G;
  const int64_t r = static_cast<int64_t>(j) * 16 + lq;
  const bool live = r < rows;
  int qi = tile.i0, qh = h * a.G;
  if (live) {
    if (rows <= 16) {                                // the one tile: small numbers
      uint32_t x, y;
      addr::div_by(lq, a.G, a.g_magic, x, y);
      qi = static_cast<int>(x);
      qh += static_cast<int>(y);
    } else {
      qi = static_cast<int>(r / a.G);
      qh += static_cast<int>(r - static_cast<int64_t>(qi) * a.G);
    }
  }
  const int hi = live ? sq.len - sq.n + qi + 1 : 0;  // sees [lo, hi)
  const int lo = a.window > 0 ? hi - a.window : 0;
  const int64_t qe = static_cast<int64_t>(sq.q0 + qi) * a.q_ts + static_cast<int64_t>(qh) * a.q_hs;
  u32x4 qf[F::kSteps];
#pragma unroll
  for (int st = 0; st < F::kSteps; ++st) {
    const int d = row_q_col<BF16, DT, E4M3>(st, lg);
    const u32x4 x = *reinterpret_cast<const u32x4*>(static_cast<const char*>(a.q) + (qe + (d < a.D ? d : 0)) * F::kES);
    qf[st] = live && d < a.D ? x : u32x4{0, 0, 0, 0};
  }
  float m = -INFINITY, lsum = 0.f;
  f32x4 o[kOC];
#pragma unroll
  for (int c = 0; c < kOC; ++c) o[c] = f32x4{0, 0, 0, 0};

  // ---- its keys ---------------------------------------------------------------------
  const int nblk = (tile.ve - tile.first + F::kBlock - 1) / F::kBlock;
  const int b_end = min(w1 * kPWaves, nblk);
  const int32_t* trow = a.table + static_cast<int64_t>(s) * a.ld_table;
  // first keys of the 8 that the lane's K rows and its V rows are of
  const int k_oct = BF16 ? 8 * (lq >> 2) : 8 * (lq >> 3);
  const int v_oct = BF16 ? 8 * lg : 8 * (lg >> 1);
  const int k_in = BF16 ? (lq & 3) : (lq & 7);       // K row within them (+ 4 for tile 1)
  const int v_in = BF16 ? 0 : 4 * (lg & 1);
  const char* k_head = static_cast<const char*>(a.k) + static_cast<int64_t>(h) * a.k_hs * F::kCS;
  const char* v_head = static_cast<const char*>(a.v) + static_cast<int64_t>(h) * a.v_hs * F::kCS;
  struct Ids {
    int k, v;
    uint32_t k_row, v_row;
  };
  const auto ids_of = [&](int b) {
    const int tb = tile.first + b * F::kBlock;
    uint32_t kp, kr, vp, vr;
    addr::div_by(static_cast<uint32_t>(addr::paged_octet(tb + k_oct, tile.ve)) >> 3, a.page_octets, a.page_magic, kp, kr);
    addr::div_by(static_cast<uint32_t>(addr::paged_octet(tb + v_oct, tile.ve)) >> 3, a.page_octets, a.page_magic, vp, vr);
    return Ids{trow[kp], trow[vp], kr * 8 + k_in, vr * 8 + v_in};
  };
  const auto load = [&](const Ids& id, PagedBlock<BF16, DT, E4M3>& x) {
    const int64_t k_page = addr::paged_page(id.k, a.num_pages), v_page = addr::paged_page(id.v, a.num_pages);
    const char* kp = k_head + (k_page * a.k_ps + id.k_row * a.k_rs) * F::kCS;
    const char* vp = v_head + (v_page * a.v_ps + id.v_row * a.v_rs) * F::kCS;
    if constexpr (E4M3) {
      x.s.k = *reinterpret_cast<const u32x2*>(a.ks + k_page * a.ks_ps + h * a.ks_hs + (id.k_row & ~7u));
      x.s.v = *reinterpret_cast<const u32x2*>(a.vs + v_page * a.vs_ps + h * a.vs_hs + (id.v_row & ~7u));
    }
#pragma unroll
    for (int t = 0; t < F::kKT; ++t)
#pragma unroll
      for (int p = 0; p < F::kKP; ++p) {
        const int d = row_k_col<BF16, DT, E4M3>(p, lg);
        x.k[t][p] = *reinterpret_cast<const u32x4*>(kp + (4 * t * a.k_rs + (d < a.D ? d : 0)) * F::kCS);
      }
#pragma unroll
    for (int t = 0; t < F::kKeys; ++t)
#pragma unroll
      for (int n = 0; n < F::kVN; ++n) {
        const int d = n * 16 * F::kVW + F::kVW * lq;
        x.v[t][n] = *reinterpret_cast<const typename VVec<F::kVW * F::kCS>::T*>(vp + (t * a.v_rs + (d < a.D ? d : 0)) * F::kCS);
      }
  };
  const int hi_min = sq.len - sq.n + tile.i0 + 1;    // keys below it and from lo_max on: seen by every row
  const int lo_max = a.window > 0 ? sq.len - sq.n + tile.i1 + 1 - a.window : 0;
  const bool pad = DT > a.D;

  const auto step = [&](int b, PagedBlock<BF16, DT, E4M3>& x) {
    const int tb = tile.first + b * F::kBlock;
    f32x4 sacc[F::kKT];
#pragma unroll
    for (int t = 0; t < F::kKT; ++t) sacc[t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int p = 0; p < F::kKP; ++p)
#pragma unroll
      for (int t = 0; t < F::kKT; ++t) {
        u32x4 kx = x.k[t][p];
        if (pad && row_k_col<BF16, DT, E4M3>(p, lg) >= a.D) kx = u32x4{0, 0, 0, 0};
        if constexpr (!E4M3 && BF16) {
          sacc[t] = mfma16_bf16(kx, qf[p], sacc[t]);
        } else if constexpr (!E4M3) {
#pragma unroll
          for (int e = 0; e < 4; ++e) sacc[t] = mfma16_f32(__uint_as_float(kx[e]), __uint_as_float(qf[p][e]), sacc[t]);
        } else if constexpr (BF16) {                 // y 2^e is exact in bf16
          const float f = scale_of(x.s.k[t], k_in);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            u32x4 ky;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              ky[2 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(kx[2 * e + w], f, false));
              ky[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(kx[2 * e + w], f, true));
            }
            sacc[t] = mfma16_bf16(ky, qf[2 * p + e], sacc[t]);
          }
        } else {
          const float f = scale_of(k_in < 4 ? x.s.k[0] : x.s.k[1], k_in & 3);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f32x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(kx[e], f, false);
            const f32x2_t up = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(kx[e], f, true);
            const float ky[4] = {lo[0], lo[1], up[0], up[1]};
#pragma unroll
            for (int w = 0; w < 4; ++w) sacc[t] = mfma16_f32(ky[w], __uint_as_float(qf[4 * p + e][w]), sacc[t]);
          }
        }
      }
    float sc[F::kKeys];
#pragma unroll
    for (int i = 0; i < F::kKeys; ++i) sc[i] = sacc[i >> 2][i & 3] * a.scale_log2;
    if (tb + F::kBlock > hi_min || tb < lo_max) {
      const int t0 = tb + F::kKeys * lg;           // the lane's first key
#pragma unroll
      for (int i = 0; i < F::kKeys; ++i) {
        const int t = t0 + i;
        if (t >= hi || t < lo) sc[i] = -INFINITY;
        // a key that no row of the tile sees may hold anything: 0 * NaN is not 0
        if (t >= tile.ve || t < tile.vs) {
#pragma unroll
          for (int n = 0; n < F::kVN; ++n)
#pragma unroll
            for (int w = 0; w < F::kVW * F::kCS / 4; ++w) x.v[i][n][w] = 0;
          if constexpr (E4M3) {                      // nor is 0 * inf: its scale is one
            const int at = (BF16 ? i : v_in + i), sh = 8 * (at & 3);
            const uint32_t one = (x.s.v[at >> 2] & ~(255u << sh)) | (127u << sh);
            x.s.v[0] = at < 4 ? one : x.s.v[0];
            x.s.v[1] = at < 4 ? x.s.v[1] : one;
          }
        }
      }
    }
    float mx = sc[0];
#pragma unroll
    for (int i = 1; i < F::kKeys; ++i) mx = fmaxf(mx, sc[i]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    // the reference point follows the maximum once it has grown by 2^8: the sums
    // stay far from their limits, and o is rarely scaled
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx);
      const float f = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);   // m = mn = -inf: nothing summed yet
      m = mn;
      lsum *= f;
#pragma unroll
      for (int c = 0; c < kOC; ++c) o[c] *= f;
    }
    const float ms = m == -INFINITY ? 0.f : m;
    float p[F::kKeys];
#pragma unroll
    for (int i = 0; i < F::kKeys; ++i) {
      p[i] = __builtin_amdgcn_exp2f(sc[i] - ms);
      lsum += p[i];
      if constexpr (E4M3 && !BF16) p[i] *= fmaxf(scale_of(v_in == 0 ? x.s.v[0] : x.s.v[1], i), 0x1p-127f);
    }
    if constexpr (BF16 && E4M3) {
      // The values' scales are the probabilities', which enter the product as two bf16 numbers,
      // off by 2^-16 of themselves, which leaves the result's own rounding: 1.6e-3 from 64 bits for
      // 256 sequences of 16 .. 2047 keys in 68.2 us, 1.7e-3 in 67.5 with one number (2^-8), as the
      // products take 9% of the cycles and 6% then.  A column's bytes of two keys are brought
      // together before they become bf16.
      const auto add = [&](const float (&w8)[8], const auto& into) {
        u32x4 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          hi[i] = pack_bf16x2(w8[2 * i], w8[2 * i + 1]);
          lo[i] = pack_bf16x2(w8[2 * i] - __uint_as_float(hi[i] << 16), w8[2 * i + 1] - __uint_as_float(hi[i] & 0xffff0000u));
        }
#pragma unroll
        for (int n = 0; n < F::kVN; ++n)
#pragma unroll
          for (int w = 0; w < F::kVW / 4; ++w)
#pragma unroll
            for (int up = 0; up < 2; ++up) {
              u32x4 vf[2];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t y = __builtin_amdgcn_perm(x.v[2 * i + 1][n][w], x.v[2 * i][n][w], up ? 0x07030602u : 0x05010400u);
                vf[0][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.f, false));
                vf[1][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.f, true));
              }
#pragma unroll
              for (int e = 0; e < 2; ++e) into(o[n * F::kVW + 4 * w + 2 * up + e], vf[e], hi, lo);
            }
      };
      // A probability times 2^-126, the least scale, has no bf16 digits left: scales below 2^-63
      // count 2^96 times over, in sums of their own.  Where every block has them (rows of zeros have
      // that scale, too) 256 sequences' decode takes 5% more, elsewhere 0.4%.
      const u32x2 less = {tiny_bytes(x.s.v[0]), tiny_bytes(x.s.v[1])};
      const bool tiny = __any((less[0] | less[1]) != 0);
      u32x2 scales = x.s.v;
      if (tiny) scales &= ~less;
      float w8[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w8[i] = p[i] * scale_of(scales[i >> 2], i & 3);
      add(w8, [](f32x4& sum, u32x4 vf, u32x4 hi, u32x4 lo) { sum = mfma16_bf16(vf, hi, mfma16_bf16(vf, lo, sum)); });
      if (tiny) {
        // converted again, or all of them would be kept from the sums before
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int n = 0; n < F::kVN; ++n)
#pragma unroll
            for (int w = 0; w < F::kVW / 4; ++w) {
              uint32_t y = x.v[i][n][w];
              asm("" : "+v"(y));
              x.v[i][n][w] = y;
            }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t code = (x.s.v[i >> 2] >> (8 * (i & 3))) & 255u;
          w8[i] = code < 64 ? p[i] * __uint_as_float((code + 96) << 23) : 0.f;
        }
        add(w8, [](f32x4& sum, u32x4 vf, u32x4 hi, u32x4 lo) {
          sum += mfma16_bf16(vf, hi, mfma16_bf16(vf, lo, f32x4{0, 0, 0, 0})) * 0x1p-96f;
        });
      }
    } else if constexpr (BF16) {
      // Probabilities enter the product in bf16, their total stays in fp32.  Each is off by
      // up to 2^-8 of itself, as the values and the result are; with values of both signs a
      // result's error against 64 bits grows to at most sqrt(2) of what its own rounding
      // leaves: 1.9e-3 for 256 sequences of 16 .. 2047 keys and 2.2e-3 for one of 131071.  As
      // the sum of two bf16 numbers each they give 1.7e-3 and take 110.7 and 106.7 us, where
      // this takes 109.0 and 104.8.
      u32x4 pf;
#pragma unroll
      for (int i = 0; i < 4; ++i) pf[i] = pack_bf16x2(p[2 * i], p[2 * i + 1]);
#pragma unroll
      for (int n = 0; n < F::kVN; ++n)
#pragma unroll
        for (int c = 0; c < F::kVW; ++c) {
          u32x4 vf;
#pragma unroll
          for (int i = 0; i < 4; ++i) vf[i] = pair16(x.v[2 * i][n][c >> 1], x.v[2 * i + 1][n][c >> 1], c & 1);
          o[n * F::kVW + c] = mfma16_bf16(vf, pf, o[n * F::kVW + c]);
        }
    } else if constexpr (E4M3) {
#pragma unroll
      for (int n = 0; n < F::kVN; ++n)
#pragma unroll
        for (int w = 0; w < F::kVW / 4; ++w)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const f32x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x.v[t][n][w], 1.f, false);
            const f32x2_t up = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x.v[t][n][w], 1.f, true);
            const float y[4] = {lo[0], lo[1], up[0], up[1]};
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n * F::kVW + 4 * w + e] = mfma16_f32(y[e], p[t], o[n * F::kVW + 4 * w + e]);
          }
    } else {
#pragma unroll
      for (int n = 0; n < F::kVN; ++n)
#pragma unroll
        for (int c = 0; c < F::kVW; ++c)
#pragma unroll
          for (int t = 0; t < 4; ++t)
            o[n * F::kVW + c] = mfma16_f32(__uint_as_float(x.v[t][n][c]), p[t], o[n * F::kVW + c]);
    }
  };
  // A block's loads are issued before the one ahead of it is used (one buffer, its keys
  // and its values refilled in turn, and three workgroups a CU: 141 us against 124 for
  // 256 sequences of 16 .. 2047 keys then), and page ids one block before them.
  int b = w0 * kPWaves + wave;
  if (b < b_end) {
    PagedBlock<BF16, DT, E4M3> cur, nxt;
    Ids id = ids_of(b);
    load(id, cur);
    id = ids_of(b + kPWaves);
    for (; b + kPWaves < b_end; b += kPWaves) {
      const Ids id2 = ids_of(b + 2 * kPWaves);
      load(id, nxt);
      step(b, cur);
      cur = nxt;
      id = id2;
    }
    step(b, cur);
  }

  // ---- the four waves' results, joined --------------------------------------------
  lsum += __shfl_xor(lsum, 16, 64);
  lsum += __shfl_xor(lsum, 32, 64);
  if (lg == 0) {
    sh.m[wave][lq] = m;
    sh.l[wave][lq] = lsum;
  }
#pragma unroll
  for (int n = 0; n < F::kVN; ++n)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      // O^T row 4 lg + v of tile (n, c): column 16 kVW n + kVW (4 lg + v) + c
      const int d = n * 16 * F::kVW + F::kVW * (4 * lg + v);
#pragma unroll
      for (int c = 0; c < F::kVW; c += 4)
        *reinterpret_cast<f32x4*>(&sh.o[wave][lq][d + c]) =
            f32x4{o[n * F::kVW + c][v], o[n * F::kVW + c + 1][v], o[n * F::kVW + c + 2][v], o[n * F::kVW + c + 3][v]};
    }
  __syncthreads();
  const int nrow = static_cast<int>(min(static_cast<int64_t>(16), rows - static_cast<int64_t>(j) * 16));
  const int64_t slot0 = static_cast<int64_t>(h) * a.row_slots + it.slot;
  float* first = a.ws + slot0 * addr::paged_partial_floats(DT);
  float* slot = first + it.part * addr::paged_partial_floats(DT);
  for (int x = tid; x < nrow * (DT / 4); x += 256) {
    const int q = x / (DT / 4), d = (x - q * (DT / 4)) * 4;
    float M = sh.m[0][q];
#pragma unroll
    for (int w = 1; w < kPWaves; ++w) M = fmaxf(M, sh.m[w][q]);
    const float ms = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    f32x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kPWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(sh.m[w][q] - ms);
      L += f * sh.l[w][q];
      acc += f * *reinterpret_cast<const f32x4*>(&sh.o[w][q][d]);
    }
    if (it.nparts > 1) {
      put_partial(slot + q * DT + d, acc);
      if (d == 0) {
        put_partial(slot + 16 * DT + q, M);
        put_partial(slot + 16 * DT + 16 + q, L);
      }
    } else {
      const int64_t rr = static_cast<int64_t>(j) * 16 + q;
      const int qo = static_cast<int>(rr / a.G);
      row_store<BF16>(a, sq.q0 + qo, h * a.G + static_cast<int>(rr - static_cast<int64_t>(qo) * a.G), d, acc, M, L);
    }
  }
  if (it.nparts > 1 && last_to_arrive(a.row_count + slot0, it.nparts, sh.last))
    row_join<BF16, DT>(a, sq, j, nrow, h, first, it.nparts, sh);
}

// Workgroups i of n of each key/value head take its parts i, 2 n - 1 - i, 2 n + i, ...:
// the parts get shorter, so whoever has a longer one has a shorter one next.  One
// start for several parts: 223 sequences of 4 .. 429 keys with 16 heads 60 us against 71
// with a workgroup for each, 1024 of 16 .. 400 with 8 heads 164 against 229.  The first
// wave lists up to 32 of a workgroup's parts in one pass over the batch.
constexpr int kRowList = 32;
template <bool BF16, int DT, bool E4M3 = false>
__global__ __launch_bounds__(256, DT == 256 ? 1 : 2) void paged_attention_kernel(PagedArgs) {
  __shared__ RowShared<DT> sh;
  __shared__ RowOrder<BF16, DT> kept[64];            // a lane's, between lists
  __shared__ RowEntry list[kRowList];
  __shared__ int parts;
  const int HK = fresh_args().HK;
  const int i = blockIdx.x / HK, h = blockIdx.x - i * HK, n = gridDim.x / HK;
  for (int k0 = 0;; k0 += kRowList) {
    if (threadIdx.x < 64) {
      const PagedArgs& a = fresh_args();
      RowOrder<BF16, DT> order;
      if (k0 == 0) {
        order.plan(a);
        kept[threadIdx.x] = order;
        if (threadIdx.x == 0) parts = order.total;
      } else {
        order = kept[threadIdx.x];
      }
      order.list_parts(a, i, n, k0, k0 + kRowList, list);
    }
    __syncthreads();
    const int total = __builtin_amdgcn_readfirstlane(parts);
    for (int k = k0; k < k0 + kRowList && k * n < total; ++k) {
      if (k * n + ((k & 1) != 0 ? n - 1 - i : i) >= total) continue;
      row_part<BF16, DT, E4M3>(fresh_args(), row_item(list[k - k0]), h, sh);
      __syncthreads();                               // every wave is past what the part left in sh, and its entry
    }
    if ((k0 + kRowList) * n >= total) break;
  }
  zero_outside<BF16>(fresh_args());
}

}  // namespace
}  // namespace gs
