// Attention of drafted tokens over a bf16 or 8-bit cache on the tensor cores (tcgen05), head widths 64, 128, 256.
//
//   out(i, h) = sum_t softmax_t(q(i, h) . k(t) / sqrt(D)) v(t),   t: the cached slots, node i's ancestors, node i
//
// The rows of a unit (sequence, KV head) are its nodes times the query heads of the KV head, row = node *
// group + head, so the cache is read once for all of them.  They are the 128 lanes of the MMA tiles:
//   S = Q K^T   M 128, N 64 keys, A = Q, B = the key tile (K-major)
//   O += P V    M 128, N D, A = P (bf16) written over S in TMEM, B = the value tile (MN-major)
// with one thread per row doing the softmax (running maximum with lazy rescaling of O, fp32 sums).  Few rows leave
// lanes idle, which costs nothing while the tiles arrive at memory speed: a 64-key tile of width 128 takes
// 512 clocks of the tensor pipe and 712 (8-bit) or 1424 (bf16) of an SM's share of the HBM rate.
//
// Two streams of S, O and softmax warps run side by side so that one's products run under the other's softmax.
// Up to 128 rows: the streams take the even and the odd key tiles and are merged at the end.  More (kWide): each
// takes 128 rows and both read every tile; Q moves to shared memory, which makes room in TMEM for two score buffers
// per stream, so that the softmax, which bounds this form, does not wait for the product before it.  Width 256 (O takes
// half of TMEM): one stream with two score buffers.
//
// Loading.  Four warps copy the rows into a ring with asynchronous 16-byte copies; pages may have any size and rows any
// 16-byte stride.  Whole tiles of bf16 rows (and 8-bit ones of width 256) in pages of a multiple of 16 come by tiled copies
// instead, one lane's work; the tiles with drafts and the last one do not, since what lies behind must be zeros.  bf16 rows land as the swizzled tiles that the products read.  8-bit codes land as they are (up to 96 KB
// per SM in flight) and eight more warps widen them to fp16 tiles, one instruction per two codes and exact.
// Keys are multiplied by their row's 2^n where fp16 holds every product (-15 <= n <= 7, values from 2^-24 to 57344); values by
// 2^(n - N), 2^N the largest of the tile, where n >= N - 15 for all of its rows and none of them is a draft.  Tiles with
// other rows keep their codes and the softmax multiplies scores and weights by the rows' factors.  P carries 11 bits, over
// bf16 caches 8.
//
// Work is cut evenly over the SMs as tree_line.cuh says, one CTA per SM.
//
// Measured (B200, 16 sequences of 8000 tokens, 40 and 8 heads of 128, with the merge): 40 rows per KV head, bf16 113 us, 8-bit
// 141; 100 rows 125 and 152; 305 rows 296 and 407, where the softmax bounds it: one warp's chain of loads, maxima, exponentials and
// stores, two such warps per scheduler.  Up to 128 rows the 8-bit form is the slower one: its codes pass shared memory twice.
#include <stddef.h>

#include "tree_line.cuh"

namespace pluto {
namespace {

constexpr int kTile = 64, kHalf = kTile / 2;   // keys of a tile, and of what the softmax takes at a time
template <bool kEight>
constexpr int kThreads = kEight ? 768 : 512;   // warps 0-3: MMA issue; 4-11: softmax; 12-15: loads; 16-23: widening
constexpr int kMaxCtas = 148;
constexpr int kUnitTiles = 3;        // query load and read-out of a unit, in tiles
constexpr float kRescale = 8.0f;     // O is rescaled when the maximum has grown by more than 2^8
constexpr float kSmallest = -118.0f;   // exponent of the value rows from which smaller ones are taken for as large: weights of up
                                       // to 2^8 times 2^118 stay finite
constexpr float kLargeScore = 1048576.0f;   // scores (in powers of two) whose own rounding is less than 2^-4
constexpr float kApart = 60.0f;        // exponents between value rows beyond which the smaller ones' weights are zero in fp16, far
                                       // from where their sum would lose them

// kWide: more than 128 rows may share a pass over the keys (never at width 256)
template <int D, bool kEight, bool kWide>   // tiles of keys, and of values
constexpr int kStages = kEight ? (D == 64 ? 6 : D == 128 && !kWide ? 3 : 2) : (D == 64 ? 10 : D == 128 ? (kWide ? 4 : 6) : 3);
// Key and value tiles as codes.  An even number: warps load and widen every other tile, and a parity tells a phase from its two
// neighbours only, so a warp has to meet every use of its slots (three slots gave a wrong result in one of a thousand calls).
// The products release the widened tiles in their order, whoever fills them, so those rings may have any length.
template <int D, bool kWide>
constexpr int kRawStages = D == 64 ? 8 : D == 128 ? (kWide ? 4 : 6) : 2;
template <int D>
constexpr int kTileBytes = kTile * D * 2;
constexpr int group_rows(int dim) { return dim == 256 ? 128 : 256; }   // rows that share one pass over the keys

// Tiled copies where pages allow them: 40 rows of width 128, bf16: 114 -> 102 us; 48 rows of width 256, 8-bit: 78 -> 74.  Narrower
// 8-bit tiles are no faster by them (135 -> 139): widening bounds those.
template <int D, bool kEight>
constexpr bool kBoxes = !kEight || D == 256;

// ---- shared memory -------------------------------------------------------------------------------------------
constexpr int kSegments = 8;         // of the ring
template <bool kWide>
constexpr int kSegmentReaders = kWide ? 14 : 13;   // warps: MMA issue, eight softmax, four loaders

template <int D, bool kEight, bool kWide>
struct Shared {
  static constexpr int kTiles = kStages<D, kEight, kWide>, kRaw = kEight ? kRawStages<D, kWide> : 1;
  static_assert(kRawStages<D, kWide> % 2 == 0, "a warp meets every use of its slots");
  uint64_t seg_full[kSegments], seg_empty[kSegments];
  uint64_t k_full[kTiles], k_empty[kTiles], v_full[kTiles], v_empty[kTiles];
  uint64_t raw_k[kRaw], raw_v[kRaw], raw_scales[kRaw], raw_empty[kRaw];
  // Softmax warps have come to a segment, with its queries: the first stream's; the second's in a pair; the second's otherwise.
  // Three, as neither stream may come to a barrier's next phase before the other has come to this one: in pairs they pass
  // a segment alone.
  uint64_t q_full[3];
  uint64_t s_full[2][2], p_half[2][2], p_full[2][2], pv_half[2][2], pv_done[2][2];   // [stream][score buffer]
  uint64_t ml_full, o_read;   // the two streams' meeting points: sums written, O read
  Segment seg[kSegments];
  uint32_t tmem;
  float2 ml[2][128];
  float unit[2][kEight ? 128 : 1];   // v_used of the rows
  // 8-bit caches: the raw tiles' scale bytes and first draft that not every node sees (-1: the range ends)
  uint8_t k_byte[kRaw][kTile], v_byte[kRaw][kTile];
  int draft_row[kRaw], border[kRaw];   // (border: the tile holds drafts)
  // ... and per tile whether the softmax has to apply the rows' factors, and the largest exponent of its value rows.  A ring
  // of three times the stages: a slot is written again once the stage of the tile two rounds on is free, and that
  // tile's scores are issued behind the product of this one, whose softmax has then read them.
  alignas(16) float k_factor[3 * kTiles][kTile];   // (read four at a time)
  float v_factor[3 * kTiles][kTile];
  int scaled[3 * kTiles], v_largest[3 * kTiles];   // scaled: kKeysScaled, kValuesScaled
  uint32_t v_top[3 * kTiles][2];                   // the rows that have it
};

// The next segment of the range, by every lane of a warp; false at its end (or when a wait ran out).
template <typename S>
__device__ __forceinline__ bool next_segment(S* sh, int& n, Segment& seg, int lane, uint32_t* status) {
  const int at = n % kSegments;
  if (!__all_sync(0xffffffffu, tree_wait(&sh->seg_full[at], (n / kSegments) & 1, status, 61))) return false;
  seg = sh->seg[at];
  ++n;
  __syncwarp();
  if (lane == 0) mbar_arrive(&sh->seg_empty[at]);
  return seg.rows > 0;
}

// ---- loaders -------------------------------------------------------------------------------------------------
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {   // zeros where it is not
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void arrive_behind_copies(uint64_t* bar) {   // when this thread's copies so far have landed
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool not_finite(uint32_t pair) {
  return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u;
}
__device__ __forceinline__ bool not_finite(const uint4& v) {
  return not_finite(v.x) || not_finite(v.y) || not_finite(v.z) || not_finite(v.w);
}
// Where (row, piece of 8 channels) of a tile lies: 64-channel slabs of 64 rows x 128 bytes, 128-byte swizzle.
__device__ __forceinline__ uint32_t tile_piece(uint32_t tile, int r, int piece) {
  return tile + (piece / 8) * (kTile * 128) + r * 128 + (((piece & 7) ^ (r & 7)) << 4);
}

__device__ __forceinline__ uint32_t load_byte(const uint8_t* p, bool there, uint32_t otherwise) {
  uint32_t v;
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.u32 %0, %3;\n\t@p ld.global.u8 %0, [%1];\n\t}"
               : "=r"(v) : "l"(p), "r"(static_cast<uint32_t>(there)), "r"(otherwise));
  return v;
}

// Four warps; a warp copies every fourth half tile (32 rows of keys and of values), a lane looking after the page and the
// scales of its row.  Nothing is used in the step that asks for it: pages are fetched one unit ahead of the
// copies, scale bytes are passed on one unit later.
template <int D, bool kEight, bool kWide>
__device__ __forceinline__ void load_tiles(const TreeArgs& a, const CUtensorMap& map_k, const CUtensorMap& map_v, int box, Shared<D, kEight, kWide>* sh, uint32_t k_ring, uint32_t v_ring, int warp, int lane) {
  constexpr int kRing = kEight ? kRawStages<D, kWide> : kStages<D, kEight, kWide>;
  constexpr int kElement = kEight ? 1 : 2, kBytes = kTile * D * kElement, kPieces = D * kElement / 16, kLoads = kPieces;
  uint64_t* k_full = kEight ? sh->raw_k : sh->k_full;
  uint64_t* v_full = kEight ? sh->raw_v : sh->v_full;
  uint32_t* status = a.pool.status;
  const int page_shift = (a.pool.page_size & (a.pool.page_size - 1)) == 0 ? __ffs(a.pool.page_size) - 1 : -1;
  const int first_row = (warp & 1) * 32, own = first_row + lane;   // row of the tile
  Segment seg;
  int seg_n = 0, n = warp >> 1, tile = 0, page = -1;   // tile number n of the range is `tile` of the segment
  bool more = next_segment(sh, seg_n, seg, lane, status);
  if (more) tile = seg.tile0 + n;
  const auto settle = [&]() {
    while (more && tile >= seg.tile1) {
      const int beyond = tile - seg.tile1;
      more = next_segment(sh, seg_n, seg, lane, status);
      if (more) tile = seg.tile0 + beyond;
    }
    const int t = tile * kTile + own;
    page = -1;
    if (!more || t >= seg.prefix + seg.count) return;
    const int block = page_shift >= 0 ? t >> page_shift : t / a.pool.page_size;
    if (block >= (a.pool.table ? a.pool.max_blocks : 1)) report_status(status, 48, kBadLength);
    else page = a.pool.table ? a.pool.table[static_cast<size_t>(seg.b) * a.pool.max_blocks + block] : seg.b;
  };
  settle();
  int passed = -1;                 // slot whose scale bytes are to be passed on
  uint32_t k_byte = 0u, v_byte = 0u;
  const auto pass_scales = [&]() {
    if (passed < 0) return;
    sh->k_byte[passed][own] = static_cast<uint8_t>(k_byte);
    sh->v_byte[passed][own] = static_cast<uint8_t>(v_byte);
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh->raw_scales[passed]);
    passed = -1;
  };
  for (;; n += 2, tile += 2, settle()) {
    const int slot = n % kRing, use = n / kRing;
    if (!more && !kEight) break;
    // (two slots: this one is freed once the last unit's scales have been passed on)
    if (kEight && kRing == 2) pass_scales();
    if (use > 0) {
      bool ok = __all_sync(0xffffffffu, tree_wait(kEight ? &sh->raw_empty[slot] : &sh->k_empty[slot], (use - 1) & 1, status, 50));
      if (!kEight) ok = ok && __all_sync(0xffffffffu, tree_wait(&sh->v_empty[slot], (use - 1) & 1, status, 51));
      if (!ok) {   // the copies in flight land (or a limit of tries passes) before their memory is given up
        for (int m = n - 2; m >= 0 && m > n - kRing; m -= 2)
          for (int tries = 0; tries < (1 << 16) && !(mbar_test(&k_full[m % kRing], m / kRing & 1) && mbar_test(&v_full[m % kRing], m / kRing & 1)); ++tries) {}
        return;
      }
    }
    if (!more) {   // the range ends, for the widening warps of this half and parity as well
      if (first_row == 0 && lane == 0) sh->draft_row[slot] = -1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->raw_scales[slot]);
      break;
    }
    const int t = tile * kTile + own, draft_row = seg.count > 1 ? max(0, seg.prefix - tile * kTile) : kTile;
    long long row_at = -1;         // byte offset of the lane's row
    size_t scale_at = 0;
    if (t < seg.prefix + seg.count) {
      if (page < 0 || (a.pool.table && page >= a.pool.num_pages)) {
        report_status(status, 48, kBadPage);   // (a slot past the pages was reported as such before)
      } else {
        const int inside = t - (page_shift >= 0 ? t >> page_shift << page_shift : t / a.pool.page_size * a.pool.page_size);
        row_at = static_cast<long long>((static_cast<size_t>(page) * a.pool.page_stride + static_cast<size_t>(inside) * a.pool.token_stride +
                                         static_cast<size_t>(seg.kv_head) * D) * kElement);
        if (kEight) scale_at = static_cast<size_t>(page) * a.pool.scale_page + static_cast<size_t>(inside) * a.pool.scale_token + seg.kv_head;
      }
    }
    // A tile before the drafts, in pages that boxes divide, comes by tiled copies of one lane.  (Rows behind the last
    // draft must be zeros, which the lanes' own copies write.)
    const bool whole = kBoxes<D, kEight> && box > 0 && (tile + 1) * kTile <= seg.prefix;
    if (whole) {
      const int inside = t - (page_shift >= 0 ? t >> page_shift << page_shift : t / a.pool.page_size * a.pool.page_size);
      const unsigned pages = a.pool.table ? a.pool.num_pages : a.batch;
      const int from = static_cast<unsigned>(page) < pages ? page : -1;   // (reported above; zeros)
      constexpr int kSlabs = kEight ? 1 : D / 64, kSlab = kTile * 128;
      if (lane == 0) {
        mbar_expect_tx(&k_full[slot], kBytes / 2);
        mbar_expect_tx(&v_full[slot], kBytes / 2);
      } else {
        mbar_arrive(&k_full[slot]);
        mbar_arrive(&v_full[slot]);
      }
      for (int r0 = 0; r0 < 32; r0 += box) {
        const int box_page = __shfl_sync(0xffffffffu, from, r0), box_inside = __shfl_sync(0xffffffffu, inside, r0);
        if (lane == 0) {
#pragma unroll
          for (int i = 0; i < kSlabs; ++i) {
            const uint32_t at = slot * kBytes + i * kSlab + (first_row + r0) * (kEight ? D : 128);
            tma_load_4d_at(k_ring + at, &map_k, i * 64, seg.kv_head, box_inside, box_page, &k_full[slot]);
            tma_load_4d_at(v_ring + at, &map_v, i * 64, seg.kv_head, box_inside, box_page, &v_full[slot]);
          }
        }
      }
      __syncwarp();
    }
#pragma unroll
    for (int side = 0; side < 2 && !whole; ++side) {
      const uint32_t to = (side ? v_ring : k_ring) + slot * kBytes;
      const char* base = static_cast<const char*>(side ? a.pool.v : a.pool.k);
#pragma unroll 4
      for (int i = 0; i < kLoads; ++i) {
        const int row = i * (32 / kPieces) + lane / kPieces, c = lane % kPieces, r = first_row + row;
        const long long at = __shfl_sync(0xffffffffu, row_at, row);
        copy16(kEight ? to + r * D + c * 16 : tile_piece(to, r, c), base + (at >= 0 ? at + c * 16 : 0), at >= 0);
      }
      if (kEight || draft_row >= first_row + 32) arrive_behind_copies(side ? &v_full[slot] : &k_full[slot]);
    }
    if (!kEight && !whole && draft_row < first_row + 32) {
      // Drafts that not every node sees: a value row that is not finite must not meet the zero weights of those that do
      // not see it.  It becomes zeros, and the key row NaN, which gives those that see it NaN scores and touches no
      // other node.  (8-bit rows: their scale byte says so, when they are widened.)  A lane looks at its own copies.
      asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 4
      for (int i = 0; i < kLoads; ++i) {
        const int r = first_row + i * (32 / kPieces) + lane / kPieces, c = lane % kPieces;
        if (r >= draft_row && not_finite(lds_b32x4(tile_piece(v_ring + slot * kBytes, r, c)))) {
          sts_b32x4(tile_piece(v_ring + slot * kBytes, r, c), 0u, 0u, 0u, 0u);
          sts_b32x4(tile_piece(k_ring + slot * kBytes, r, c), 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
        }
      }
      mbar_arrive(&k_full[slot]);
      mbar_arrive(&v_full[slot]);
    }
    if (kEight) {
      pass_scales();
      // rows that are not there: keys of an ordinary scale, values of the smallest, which no reference is taken from
      k_byte = load_byte(a.pool.k_scales + scale_at, row_at >= 0, 127u);
      v_byte = load_byte(a.pool.v_scales + scale_at, row_at >= 0, 0u);
      passed = slot;
      if (first_row == 0 && lane == 0) {
        sh->draft_row[slot] = draft_row;
        sh->border[slot] = (tile + 1) * kTile > seg.prefix;
      }
    }
  }
  if (kEight) pass_scales();
}

// ---- 8-bit codes to fp16 -------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t halves_of(uint32_t codes) {   // two codes in the low 16 bits -> two fp16
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(codes)));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// A row's scale byte: 2^n times any of its codes is exact in fp16 for -15 <= n <= 7 (2^-24 to 57344; n = 0 stands in for
// rows that are not finite, whose codes are NaN).
enum : int { kKeysScaled = 1, kValuesScaled = 2 };   // by the softmax
constexpr uint32_t kHalfOne = 0x3c003c00u;
__device__ __forceinline__ bool fits_fp16(uint32_t byte) { return byte == 255u || (byte >= 112u && byte <= 134u); }
__device__ __forceinline__ uint32_t half_power(uint32_t byte) {
  const uint32_t h = byte == 255u ? 0x3c00u : byte >= 113u ? (byte - 112u) << 10 : 0x200u;   // 2^-15 is subnormal
  return h | h << 16;
}

// Eight warps: every fourth half of the key tiles, or of the value tiles, each.
template <int D, bool kWide>
__device__ __forceinline__ void widen_tiles(Shared<D, true, kWide>* sh, uint32_t raw_ring, uint32_t ring, uint32_t* status, int warp, int lane, bool values) {
  constexpr int kTiles = kStages<D, true, kWide>, kRaw = kRawStages<D, kWide>, kPieces = D / 16, kStep = 32 / kPieces;   // rows per step
  const int first_row = (warp & 1) * 32;
  const int row = lane / kPieces, c = lane % kPieces;
  // Channels 16c .. 16c + 15 are pieces 2c and 2c + 1 of the tile's row; odd slabs store the second first, so that eight lanes
  // hit all banks once.  A step is kStep rows, so the swizzle of the two pieces repeats every 8 / kStep steps.
  const int second = c / 4 & 1, slab = c / 4 * (kTile * 128), p0 = (2 * c + second) & 7, p1 = (2 * c + 1 - second) & 7;
  for (int n = warp >> 1;; n += 2) {
    const int slot = n % kRaw, stage = n % kTiles, use = n / kTiles, scale_slot = n % (3 * kTiles);
    if (!__all_sync(0xffffffffu, tree_wait(&sh->raw_scales[slot], (n / kRaw) & 1, status, 47))) return;
    const int draft_row = sh->draft_row[slot];
    if (draft_row < 0) return;
    // the rows' factors: in the codes for all rows of the tile or for none, the values' relative to the largest (`top`)
    const uint32_t k[2] = {sh->k_byte[slot][lane], sh->k_byte[slot][lane + 32]}, v[2] = {sh->v_byte[slot][lane], sh->v_byte[slot][lane + 32]};
    const bool k_fits = __all_sync(0xffffffffu, fits_fp16(k[0]) && fits_fp16(k[1]));
    const uint32_t top = __reduce_max_sync(0xffffffffu, max(v[0] == 255u ? 0u : v[0], v[1] == 255u ? 0u : v[1]));
    const bool v_fits = sh->border[slot] == 0 && __all_sync(0xffffffffu, min(v[0], v[1]) + 15u >= top);
    const uint32_t own_k = first_row ? k[1] : k[0], own_v = first_row ? v[1] : v[0];   // of row first_row + lane
    uint32_t factor = kHalfOne;
    if (values ? v_fits : k_fits) factor = half_power(!values ? own_k : own_v == 255u ? 255u : own_v + 127u - top);
    // Of drafts that not every node sees, values that are not finite are stored as zeros and their keys as NaN (see above).
    const bool hidden = own_v == 255u && first_row + lane >= draft_row;
    if (!values && hidden) factor = 0x7fff7fffu;
    const unsigned zeros = __ballot_sync(0xffffffffu, values && hidden);
    if (use > 0 && !__all_sync(0xffffffffu, tree_wait(values ? &sh->v_empty[stage] : &sh->k_empty[stage], (use - 1) & 1, status, values ? 46 : 45))) return;
    if (!values && first_row == 0) {
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        if (!k_fits) sh->k_factor[scale_slot][lane + 32 * o] = k[o] == 255u ? 1.0f : e8m0_value(k[o]);
        sh->v_factor[scale_slot][lane + 32 * o] = v_fits || v[o] == 255u ? 1.0f : e8m0_value(v[o]);
        const unsigned at_top = __ballot_sync(0xffffffffu, v[o] == top);
        if (lane == 0) sh->v_top[scale_slot][o] = at_top;
      }
      if (lane == 0) {
        sh->scaled[scale_slot] = (k_fits ? 0 : kKeysScaled) | (v_fits ? 0 : kValuesScaled);
        sh->v_largest[scale_slot] = static_cast<int>(top) - 127;
      }
    }
    if (!__all_sync(0xffffffffu, tree_wait(values ? &sh->raw_v[slot] : &sh->raw_k[slot], (n / kRaw) & 1, status, 44))) return;
    uint32_t from = raw_ring + slot * (kTile * D) + (first_row + row) * D + c * 16;
    uint32_t to = ring + stage * kTileBytes<D> + slab + (first_row + row) * 128;
#pragma unroll 4
    for (int i = 0; i < 32 / kStep; ++i) {
      const int r = i * kStep + row, swizzle = r & 7;
      const uint32_t f = __shfl_sync(0xffffffffu, factor, r);
      const uint64_t first = lds_b64(from + second * 8), other = lds_b64(from + 8 - second * 8);
      uint32_t x = static_cast<uint32_t>(first), y = static_cast<uint32_t>(first >> 32);
      uint32_t z = static_cast<uint32_t>(other), w = static_cast<uint32_t>(other >> 32);
      if (zeros != 0u && (zeros >> r & 1u)) x = y = z = w = 0u;
      sts_b32x4(to + ((p0 ^ swizzle) << 4), mul_f16x2(halves_of(x), f), mul_f16x2(halves_of(x >> 16), f), mul_f16x2(halves_of(y), f),
                mul_f16x2(halves_of(y >> 16), f));
      sts_b32x4(to + ((p1 ^ swizzle) << 4), mul_f16x2(halves_of(z), f), mul_f16x2(halves_of(z >> 16), f), mul_f16x2(halves_of(w), f),
                mul_f16x2(halves_of(w >> 16), f));
      from += kStep * D;
      to += kStep * 128;
    }
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(values ? &sh->v_full[stage] : &sh->k_full[stage]);
      mbar_arrive(&sh->raw_empty[slot]);
    }
  }
}

template <int D, bool kEight, bool kWide>
constexpr int kRingBytes = 2 * kStages<D, kEight, kWide> * kTileBytes<D> + (kEight ? 2 * kRawStages<D, kWide> * kTile * D : 0);
template <int D, bool kWide>
constexpr int kQueryBytes = kWide ? 128 * D * 2 : 0;   // of a stream, in shared memory

template <int D, bool kEight, bool kWide>
__global__ void __launch_bounds__(kThreads<kEight>, 1) tree_decode_sm100(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, int box, TreeArgs a, LineShape shape) {
  constexpr bool kOneO = D == 256;                       // one stream
  constexpr int kBuffers = kOneO || kWide ? 2 : 1;       // of scores, per stream
  constexpr uint32_t kColO1 = D, kColS = kOneO ? D : 2 * D, kColQ = kColS + (kOneO ? 1 : 2) * kBuffers * kTile;   // (kWide: the queries lie in shared memory)
  static_assert(kColQ + (kWide ? 0 : D / 2) <= 512 && !(kOneO && kWide), "tensor memory");
  const auto buffer_of = [](int t) { return kBuffers == 2 ? t & 1 : 0; };   // of the stream's tile t
  const auto phase_of = [](int t) { return kBuffers == 2 ? t >> 1 & 1 : t & 1; };
  constexpr uint32_t kBf16 = 1u << 7 | 1u << 10;   // operand types: bf16, or fp16 for 8-bit caches
  constexpr uint32_t kIdescQK = umma_idesc_bf16(128, kTile, false) ^ (kEight ? kBf16 : 0u);
  constexpr uint32_t kIdescPV = umma_idesc_bf16(128, D, true) ^ (kEight ? kBf16 : 0u);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Shared<D, kEight, kWide>* sh = reinterpret_cast<Shared<D, kEight, kWide>*>(smem + kRingBytes<D, kEight, kWide> + 2 * kQueryBytes<D, kWide>);
  const uint32_t k_ring = smem_u32(smem), v_ring = k_ring + kStages<D, kEight, kWide> * kTileBytes<D>;
  const uint32_t raw_k = v_ring + kStages<D, kEight, kWide> * kTileBytes<D>, raw_v = raw_k + kRawStages<D, kWide> * kTile * D;   // 8-bit caches
  const uint32_t queries = k_ring + kRingBytes<D, kEight, kWide>;   // slabs of 64 channels, 128 rows of 128 bytes, swizzled
  const int warp = uniform_warp_index(), lane = threadIdx.x % 32;
  pdl_launch_dependents();   // the merge may be placed as SMs free up; it waits for this grid's end

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages<D, kEight, kWide>; ++s) {
      mbar_init(&sh->k_full[s], kEight ? 2 : 64);
      mbar_init(&sh->v_full[s], kEight ? 2 : 64);
      mbar_init(&sh->k_empty[s], kWide ? 2 : 1);   // (the streams each, or the one that has the tile twice)
      mbar_init(&sh->v_empty[s], kWide ? 2 : 1);
    }
    if (kEight) {
      for (int r = 0; r < kRawStages<D, kWide>; ++r) {
        mbar_init(&sh->raw_k[r], 64);
        mbar_init(&sh->raw_v[r], 64);
        mbar_init(&sh->raw_scales[r], 2);
        mbar_init(&sh->raw_empty[r], 4);
      }
    }
    for (int i = 0; i < kSegments; ++i) {
      mbar_init(&sh->seg_full[i], 1);
      mbar_init(&sh->seg_empty[i], kSegmentReaders<kWide>);
    }
    for (int x = 0; x < 2; ++x) {
      for (int buffer = 0; buffer < 2; ++buffer) {
        mbar_init(&sh->s_full[x][buffer], 1);
        mbar_init(&sh->p_half[x][buffer], 4);
        mbar_init(&sh->p_full[x][buffer], 4);
        mbar_init(&sh->pv_half[x][buffer], 1);
        mbar_init(&sh->pv_done[x][buffer], 1);
      }
    }
    for (int i = 0; i < 3; ++i) mbar_init(&sh->q_full[i], 4);
    mbar_init(&sh->ml_full, 8);
    mbar_init(&sh->o_read, 8);
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(&sh->tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem;
  uint32_t* status = a.pool.status;

  // Register file: 512 threads x 128, nothing to move; or 768 x 80 (of 480 per thread of six warpgroups: issue 56,
  // softmax 2 x 112, loads 56, widening 2 x 72).
  if (warp < 4) {
    if (kEight) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0 || (warp == 2 && kWide)) {
      // ---------------------------------------------------------------- MMA issue
      // A warp per stream where both read every tile; else warp 0 for both, as every tile has to be awaited in its order (a
      // parity tells a phase from its neighbours only).
      int tile_n = 0, own_0 = 0, own_1 = 0, segments = 0, pairs = 0, others = 0;   // so far: tiles, those of the streams, ...
      bool ok = true;
      int seg_n = 0;
      Segment seg;
      while (ok && next_segment(sh, seg_n, seg, lane, status)) {
        const int tiles = __shfl_sync(0xffffffffu, seg.tile1 - seg.tile0, 0);
        const bool pair = kWide && __shfl_sync(0xffffffffu, seg.rows > 128 ? 1 : 0, 0), every = pair || kOneO;   // every: all tiles are a stream's
        if (warp == 0) {
          ok = __all_sync(0xffffffffu, tree_wait(&sh->q_full[0], segments++ & 1, status, 52));
          if (ok && !every) ok = __all_sync(0xffffffffu, tree_wait(&sh->q_full[2], others++ & 1, status, 52));
        } else if (pair) {
          ok = __all_sync(0xffffffffu, tree_wait(&sh->q_full[1], pairs++ & 1, status, 52));
        }
        if (!ok) break;
        const uint64_t q_desc = umma_desc_sw128(queries + (pair && warp ? kQueryBytes<D, kWide> : 0), 16, 1024);
        const auto issue_qk = [&](int x, int u) -> bool {
          const int n = tile_n + (every ? u : 2 * u + x), stage = n % kStages<D, kEight, kWide>, buffer = buffer_of((x ? own_1 : own_0) + u);
          if (!__all_sync(0xffffffffu, tree_wait(&sh->k_full[stage], (n / kStages<D, kEight, kWide>) & 1, status, 53))) return false;
          fence_proxy_async();   // the loaders' stores, before the tensor cores read them
          tc_fence_after();
          const uint64_t k_desc = umma_desc_sw128(k_ring + stage * kTileBytes<D>, 16, 1024);
          const uint32_t s_at = tmem + kColS + (kBuffers * x + buffer) * kTile;
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              const uint64_t k_at = k_desc + (((ks / 4) * (kTile * 128) + (ks % 4) * 32) >> 4);
              if (!kWide) umma_ts(s_at, tmem + kColQ + ks * 8, k_at, kIdescQK, ks > 0);
              else umma_ss(s_at, q_desc + (((ks / 4) * (128 * 128) + (ks % 4) * 32) >> 4), k_at, kIdescQK, ks > 0);
            }
            tc_commit(&sh->s_full[x][buffer]);
            tc_commit(&sh->k_empty[stage]);
            if (kWide && !every) tc_commit(&sh->k_empty[stage]);
          }
          __syncwarp();
          return true;
        };
        const auto issue_pv = [&](int x, int u) -> bool {
          const int n = tile_n + (every ? u : 2 * u + x), stage = n % kStages<D, kEight, kWide>, t = (x ? own_1 : own_0) + u;
          const int buffer = buffer_of(t), phase = phase_of(t);
          if (!__all_sync(0xffffffffu, tree_wait(&sh->v_full[stage], (n / kStages<D, kEight, kWide>) & 1, status, 54))) return false;
          fence_proxy_async();
          const uint64_t v_desc = umma_desc_sw128(v_ring + stage * kTileBytes<D>, kTile * 128, 1024);
          const uint32_t o = tmem + x * kColO1, p = tmem + kColS + (kBuffers * x + buffer) * kTile;
          // the weights come in two halves of the tile's keys; the first half's product runs under the second's softmax
          if (!__all_sync(0xffffffffu, tree_wait(&sh->p_half[x][buffer], phase, status, 55))) return false;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < kTile / 32; ++ks) umma_ts(o, p + ks * 8, v_desc + ks * (2048 >> 4), kIdescPV, u > 0 || ks > 0);
            tc_commit(&sh->pv_half[x][buffer]);
          }
          __syncwarp();
          if (!__all_sync(0xffffffffu, tree_wait(&sh->p_full[x][buffer], phase, status, 55))) return false;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int ks = kTile / 32; ks < kTile / 16; ++ks) umma_ts(o, p + ks * 8, v_desc + ks * (2048 >> 4), kIdescPV, true);
            tc_commit(&sh->pv_done[x][buffer]);
            tc_commit(&sh->v_empty[stage]);
            if (kWide && !every) tc_commit(&sh->v_empty[stage]);
          }
          __syncwarp();
          return true;
        };
        // Where a stream reads every tile and has two score buffers, the next tile's scores are there when the softmax has
        // ended one.  (On alternate tiles two would keep four tiles in the rings.)
        const int ahead = kBuffers == 2 && every ? 2 : 1;
        const int tiles_0 = every ? tiles : (tiles + 1) / 2, tiles_1 = every ? tiles : tiles / 2;
        const int first = pair ? warp >> 1 : 0, last = every ? first : warp ? -1 : 1;
#pragma unroll 1
        for (int u = 0; u < tiles_0 + ahead && ok; ++u)
#pragma unroll 1
          for (int x = first; x <= last && ok; ++x) {
            const int own = x ? tiles_1 : tiles_0;
            if (u >= ahead && u - ahead < own) ok = issue_pv(x, u - ahead);
            if (ok && u < own) ok = issue_qk(x, u);
          }
        tile_n += tiles;
        own_0 += tiles_0;
        own_1 += tiles_1;
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- the range's segments
      Cursor cursor;
      cursor.seek(a, shape, blockIdx.x, lane);
      bool more = true;
      for (int n = 0; more; ++n) {
        const int at = n % kSegments;
        Segment seg{};
        more = cursor.next(a, shape, seg);
        if (n >= kSegments && !__all_sync(0xffffffffu, tree_wait(&sh->seg_empty[at], (n / kSegments - 1) & 1, status, 62))) break;
        if (lane == 0) {
          if (!more) seg.rows = 0;
          sh->seg[at] = seg;
          mbar_arrive(&sh->seg_full[at]);
        }
        __syncwarp();
      }
    }
  } else if (warp < 12) {
    if (kEight) asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
    // ------------------------------------------------------------------ softmax, one thread per row
    const int x = (warp - 4) / 4, quarter = warp & 3, row = quarter * 32 + lane, group = a.group;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const float scale_log2 = a.scale * 1.4426950408889634f;
    const Partials parts = partials_of(a, shape);
    const bool gate_pieces = gate_in_pieces(a);
    // tiles of the range; those of this stream and of the other; meetings of the streams
    int tile_n = 0, own_n = 0, other_n = 0, met = 0;
    bool ok = true;
    int seg_n = 0;
    Segment seg;
    // (at width 256 the second warpgroup only keeps the ring of segments going)
    while (next_segment(sh, seg_n, seg, lane, status)) {
      if (kOneO && x == 1) continue;
      const bool pair = kWide && seg.rows > 128;
      const int tiles = seg.tile1 - seg.tile0, own_row = (pair ? x * 128 : 0) + row;
      const bool live = own_row < seg.rows, warp_live = (pair ? x * 128 : 0) + quarter * 32 < seg.rows;
      const int r = seg.row0 + own_row, node = r / group, head = seg.kv_head * group + r % group;
      const size_t token = static_cast<size_t>(seg.b) * a.nodes + node;
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + (token * a.q_heads + head) * D);
      float row_scale = scale_log2;   // of the scores as the tensor cores return them, into powers of two
      float q_scale = 1.0f;
      if (kEight && warp_live) {
        // fp16 holds the row exactly once its largest value is between 1 and 2 (what is below 2^-14 of that loses bits
        // beyond those that the row's scores have); the scores get the power of two back
        uint32_t largest = 0u;
#pragma unroll 4
        for (int i = 0; i < D / 8; ++i) {
          const uint4 v = live ? q[i] : make_uint4(0u, 0u, 0u, 0u);
          largest = max(largest, max(max(v.x & 0x7fffu, v.y & 0x7fffu), max(v.z & 0x7fffu, v.w & 0x7fffu)));
          largest = max(largest, max(max(v.x & 0x7fff0000u, v.y & 0x7fff0000u), max(v.z & 0x7fff0000u, v.w & 0x7fff0000u)) >> 16);
        }
        const uint32_t e = min(max(largest >> 7, 2u), 252u);
        q_scale = __uint_as_float((254u - e) << 23);
        row_scale = scale_log2 * __uint_as_float(e << 23);
      }
      // ---- the queries, into shared memory or TMEM
      if (warp_live && (pair || x == 0)) {
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint4 v = live ? q[c * 8 + i] : make_uint4(0u, 0u, 0u, 0u);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
          }
          if (kEight) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              w[i] = pack_f16(bf16_lo(w[i]) * q_scale, bf16_hi(w[i]) * q_scale);
          }
          if (!kWide) {
            tmem_st32(lanes + kColQ + c * 32, w);
          } else {
            const uint32_t to = queries + x * kQueryBytes<D, kWide> + c * (128 * 128) + row * 128;
#pragma unroll
            for (int i = 0; i < 8; ++i) sts_b32x4(to + ((i ^ (row & 7)) << 4), w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
          }
        }
        if (!kWide) {
          tmem_wait_st();
          tc_fence_before();
        } else {
          fence_proxy_async();
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->q_full[x == 0 ? 0 : pair ? 1 : 2]);
      // ---- which drafts the row sees: one bit per node
      uint64_t seen_lo = 0, seen_hi = 0;
      if (seg.tile1 * kTile > seg.prefix) {
        if (a.parents) {
          if (live) {
            const int32_t* parents = a.parents + static_cast<size_t>(seg.b) * a.nodes;   // (L1 after the first step)
            for (int i = node; i >= 0;) {
              if (i < 64) seen_lo |= 1ull << i;
              else seen_hi |= 1ull << (i - 64);
              const int up = parents[i];
              if (up < -1 || up >= i) report_status(status, 49, kBadDraft);   // taken as a first token's
              i = up < i ? up : -1;
            }
          }
        } else if (live) {
          seen_lo = node >= 63 ? ~0ull : (2ull << node) - 1;
          seen_hi = node >= 127 ? ~0ull : node >= 64 ? (2ull << (node - 64)) - 1 : 0;
        }
      }
      // ---- the tiles of this stream
      // Weights are w = 2^(score * row_scale - m_used * row_scale), and l their sum.  For 8-bit caches v_used is the largest
      // exponent of the value rows that the row has seen so far and O is kept relative to 2^v_used, so that a weight times its
      // value row's 2^n, which is what enters the product, fits fp16.
      float m_used = -INFINITY, m_true = -INFINITY, l = 0.0f, v_used = kEight ? kSmallest : 0.0f;
      const bool every = pair || kOneO;
      const int own = every ? tiles : (tiles + 1 - x) / 2;
      for (int u = 0; u < own && ok; ++u) {
        // A parity tells the phase that is awaited from its two neighbours only.  Every barrier of a score buffer completes
        // once per tile in it, and a tile's scores are committed behind the products of the buffer's last tile.
        const int j = every ? u : 2 * u + x, t = own_n + u, buffer = buffer_of(t);
        ok = __all_sync(0xffffffffu, tree_wait(&sh->s_full[x][buffer], phase_of(t), status, 56));
        if (!ok) break;
        const uint32_t s_at = lanes + kColS + (kBuffers * x + buffer) * kTile;
        const int slot = (tile_n + j) % (3 * kStages<D, kEight, kWide>);
        const uint32_t k_factor = smem_u32(sh->k_factor[slot]), v_factor = smem_u32(sh->v_factor[slot]);
        const int scaled = kEight && warp_live ? sh->scaled[slot] : 0;   // tiles with drafts, and the rare one that fp16 does not hold
        const int behind = (seg.tile0 + j) * kTile - seg.prefix;   // of the drafts' first slot
        uint64_t seen = ~0ull;
        if (behind > -kTile)
          seen = behind >= 64  ? seen_hi >> (behind - 64)
                 : behind > 0  ? seen_lo >> behind | seen_hi << (64 - behind)
                 : behind == 0 ? seen_lo
                               : seen_lo << -behind | ((1ull << -behind) - 1);
        float v_largest = kEight ? static_cast<float>(sh->v_largest[slot]) : 0.0f;
        if (kEight && behind > -kTile && v_largest > v_used && warp_live) {   // of the drafts' tiles only rows that this one sees count
          if (((static_cast<uint32_t>(seen) & sh->v_top[slot][0]) | (static_cast<uint32_t>(seen >> 32) & sh->v_top[slot][1])) == 0u) {
            uint32_t most = 0u;
#pragma unroll 2
            for (int i = 0; i < kTile; i += 4) {
              const uint4 factor = lds_b32x4(v_factor + i * 4);
              const uint32_t bits = static_cast<uint32_t>(seen >> i);
              most = max(max(most, bits & 1u ? factor.x : 0u), max(bits & 2u ? factor.y : 0u, max(bits & 4u ? factor.z : 0u, bits & 8u ? factor.w : 0u)));
            }
            v_largest = static_cast<float>(static_cast<int>(most >> 23) - 127);
          }
        }
        const float v_tile = fmaxf(v_used, v_largest);
        // Whole tiles' weights are taken times 2^-below; where nothing of that would be left in fp16, or the rows differ, the
        // weights get their factors behind the sum.
        const float below = v_tile - v_largest;
        const bool apart = kEight && ((scaled & kValuesScaled) != 0 || below > kApart);
        const float shift = apart ? 0.0f : below;
        // Half of the tile's keys at a time, in a loop: its code then fits the instruction caches beside the other
        // warps' (straight-line code of 64 columns took twice as long), and the first half's product starts earlier.
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          if (warp_live) {
            if (h == 0) tc_fence_after();
            uint32_t s[32];
            tmem_ld32(s_at + h * 32, s);
            tmem_wait_ld();
            // The weights are taken relative to the maximum so far, so that their way does not lead through this one's; where it
            // has grown too far, the half is done again.
            const auto take_maximum = [&]() {
              float mx[4] = {m_true, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
              for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
              m_true = max3(mx[0], mx[1], fmaxf(mx[2], mx[3]));
            };
            float reference = m_used == -INFINITY ? 0.0f : m_used * row_scale;   // (nothing seen yet: any)
            const bool large = fabsf(reference) > kLargeScore;                   // its rounding would be an exponent
            // (one branch: a warp's way through its tile is what this form waits for)
            if ((scaled & kKeysScaled) != 0 || behind > -kTile || large) {
              if (scaled & kKeysScaled) {
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i] = __float_as_uint(__uint_as_float(s[i]) * lds_f32(k_factor + (h * 32 + i) * 4));
              }
              if (behind > -kTile) {
                const uint32_t bits = static_cast<uint32_t>(seen >> (h * 32));
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (!(bits >> i & 1u)) s[i] = 0xff800000u;
              }
              take_maximum();
              if (large) {
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i] = __float_as_uint(__uint_as_float(s[i]) - m_used);
                reference = 0.0f;
              }
            } else {
              take_maximum();
            }
            reference += shift;
            const uint64_t scale2 = f2_pack(row_scale, row_scale), neg2 = f2_pack(-reference, -reference);
            uint64_t sum2[2] = {0ull, 0ull};
            uint32_t packed[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float p0, p1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), scale2, neg2), p0, p1);
              p0 = fast_exp2(p0);
              p1 = fast_exp2(p1);
              sum2[(i >> 1) & 1] = f2_add(sum2[(i >> 1) & 1], f2_pack(p0, p1));
              if (kEight) {   // (kept apart from the products with the rows' factors below)
                s[i] = __float_as_uint(p0);
                s[i + 1] = __float_as_uint(p1);
              } else {
                packed[i / 2] = pack_bf16(p0, p1);
              }
            }
            const bool grow = (m_true - m_used) * row_scale > kRescale;
            if (__any_sync(0xffffffffu, grow || v_tile > v_used || apart)) {
              if (!kEight || __any_sync(0xffffffffu, grow || v_tile > v_used)) {
                const float less = grow ? (m_used - m_true) * row_scale : 0.0f, factor = fast_exp2(less + (v_used - v_tile));
                if (grow) m_used = m_true;
                v_used = v_tile;
                l *= kEight ? fast_exp2(less) : factor;
                if (u > 0 || h == 1) {
                  // every product into this O must have ended: the first half's, or the previous tile's second
                  ok = __all_sync(0xffffffffu, tree_wait(h ? &sh->pv_half[x][buffer] : &sh->pv_done[x][buffer_of(t - 1)], phase_of(h ? t : t - 1), status, 57));
                  if (!ok) break;
                  tc_fence_after();
#pragma unroll 1
                  for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16];
                    const uint32_t o_at = lanes + x * kColO1 + c * 16;
                    tmem_ld16(o_at, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                    tmem_st16(o_at, o);
                  }
                  tmem_wait_st();
                }
                --h;
                continue;
              }
              if (apart) {
                const float down = scaled & kValuesScaled ? power_of_two(-v_tile) : 0.0f;
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                  const uint4 factor = lds_b32x4(v_factor + (h * 32 + i) * 4);
                  s[i] = __float_as_uint(__uint_as_float(s[i]) * down * __uint_as_float(factor.x));
                  s[i + 1] = __float_as_uint(__uint_as_float(s[i + 1]) * down * __uint_as_float(factor.y));
                  s[i + 2] = __float_as_uint(__uint_as_float(s[i + 2]) * down * __uint_as_float(factor.z));
                  s[i + 3] = __float_as_uint(__uint_as_float(s[i + 3]) * down * __uint_as_float(factor.w));
                }
              }
            }
            if (kEight) {
#pragma unroll
              for (int i = 0; i < 32; i += 2) packed[i / 2] = pack_f16(__uint_as_float(s[i]), __uint_as_float(s[i + 1]));
            }
            tmem_st16(s_at + h * 16, packed);
            float a0, a1, b0, b1;
            f2_unpack(sum2[0], a0, a1);
            f2_unpack(sum2[1], b0, b1);
            l += kEight ? ((a0 + a1) + (b0 + b1)) * power_of_two(shift) : (a0 + a1) + (b0 + b1);
            tmem_wait_st();
            tc_fence_before();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(h ? &sh->p_full[x][buffer] : &sh->p_half[x][buffer]);
        }
      }
      if (!ok) break;
      const bool merged = !pair && !kOneO;
      tile_n += tiles;
      own_n += own;
      other_n += every ? tiles : tiles - own;
      // this stream's last product
      if (own > 0) ok = __all_sync(0xffffffffu, tree_wait(&sh->pv_done[x][buffer_of(own_n - 1)], phase_of(own_n - 1), status, 58));
      if (!ok) break;
      tc_fence_after();
      // ---- read-out: rows of one stream, or the two streams' halves of the keys merged, half of the channels each
      // log2 units from here: sums relative to 2^m, O to 2^(m + v)
      float m = m_used == -INFINITY ? m_used : m_used * row_scale, f0 = 1.0f, f1 = 0.0f, v = v_used;
      bool both = false;
      if (merged) {
        sh->ml[x][row] = make_float2(m, l);
        if (kEight) sh->unit[x][row] = v_used;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->ml_full);
        ok = __all_sync(0xffffffffu, tree_wait(&sh->ml_full, met & 1, status, 59));
        // (the other stream has seen its last product end before it arrived there: this returns at once)
        if (ok && (x == 1 || tiles > 1))
          ok = __all_sync(0xffffffffu, tree_wait(&sh->pv_done[1 - x][buffer_of(other_n - 1)], phase_of(other_n - 1), status, 58));
        if (!ok) break;
        tc_fence_after();
        const float2 one = sh->ml[0][row], two = sh->ml[1][row];
        both = tiles > 1;
        m = both ? fmaxf(one.x, two.x) : one.x;
        const float m_safe = m == -INFINITY ? 0.0f : m;
        f0 = fast_exp2(one.x - m_safe);
        f1 = both ? fast_exp2(two.x - m_safe) : 0.0f;
        l = both ? one.y * f0 + two.y * f1 : one.y * f0;
        if (kEight) {   // O in the larger of the two units
          const float v0 = sh->unit[0][row], v1 = both ? sh->unit[1][row] : v0, step = (two.x - one.x) + (v1 - v0);
          const bool second = both && two.x != -INFINITY && step > 0.0f;
          f0 = second ? fast_exp2(-step) : 1.0f;
          f1 = second ? 1.0f : both && two.x != -INFINITY ? fast_exp2(step) : 0.0f;
          v = second ? v1 + (two.x - m) : one.x == -INFINITY ? v0 : v0 + (one.x - m);
        }
      }
      if (warp_live) {
        const int slot = 2 * blockIdx.x + seg.slot;
        const float drop = kEight && !seg.whole ? part_drop(l) : 0.0f;
        float inverse = seg.whole ? (l == 0.0f ? 0.0f : 1.0f / l) : power_of_two(-drop);
        if (kEight) {   // O's unit, with either factor: beside small values the product of both might not be a normal number
          const float unit = exp2f(v);
          f0 *= v < -60.0f ? unit : 1.0f;
          f1 *= v < -60.0f ? unit : 1.0f;
          inverse *= v < -60.0f ? 1.0f : unit;
        }
        float* acc = parts.acc + (static_cast<size_t>(slot) * parts.rows + own_row) * D;
        const int c0 = merged ? x * (D / 32) : 0, c1 = merged ? c0 + D / 32 : D / 16;
#pragma unroll 1
        for (int c = c0; c < c1; ++c) {
          uint32_t o[16];
          tmem_ld16(lanes + (merged ? 0u : x * kColO1) + c * 16, o);
          if (both) {
            uint32_t o2[16];
            tmem_ld16(lanes + kColO1 + c * 16, o2);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f0 + __uint_as_float(o2[i]) * f1);
          } else {
            tmem_wait_ld();
            if (kEight) {
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f0);
            }
          }
          if (!live) {
            // (a lane without a row only takes part in the reads)
          } else if (seg.whole) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(o[8 * h + i]) * inverse;
              store_out8(a, token, head, c * 16 + 8 * h, v, gate_pieces);
            }
          } else {
            if (kEight) {
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * inverse);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
              reinterpret_cast<uint4*>(acc + c * 16)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
          __syncwarp();
        }
        if (live && (x == 0 || pair)) {
          if (!seg.whole) parts.ml[static_cast<size_t>(slot) * parts.rows + own_row] = make_float2(m + drop, l * power_of_two(-drop));
          else if (a.lse) a.lse[token * a.q_heads + head] = (m == -INFINITY ? 0.0f : m * 0.6931471805599453f) + logf(l);
        }
        tc_fence_before();
      }
      if (merged) {   // both have read both accumulators (and sums) before either stream's next product
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->o_read);
        ok = __all_sync(0xffffffffu, tree_wait(&sh->o_read, met++ & 1, status, 60));
        if (!ok) break;
      }
    }
  } else {
    // ------------------------------------------------------------------ loads, widening
    if (warp < 16) {
      if (kEight) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
      load_tiles<D, kEight, kWide>(a, map_k, map_v, box, sh, kEight ? raw_k : k_ring, kEight ? raw_v : v_ring, warp - 12, lane);
      asm volatile("cp.async.wait_all;" ::: "memory");   // (landed long ago unless a wait ran out)
    } else {
      if constexpr (kEight) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        widen_tiles<D, kWide>(sh, warp < 20 ? raw_k : raw_v, warp < 20 ? k_ring : v_ring, status, warp & 3, lane, warp >= 20);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

constexpr LineShape line_shape(int dim) { return {6, kUnitTiles, dim == 256 ? 7 : 8, kMaxCtas, 1}; }

template <int D, bool kEight, bool kWide>
cudaError_t launch_kernel(cudaStream_t stream, const TreeArgs& a) {
  constexpr LineShape shape = line_shape(D);
  static_assert(1 << shape.tile_shift == kTile && 1 << shape.rows_shift == group_rows(D), "line");
  const long long units = static_cast<long long>(a.batch) * a.kv_heads * ((a.nodes * a.group + group_rows(D) - 1) / group_rows(D));
  const long long tiles = units * ((static_cast<long long>(a.max_prefix) + a.nodes + kTile - 1) / kTile);
  constexpr int kBytes = kRingBytes<D, kEight, kWide> + 2 * kQueryBytes<D, kWide> + static_cast<int>(sizeof(Shared<D, kEight, kWide>)) + 1024;
  static_assert(kBytes <= 227 * 1024, "shared memory");
  using S = Shared<D, kEight, kWide>;
  static_assert(offsetof(S, k_factor) % 16 == 0 && offsetof(S, ml) % 8 == 0 && alignof(S) == 16, "alignment");
  // tokens of a tiled copy; 0: rows by the lanes' own copies
  const int box = !kBoxes<D, kEight> ? 0 : tree_pool_fits(a, kHalf) ? kHalf : tree_pool_fits(a, kHalf / 2) ? kHalf / 2 : 0;
  CUtensorMap map_k{}, map_v{};
  if (box > 0 && (!tree_pool_map(&map_k, a.pool.k, a, box, kEight ? D : 64, kEight ? 0 : 128) || !tree_pool_map(&map_v, a.pool.v, a, box, kEight ? D : 64, kEight ? 0 : 128)))
    return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(tree_decode_sm100<D, kEight, kWide>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
  if (e != cudaSuccess) return e;
  tree_decode_sm100<D, kEight, kWide><<<static_cast<unsigned>(tiles < kMaxCtas ? tiles : kMaxCtas), kThreads<kEight>, kBytes, stream>>>(map_k, map_v, box, a, shape);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return tree_decode_merge(stream, a, shape);
}

template <int D, bool kEight>
cudaError_t launch(cudaStream_t stream, const TreeArgs& a) {
  if constexpr (D < 256) {
    if (a.nodes * a.group > 128) return launch_kernel<D, kEight, true>(stream, a);
  }
  return launch_kernel<D, kEight, false>(stream, a);
}

}  // namespace

bool tree_decode_tc_supported(const TreeArgs& a) { return line_fits(a, line_shape(a.dim)); }

size_t tree_decode_tc_workspace_bytes(int nodes, int q_heads, int kv_heads, int dim) {
  return line_workspace_bytes(line_shape(dim), nodes, q_heads, kv_heads, dim);
}

cudaError_t tree_decode_tc(cudaStream_t stream, const TreeArgs& a) {
  const bool eight = a.pool.store == kStoreE4m3;
  if (a.dim == 64) return eight ? launch<64, true>(stream, a) : launch<64, false>(stream, a);
  if (a.dim == 128) return eight ? launch<128, true>(stream, a) : launch<128, false>(stream, a);
  return eight ? launch<256, true>(stream, a) : launch<256, false>(stream, a);
}

}  // namespace pluto
