// Attention of drafted tokens over a bf16 or 8-bit cache where few rows share a KV head (nodes * query heads per KV head
// at most 16, at width 256 at most 8): single tokens and short drafts.  The cache is read once; the arithmetic has to stay
// out of the way:
//   S^T = K Q^T    tokens x rows, mma.sync m16n8k16 with fp32 accumulation: sixteen tokens are the 16-row operand
//   O^T += V^T P^T channels x rows: sixteen channels are, the rows are the columns, eight to a product
// so that up to eight rows waste nothing (rows as the 16-row operand took twice the products).
//
// A warp works alone: it streams its range of the line (tree_line.cuh) in steps of sixteen tokens through a ring of its
// own in shared memory, so its main loop meets no other warp.  One lane fetches a step with tiled TMA copies over a
// map of the page pool (column, KV head, token in page, page); a step lies in one page, which is what limits the
// kernel to page sizes that sixteen divides and to caches of one page per sequence.  The queries of a unit come
// through the ring as a step of their own.  Neighbouring warps take the KV heads of the same tokens, whose rows
// neighbour in memory: 24 ragged sequences, 40 and 8 heads of 128, 8-bit: 54 us, 66 with ranges head by head.
//
// The codes of an 8-bit cache become MMA operands in registers, one instruction per two codes and exact.  The order of
// the channels in a product is free as long as both operands share it, so a lane takes whole 16-byte pieces: of the
// keys the pieces of its rows, of the values the piece of its channels from four rows, paired by byte permutes.  The
// rows' powers of two stay out of the products: a key's multiplies its scores, a value's its weights behind their
// sum, relative to the largest so far so that the products fit fp16 (P carries 11 bits).  Over bf16 caches P enters as a bf16 part and
// its bf16 remainder, 16 bits, as in gqa_decode.cu.  P^T leaves the score layout by movmatrix, and a lane compares its
// scores with the reference of their rows by itself: the maximum is reduced over lanes only when one has to move.
//
// Measured (B200, 16 sequences of 8000 tokens, 40 and 8 heads of 128, one token): bf16 90 us, 5.8 TB/s of cache; 8-bit
// 56 us, 4.7 TB/s.  There, three warps per scheduler issue in half of the cycles, the rest are fixed latencies between dependent
// instructions, and DRAM stands at 61 %.  Four CTAs per SM at 128 registers took 60.
#include "tree_line.cuh"

namespace pluto {
namespace {

constexpr int kTile = 16;          // tokens of a step
constexpr int kWarps = 4;
constexpr float kRescale = 8.0f;   // the accumulator is rescaled when the maximum has grown by more than 2^8
constexpr float kSmallest = -118.0f;   // exponent of the value rows from which smaller ones are taken for as large: weights of up
                                       // to 2^8 times 2^118 stay finite

template <int D, bool kEight>
constexpr int kRowBytes = D * (kEight ? 1 : 2);
template <int D, bool kEight>
constexpr int kStageBytes = 2 * kTile * kRowBytes<D, kEight>;   // keys, then values
// CTAs per SM, and steps in the ring of a warp: as many warps as their registers allow, and 96 KB or more in flight per SM
template <int D, bool kEight>
constexpr int kCtas = D == 256 ? (kEight ? 2 : 1) : D == 128 ? 3 : 4;
template <int D, bool kEight>
constexpr int kStages = D == 256 ? 3 : D == 128 ? (kEight ? 4 : 2) : (kEight ? 6 : 3);
constexpr int kSegments = 8;   // of a warp's range that its copies are ahead by, at most (a step each)

// What a warp has beside its ring.  Scale bytes come as the aligned words that hold them, [0]: keys, [1]: values, with the
// byte's place in the word.
template <int kS, bool kEight>
struct WarpState {
  uint64_t full[kS];
  Cursor ahead;
  Segment segments[kSegments];
  uint32_t words[kEight ? kS : 1][32];
  uint8_t places[kEight ? kS : 1][32];
};

__device__ __forceinline__ void copy4(uint32_t to, const void* from, bool there) {   // zero where it is not
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void arrive_behind_copies(uint64_t* bar) {   // when this thread's copies so far have landed
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void bulk_load_at(uint32_t to, const void* from, uint32_t bytes, uint64_t* bar) {   // all multiples of 16
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes),
               "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint32_t halves_of(uint32_t codes) {   // two codes in the low 16 bits -> two fp16
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(codes)));
  return r;
}
// d += a b: a 16 x 16, b 16 x 8
template <bool kEight>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (kEight)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {   // of an 8 x 8 matrix of 16-bit values, a row per four lanes
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ bool not_finite(uint32_t pair) {
  return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u;
}

// Byte offset of 16-byte piece c of row r in a tile: slabs of 128 bytes (64 where a row has no more), swizzled by the copies,
// so that the reads below, which take the same piece of several rows, hit all banks.
template <int kBytes>
__device__ __forceinline__ uint32_t piece_at(int r, int c) {
  return kBytes == 64 ? r * 64 + ((c ^ (r >> 1 & 3)) << 4) : (c / 8) * (kTile * 128) + r * 128 + (((c ^ r) & 7) << 4);
}

template <int D, bool kEight, bool kHalf>   // kHalf: at most eight rows
__global__ void __launch_bounds__(kWarps * 32, kCtas<D, kEight>) tree_decode_mma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, TreeArgs a, LineShape shape) {
  constexpr int kBytes = kRowBytes<D, kEight>, kPieces = kBytes / 16, kS = kStages<D, kEight>;
  constexpr int kN = kHalf ? 1 : 2, kR = 2 * kN;        // blocks of eight rows; rows of a lane: 8 n + 2 t4 + e
  constexpr int kChunks = kPieces < 4 ? 1 : kPieces / 4, kSteps = kEight ? 4 : 2;   // pieces of a key row per lane, k steps per piece
  constexpr int kBlocks = D / 16;                       // accumulator blocks of sixteen channels
  static_assert(kChunks * kSteps == D / 16, "channels");
  using State = WarpState<kS, kEight>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = uniform_warp_index(), lane = threadIdx.x % 32, quad = lane / 4, t4 = lane % 4;
  const uint32_t ring = base + warp * kS * kStageBytes<D, kEight>;
  State* own = reinterpret_cast<State*>(smem_raw + (base - smem_u32(smem_raw)) + kWarps * kS * kStageBytes<D, kEight>) + warp;
  uint32_t* status = a.pool.status;
  const int page_shift = (a.pool.page_size & (a.pool.page_size - 1)) == 0 ? __ffs(a.pool.page_size) - 1 : -1;
  const int group = a.group;
  const float scale_log2 = a.scale * 1.4426950408889634f;
  const Partials parts = partials_of(a, shape);
  const bool gate_pieces = gate_in_pieces(a);
  pdl_launch_dependents();   // the merge may be placed as SMs free up; it waits for this grid's end

  const int worker = blockIdx.x * kWarps + warp;
  if (lane == 0) {
    for (int i = 0; i < kS; ++i) mbar_init(&own->full[i], kEight ? 33 : 1);
    mbar_fence_init();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  // ---- copies: the next step to issue, kS - 1 ahead of the one that is worked on; what says which one lives in shared
  // memory (the registers are the products')
  {
    Cursor cursor;
    cursor.seek(a, shape, worker, lane);
    if (lane == 0) own->ahead = cursor;
  }
  __syncwarp();
  bool started = false;
  int tile = 0, last = 0, page = 0, inside = 0, to_slot = 0, listed = 0;   // of the next step: its tile, the segment's end, its page and place in it, its slot
  int load_b = 0, load_head = 0, load_end = 0, load_rows = 0;              // of the segment: sequence, KV head, tokens, rows still to be fetched
  const unsigned pages = a.pool.table ? a.pool.num_pages : a.batch, blocks = a.pool.table ? a.pool.max_blocks : 1;
  const uint8_t* scales = lane < kTile ? a.pool.k_scales : a.pool.v_scales;   // lanes 0-15: the keys', 16-31: the values'
  const uint32_t scale_page = static_cast<uint32_t>(a.pool.scale_page), scale_token = static_cast<uint32_t>(a.pool.scale_token);
  const auto issue = [&]() {   // (the first call only finds the first step)
    if (started) {
      if (tile >= last) return;
      const int slot_now = to_slot;
      to_slot = to_slot + 1 == kS ? 0 : to_slot + 1;
      if (load_rows > 0) {   // the queries come first, through the ring as well: a load would wait behind all copies of the SM
        const int nodes = load_rows / group, bytes = group * D * 2;
        if (lane == 0) mbar_expect_tx(&own->full[slot_now], nodes * bytes);
        __syncwarp();
        if (lane < nodes)
          bulk_load_at(ring + slot_now * kStageBytes<D, kEight> + lane * bytes,
                    static_cast<const __nv_bfloat16*>(a.q) + ((static_cast<size_t>(load_b) * a.nodes + lane) * a.q_heads + load_head * group) * D, bytes,
                    &own->full[slot_now]);
        if (kEight) mbar_arrive(&own->full[slot_now]);
        load_rows = 0;
        return;
      }
      if (static_cast<unsigned>(page) >= pages) {
        report_status(status, 48, kBadPage);   // (a slot past the pages was reported as such before)
        page = -1;                             // the copies read zeros there
      }
      if (lane == 0) {
        const uint32_t to = ring + slot_now * kStageBytes<D, kEight>;
        constexpr int kSlabs = kBytes == 64 ? 1 : kBytes / 128, kColumns = D / kSlabs, kSlab = kTile * kBytes / kSlabs;
        mbar_expect_tx(&own->full[slot_now], kStageBytes<D, kEight>);
#pragma unroll
        for (int i = 0; i < kSlabs; ++i) {
          tma_load_4d_at(to + i * kSlab, &map_k, i * kColumns, load_head, inside, page, &own->full[slot_now]);
          tma_load_4d_at(to + kTile * kBytes + i * kSlab, &map_v, i * kColumns, load_head, inside, page, &own->full[slot_now]);
        }
      }
      if (kEight) {
        const int row = lane % kTile;
        const bool there = page >= 0 && tile * kTile + row < load_end;
        const uint8_t* byte = scales + load_head;
        if (there) byte += static_cast<uint64_t>(static_cast<uint32_t>(page)) * scale_page + static_cast<uint64_t>(static_cast<uint32_t>(inside + row)) * scale_token;
        const uintptr_t at = reinterpret_cast<uintptr_t>(byte);
        own->places[slot_now][lane] = static_cast<uint8_t>(at & 3u);
        copy4(smem_u32(&own->words[slot_now][lane]), reinterpret_cast<const void*>(at & ~static_cast<uintptr_t>(3)), there);
        arrive_behind_copies(&own->full[slot_now]);
      }
      ++tile;
    }
    started = true;
    if (tile >= last) {   // the next segment
      Cursor cursor = own->ahead;
      Segment load{};
      const bool more = cursor.next(a, shape, load);   // (rows 0 behind the last)
      __syncwarp();
      if (lane == 0) {
        own->ahead = cursor;
        own->segments[listed % kSegments] = load;
      }
      __syncwarp();
      ++listed;
      tile = more ? load.tile0 : 0;
      last = more ? load.tile1 : 0;
      load_b = load.b;
      load_head = load.kv_head;
      load_end = load.prefix + load.count;
      if (blocks == 1u && load_end > a.pool.page_size) {   // the only page may end inside a step: the copies read zeros behind it,
        report_status(status, 48, kBadLength);             // and no scale is read there
        load_end = a.pool.page_size;
      }
      if (!more) return;
      load_rows = load.rows;
    }
    const int t0 = tile * kTile, block = page_shift >= 0 ? t0 >> page_shift : t0 / a.pool.page_size;
    inside = t0 - block * a.pool.page_size;
    if (static_cast<unsigned>(block) >= blocks) {
      report_status(status, 48, kBadLength);
      page = -1;
    } else {
      page = a.pool.table ? a.pool.table[static_cast<size_t>(load_b) * a.pool.max_blocks + block] : load_b;
    }
  };
  // A wait that runs out is reported and the warp goes on: the results are worth nothing then, but every copy has been waited
  // for when its memory is given up.
  // One loop over the steps of the range, so that every piece of code is there once: a range of few steps is as long as
  // the fetching of its instructions takes.
  Segment seg{};
  int primed = 0, slot = 0, round = 0, n = 0, j = 0;   // slot and round of the ring
  uint32_t qf[D / 16][kN][2], seen[kR];
  float row_scale[kR], m_used[kR], v_used[kEight ? kR : 1], l[kR], o[kBlocks][kN][4], v_low = 0.0f;
#pragma unroll 1
  while (true) {
    issue();
    if (primed < kS) {   // (a call without a step, and steps but one of the ring)
      ++primed;
      continue;
    }
    if (j >= seg.tile1) {   // (the first time: 0 >= 0)
    if (seg.rows > 0) {
    // ---- the unit's part; its result where the whole unit is here
    const int part = 2 * worker + seg.slot;
    float* acc = parts.acc + static_cast<size_t>(part) * parts.rows * D;
#pragma unroll
    for (int i = 0; i < kR; ++i) {
#pragma unroll
      for (int lanes = 4; lanes < 32; lanes *= 2) l[i] += __shfl_xor_sync(0xffffffffu, l[i], lanes);
      const int nb = i / 2, e = i % 2, r = nb * 8 + 2 * t4 + e;
      if (r >= seg.rows) continue;
      float* to = acc + r * D;
      float drop = 0.0f;
      if constexpr (kEight) {
        constexpr int kWidth = D == 64 ? 8 : 16;   // neighbouring channels of a lane
        drop = part_drop(l[i]);
        const float down = power_of_two(-drop), up = power_of_two(v_used[i]);
        l[i] *= down;
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) {
          o[m][nb][e] = o[m][nb][e] * down * up;
          o[m][nb][2 + e] = o[m][nb][2 + e] * down * up;
        }
#pragma unroll
        for (int set = 0; set < (D == 256 ? 2 : 1); ++set)
#pragma unroll
          for (int k = 0; k < kWidth; k += 4) {
            const int m = set * 8 + k / 2;
            *reinterpret_cast<float4*>(to + set * 128 + quad * kWidth + k) = make_float4(o[m][nb][e], o[m][nb][2 + e], o[m + 1][nb][e], o[m + 1][nb][2 + e]);
          }
      } else {
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) {
          to[m * 16 + quad] = o[m][nb][e];
          to[m * 16 + 8 + quad] = o[m][nb][2 + e];
        }
      }
      if (quad == 0) parts.ml[static_cast<size_t>(part) * parts.rows + r] = make_float2(m_used[i] + drop, l[i]);
    }
    if (seg.whole) {   // (through the slot that the warp has anyway: rows in the order of memory, and one piece of code)
      __syncwarp();
      constexpr int kEights = D / 8;
#pragma unroll 1
      for (int i = lane; i < seg.rows * kEights; i += 32) {
        const int r = i / kEights, d = i % kEights * 8, node = r / group, head = seg.kv_head * group + r % group;
        const size_t token = static_cast<size_t>(seg.b) * a.nodes + node;
        const float2 ml = parts.ml[static_cast<size_t>(part) * parts.rows + r];
        const float inverse = ml.y == 0.0f ? 0.0f : 1.0f / ml.y;
        const float4 u = *reinterpret_cast<const float4*>(acc + r * D + d), v = *reinterpret_cast<const float4*>(acc + r * D + d + 4);
        const float x[8] = {u.x * inverse, u.y * inverse, u.z * inverse, u.w * inverse, v.x * inverse, v.y * inverse, v.z * inverse, v.w * inverse};
        store_out8(a, token, head, d, x, gate_pieces);
        if (d == 0 && a.lse) a.lse[token * a.q_heads + head] = (ml.x == -INFINITY ? 0.0f : ml.x * 0.6931471805599453f) + logf(ml.y);
      }
      __syncwarp();
    }
    }
    seg = own->segments[n++ % kSegments];
    if (seg.rows == 0) break;
    j = seg.tile0;
    tree_wait(&own->full[slot], round & 1, status, 50);
    __syncwarp();
    const uint32_t rows_at = ring + slot * kStageBytes<D, kEight>;
    // ---- the queries: B fragments of row 8 nb + quad, channels in the order of the keys' pieces
    float of_row[kN];       // scale of the row's scores
    uint32_t bits_of[kN];   // which drafts it sees: one bit per node
#pragma unroll
    for (int nb = 0; nb < kN; ++nb) {
      const int r = nb * 8 + quad;
      const bool live = r < seg.rows;
      uint32_t largest = 0u;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int c = kPieces < 8 ? t4 : 2 * t4 + (i & 1) + 8 * (i >> 1);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          const uint64_t w = live ? lds_b64(rows_at + (r * D + c * (kEight ? 16 : 8) + 4 * k) * 2) : 0ull;
          const uint32_t lo = static_cast<uint32_t>(w), hi = static_cast<uint32_t>(w >> 32);
          qf[i * kSteps + k][nb][0] = lo;
          qf[i * kSteps + k][nb][1] = hi;
          largest = max(largest, max(max(lo & 0x7fffu, hi & 0x7fffu), max(lo & 0x7fff0000u, hi & 0x7fff0000u) >> 16));
        }
      }
      of_row[nb] = scale_log2;
      if (kEight) {
        // fp16 holds the row exactly once its largest value is between 1 and 2 (what is below 2^-14 of that loses bits
        // beyond those that the row's scores have); the scores get the power of two back
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        const uint32_t e = min(max(largest >> 7, 2u), 252u);
        const float down = __uint_as_float((254u - e) << 23);
        of_row[nb] = scale_log2 * __uint_as_float(e << 23);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t& w = qf[k][nb][u];
            w = pack_f16(bf16_lo(w) * down, bf16_hi(w) * down);
          }
      }
      bits_of[nb] = 0u;
      if (seg.tile1 * kTile > seg.prefix && live) {
#pragma unroll 1
        for (int i = r / group; i >= 0;) {
          bits_of[nb] |= 1u << i;
          const int up = a.parents ? a.parents[static_cast<size_t>(seg.b) * a.nodes + i] : i - 1;
          if (up < -1 || up >= i) report_status(status, 49, kBadDraft);   // taken as a first token's
          i = up < i ? up : -1;
        }
      }
    }
    __syncwarp();
    // Weights are 2^(score * row_scale - m_used).  For 8-bit caches v_used is the largest exponent of the value rows seen so far
    // and O is kept relative to 2^v_used, so that a weight times its value row's 2^n, which is what enters the product, fits fp16.
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      row_scale[i] = __shfl_sync(0xffffffffu, of_row[i / 2], (2 * t4 + i % 2) * 4);
      seen[i] = __shfl_sync(0xffffffffu, bits_of[i / 2], (2 * t4 + i % 2) * 4);
      m_used[i] = -INFINITY;
      if (kEight) v_used[i] = kSmallest;
      l[i] = 0.0f;
    }
    if (kEight) v_low = kSmallest;
#pragma unroll
    for (int m = 0; m < kBlocks; ++m)
#pragma unroll
      for (int nb = 0; nb < kN; ++nb)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[m][nb][i] = 0.0f;
    if (++slot == kS) {
      slot = 0;
      ++round;
    }
    continue;
    }
      tree_wait(&own->full[slot], round & 1, status, 50);
      __syncwarp();
      const uint32_t k_tile = ring + slot * kStageBytes<D, kEight>, v_tile = k_tile + kTile * kBytes;
      const int behind = j * kTile - seg.prefix;   // of the drafts' first slot
      const bool border = behind > -kTile;         // the step holds drafts, or ends the sequence
      uint32_t scale = 127u;                       // lanes 0-15: of the keys, 16-31: of the values
      if (kEight) scale = own->words[slot][lane] >> (8 * own->places[slot][lane]) & 0xffu;
      uint32_t hidden = 0u;                        // tokens whose value row is not finite, among drafts that not every row sees
      if (border) {
        // Rows behind the last draft hold anything.  Neither they nor value rows that are not finite may meet the zero
        // weights of the rows that do not see them: they become zeros, and those that see the latter get NaN scores.
        const int live = seg.count - behind;
        uint32_t clear = live < kTile ? 0xffffu << live & 0xffffu : 0u;
        if (seg.count > 1) {
          if (kEight) {
            hidden = __ballot_sync(0xffffffffu, lane >= kTile && lane - kTile + behind >= 0 && scale == 255u) >> kTile;
          } else {
#pragma unroll 2
            for (int i = 0; i < kPieces / 2; ++i) {
              const int row = i * (32 / kPieces) + lane / kPieces;
              const uint4 w = lds_b32x4(v_tile + piece_at<kBytes>(row, lane % kPieces));
              if (row + behind >= 0 && (not_finite(w.x) || not_finite(w.y) || not_finite(w.z) || not_finite(w.w))) hidden |= 1u << row;
            }
            hidden = __reduce_or_sync(0xffffffffu, hidden);
          }
          hidden &= ~clear;
          clear |= hidden;
        }
        if (clear) {
#pragma unroll 1
          for (int i = lane; i < kTile * kPieces; i += 32)
            if (clear >> (i / kPieces) & 1u) sts_b32x4(v_tile + piece_at<kBytes>(i / kPieces, i % kPieces), 0u, 0u, 0u, 0u);
          fence_proxy_async();   // (the slot's next copies write behind these stores)
          __syncwarp();
        }
      }
      // factors: a key row that is not finite makes its scores NaN; the codes of such a value row are NaN, or zeros here
      const float own_factor = scale == 255u ? (lane < kTile ? __uint_as_float(0x7fc00000u) : 1.0f) : e8m0_value(scale);
      // ---- S^T = K Q^T: sixteen tokens by the rows, two accumulators each (the chain of products is what a step waits for)
      float st[kN][4] = {}, st2[kN][4] = {};
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int c = kPieces < 8 ? t4 : 2 * t4 + (i & 1) + 8 * (i >> 1);
        const uint4 w0 = lds_b32x4(k_tile + piece_at<kBytes>(quad, c)), w1 = lds_b32x4(k_tile + piece_at<kBytes>(8 + quad, c));
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          uint32_t a0, a1, a2, a3;
          if (kEight) {
            const uint32_t lo = k == 0 ? w0.x : k == 1 ? w0.y : k == 2 ? w0.z : w0.w, hi = k == 0 ? w1.x : k == 1 ? w1.y : k == 2 ? w1.z : w1.w;
            a0 = halves_of(lo);
            a1 = halves_of(hi);
            a2 = halves_of(lo >> 16);
            a3 = halves_of(hi >> 16);
          } else {
            a0 = k == 0 ? w0.x : w0.z;
            a1 = k == 0 ? w1.x : w1.z;
            a2 = k == 0 ? w0.y : w0.w;
            a3 = k == 0 ? w1.y : w1.w;
          }
#pragma unroll
          for (int nb = 0; nb < kN; ++nb) mma<kEight>(k & 1 ? st2[nb] : st[nb], a0, a1, a2, a3, qf[i * kSteps + k][nb][0], qf[i * kSteps + k][nb][1]);
        }
      }
      // ---- the tokens of this lane: quad and quad + 8; its rows: 8 nb + 2 t4 + e
      float k_factor[2] = {1.0f, 1.0f}, v_factor[2] = {1.0f, 1.0f};
      if (kEight) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          k_factor[u] = __shfl_sync(0xffffffffu, own_factor, 8 * u + quad);
          v_factor[u] = __shfl_sync(0xffffffffu, own_factor, kTile + 8 * u + quad);
        }
      }
      float x[kR][2];
#pragma unroll
      for (int i = 0; i < kR; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          x[i][u] = (st[i / 2][2 * u + i % 2] + st2[i / 2][2 * u + i % 2]) * row_scale[i];
          if (kEight) x[i][u] *= k_factor[u];
        }
      if (border) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int token = 8 * u + quad, draft = token + behind;
#pragma unroll
          for (int i = 0; i < kR; ++i) {
            if (hidden >> token & 1u) x[i][u] = __uint_as_float(0x7fc00000u);
            if (draft >= 0 && (draft >= 16 || !(seen[i] >> draft & 1u))) x[i][u] = -INFINITY;
          }
        }
      }
      // ---- the references are moved rarely: when a score, or the exponent of a value row, has grown beyond them
      const float v_power[2] = {static_cast<float>(static_cast<int>(__float_as_uint(v_factor[0]) >> 23) - 127),
                                static_cast<float>(static_cast<int>(__float_as_uint(v_factor[1]) >> 23) - 127)};
      bool move = kEight && fmaxf(v_power[0], v_power[1]) > v_low;
#pragma unroll
      for (int i = 0; i < kR; ++i) move = move || fmaxf(x[i][0], x[i][1]) - m_used[i] > kRescale;
      if (__any_sync(0xffffffffu, move)) {
        if (kEight) v_low = INFINITY;
#pragma unroll
        for (int i = 0; i < kR; ++i) {
          float m = fmaxf(x[i][0], x[i][1]), v = 0.0f;
          if (kEight) {
            v = v_used[i];
            if (x[i][0] != -INFINITY) v = fmaxf(v, v_power[0]);   // (of the rows that are seen)
            if (x[i][1] != -INFINITY) v = fmaxf(v, v_power[1]);
          }
#pragma unroll
          for (int lanes = 4; lanes < 32; lanes *= 2) {
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, lanes));
            if (kEight) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, lanes));
          }
          const bool grow = m - m_used[i] > kRescale;
          const float less = grow ? m_used[i] - m : 0.0f, factor = fast_exp2(kEight ? less + (v_used[i] - v) : less);
          if (grow) m_used[i] = m;
          l[i] *= kEight ? fast_exp2(less) : factor;
          if (kEight) {
            v_used[i] = v;
            v_low = fminf(v_low, v);
          }
#pragma unroll
          for (int k = 0; k < kBlocks; ++k) {
            o[k][i / 2][i % 2] *= factor;
            o[k][i / 2][2 + i % 2] *= factor;
          }
        }
      }
      uint32_t p[kN][2], rest[kN][2];   // [rows][tokens 0-7, 8-15]: B fragments
#pragma unroll
      for (int nb = 0; nb < kN; ++nb)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float w[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int i = 2 * nb + e;
            w[e] = fast_exp2(x[i][u] - (m_used[i] == -INFINITY ? 0.0f : m_used[i]));   // (nothing seen yet: any)
            l[i] += w[e];
            if (kEight) w[e] = w[e] * power_of_two(-v_used[i]) * v_factor[u];
          }
          if (kEight) {
            p[nb][u] = transposed(pack_f16(w[0], w[1]));
          } else {
            const uint32_t most = pack_bf16(w[0], w[1]);
            p[nb][u] = transposed(most);
            rest[nb][u] = transposed(pack_bf16(w[0] - bf16_lo(most), w[1] - bf16_hi(most)));
          }
        }
      // ---- O^T += V^T P^T
      if constexpr (kEight) {
        // rows quad and quad + 8 of block m are channels 16 quad + 2 m and 2 m + 1 (8 quad at width 64), columns the tokens
        // 2 t4, 2 t4 + 1 and 8 further
        constexpr int kWords = D == 64 ? 2 : 4;   // words of a row a lane takes
#pragma unroll
        for (int set = 0; set < (D == 256 ? 2 : 1); ++set) {
          uint32_t w[4][kWords];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int row = 2 * t4 + (u & 1) + 8 * (u >> 1);
            if constexpr (D == 64) {
              const uint64_t half = lds_b64(v_tile + piece_at<kBytes>(row, quad / 2) + (quad & 1) * 8);
              w[u][0] = static_cast<uint32_t>(half);
              w[u][1] = static_cast<uint32_t>(half >> 32);
            } else {
              const uint4 v = lds_b32x4(v_tile + piece_at<kBytes>(row, set * 8 + quad));
              w[u][0] = v.x; w[u][1] = v.y; w[u][2] = v.z; w[u][3] = v.w;
            }
          }
#pragma unroll
          for (int k = 0; k < kWords; ++k)
#pragma unroll
            for (int pair = 0; pair < 2; ++pair) {   // bytes 0, 1 and 2, 3 of the word
              const uint32_t ab = __byte_perm(w[0][k], w[1][k], pair ? 0x7362 : 0x5140), cd = __byte_perm(w[2][k], w[3][k], pair ? 0x7362 : 0x5140);
              const uint32_t a0 = halves_of(ab), a1 = halves_of(ab >> 16), a2 = halves_of(cd), a3 = halves_of(cd >> 16);
#pragma unroll
              for (int nb = 0; nb < kN; ++nb) mma<kEight>(o[set * 8 + 2 * k + pair][nb], a0, a1, a2, a3, p[nb][0], p[nb][1]);
            }
        }
      } else {
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) {
          uint32_t vf[4];
          ldmatrix_x4_trans(vf, v_tile + piece_at<kBytes>((lane / 16) * 8 + lane % 8, m * 2 + (lane / 8 & 1)));
#pragma unroll
          for (int nb = 0; nb < kN; ++nb) {
            mma<kEight>(o[m][nb], vf[0], vf[1], vf[2], vf[3], p[nb][0], p[nb][1]);
            mma<kEight>(o[m][nb], vf[0], vf[1], vf[2], vf[3], rest[nb][0], rest[nb][1]);
          }
        }
      }
      __syncwarp();   // the slot is free for the next issue
      if (++slot == kS) {
        slot = 0;
        ++round;
      }
      ++j;
  }
}

template <int D, bool kEight>
LineShape line_shape(const TreeArgs& a) {   // (many heads would leave workers over)
  return {4, 3, 4, 148 * kCtas<D, kEight> * kWarps, a.kv_heads <= 64 ? a.kv_heads : 1};
}

template <int D, bool kEight, bool kHalf>
cudaError_t launch_rows(cudaStream_t stream, const TreeArgs& a) {
  const LineShape shape = line_shape<D, kEight>(a);
  constexpr int kBytes = kWarps * (kStages<D, kEight> * kStageBytes<D, kEight> + static_cast<int>(sizeof(WarpState<kStages<D, kEight>, kEight>))) + 1024;
  static_assert((kBytes + 1024) * kCtas<D, kEight> <= 228 * 1024, "shared memory");
  CUtensorMap map_k, map_v;
  constexpr int kColumns = (kRowBytes<D, kEight> < 128 ? kRowBytes<D, kEight> : 128) / (kEight ? 1 : 2);
  if (!tree_pool_map(&map_k, a.pool.k, a, kTile, kColumns, kColumns * (kEight ? 1 : 2)) || !tree_pool_map(&map_v, a.pool.v, a, kTile, kColumns, kColumns * (kEight ? 1 : 2)))
    return cudaErrorInvalidValue;
  const long long tiles = static_cast<long long>(a.batch) * a.kv_heads * ((static_cast<long long>(a.max_prefix) + a.nodes + kTile - 1) / kTile);
  const long long ctas = (tiles + kWarps - 1) / kWarps, most = 148 * kCtas<D, kEight>;
  cudaError_t e = cudaFuncSetAttribute(tree_decode_mma_kernel<D, kEight, kHalf>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
  if (e != cudaSuccess) return e;
  tree_decode_mma_kernel<D, kEight, kHalf><<<static_cast<unsigned>(ctas < most ? ctas : most), kWarps * 32, kBytes, stream>>>(map_k, map_v, a, shape);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return tree_decode_merge(stream, a, shape);
}

template <int D, bool kEight>
cudaError_t launch(cudaStream_t stream, const TreeArgs& a) {
  if constexpr (D == 256) return launch_rows<D, kEight, true>(stream, a);
  else return a.nodes * a.group <= 8 ? launch_rows<D, kEight, true>(stream, a) : launch_rows<D, kEight, false>(stream, a);
}

}  // namespace

// Up to sixteen rows, the columns of two products (eight at width 256, whose accumulators fill the registers then), in pages
// that a step divides.  16 x 8000 tokens, bf16 and 8-bit, us here against tree_decode_sm100: width 128, 1 row 87 : 105 and
// 54 : 134, 8 rows 91 : 107 and 58 : 136, 16 rows 98 : 107 and 79 : 136; width 256, 6 rows 92 : 91 and 62 : 110; 24 x 4000, width 64,
// 16 rows 68 : 116 and 65 : 144.  Other pages (of 24) leave 5 rows of width 128 to the latter: 117 and 136 against 90 and 56.
bool tree_decode_mma_supported(const TreeArgs& a) {
  return a.nodes * a.group <= (a.dim == 256 ? 8 : 16) && tree_pool_fits(a, kTile) &&
         a.pool.scale_page < (1ull << 32) && a.pool.scale_token < (1ull << 32) &&
         line_fits(a, {4, 3, 4, 0, 1});
}

size_t tree_decode_mma_workspace_bytes(int nodes, int q_heads, int kv_heads, int dim) {
  return line_workspace_bytes({4, 3, 4, 148 * (dim == 256 ? 2 : dim == 128 ? 3 : 4) * kWarps, 1}, nodes, q_heads, kv_heads, dim);   // (for either storage)
}

cudaError_t tree_decode_mma(cudaStream_t stream, const TreeArgs& a) {
  const bool eight = a.pool.store == kStoreE4m3;
  if (a.dim == 64) return eight ? launch<64, true>(stream, a) : launch<64, false>(stream, a);
  if (a.dim == 128) return eight ? launch<128, true>(stream, a) : launch<128, false>(stream, a);
  return eight ? launch<256, true>(stream, a) : launch<256, false>(stream, a);
}

}  // namespace pluto
