// Attention of drafted tokens over a bf16 or 8-bit cache on the tensor cores (tcgen05), head widths 64, 128, 256.
//
//   out(i, h) = sum_t softmax_t(q(i, h) . k(t) / sqrt(D)) v(t),   t: the cached slots, node i's ancestors, node i
//
// The rows of a unit (sequence, KV head) are its nodes times the query heads of the KV head, row = node *
// group + head, so the cache is read once for all of them.  They are the 128 lanes of the MMA tiles:
//   S = Q K^T   M 128, N 64 keys, A = Q held in TMEM for the whole unit, B = the key tile (K-major)
//   O += P V    M 128, N D, A = P (bf16) written over S in TMEM, B = the value tile (MN-major)
// with one thread per row doing the softmax (running maximum with lazy rescaling of O, fp32 sums).  Few rows leave
// lanes idle, which costs nothing while the tiles arrive at memory speed: a 64-key tile of width 128 takes
// 512 clocks of the tensor pipe and 712 (8-bit) or 1424 (bf16) of an SM's share of the HBM rate.
//
// Two streams of S, O and softmax warps run side by side so that one's products run under the other's softmax.
// Up to 128 rows: the streams take the even and the odd key tiles and are merged at the end.  More: each
// takes 128 rows and both read every tile.  Width 256 (O takes half of TMEM): one O, two buffers of S.
//
// Loading.  Eight warps fetch 16 bytes per lane from the pages into registers, up to 64 KB per SM in flight, and store
// them as 128-byte-swizzled bf16 tiles; pages may have any size and rows any 16-byte stride.  8-bit codes
// are widened on the way: the code's bits shifted into a bf16 are the value times 2^-120, and one packed
// product with 2^(120 + n) gives the exact value (no rounding: see draft_rows.cuh), so what follows is one
// kernel for both.  (Copies of raw codes through shared memory would add a third to its traffic, which
// binds before HBM does.)
//
// Work is cut evenly over the SMs whatever the lengths: the units' key tiles, each unit with a few more for what
// it costs besides, form one line that is cut into equal ranges, one per CTA.  A CTA walks the units of its range; one that
// it holds whole it writes out, of the others it leaves (accumulator, maximum, sum) in the workspace, and a
// second kernel merges a cut unit's parts in the order of the keys.  The cut follows from the lengths alone.
#include "draft_rows.cuh"

namespace pluto {
namespace {

constexpr int kTile = 64;            // keys
constexpr int kThreads = 640;        // warps 0-3: MMA issue; 4-11: softmax; 12-15: keys; 16-19: values
constexpr int kMaxCtas = 148;
constexpr int kUnitTiles = 3;        // what a unit costs besides its tiles (query load, read-out), in tiles
constexpr float kRescale = 8.0f;     // O is rescaled when the maximum has grown by more than 2^8

template <int D>
constexpr int kStages = D == 64 ? 10 : D == 128 ? 6 : 3;
template <int D>
constexpr int kTileBytes = kTile * D * 2;
template <int D>
constexpr int kGroupRows = D == 256 ? 128 : 256;   // rows that share one pass over the keys

constexpr int group_rows(int dim) { return dim == 256 ? 128 : 256; }

// ---- the line of work ----------------------------------------------------------------------------------------
struct Sequence {
  int prefix, count, tiles, units;
};
__device__ __forceinline__ Sequence sequence_at(const TreeArgs& a, int b) {
  Sequence s;
  s.count = draft_count(a.counts, b, a.nodes, a.pool.status, 47);
  s.prefix = a.prefix[b];
  if (s.prefix < 0 || s.prefix > a.max_prefix) {
    report_status(a.pool.status, 47, kBadLength);
    s.prefix = s.prefix < 0 ? 0 : a.max_prefix;
  }
  const int rows = s.count * (a.q_heads / a.kv_heads), per = group_rows(a.dim);
  s.tiles = (s.prefix + s.count + kTile - 1) / kTile;
  s.units = a.kv_heads * ((rows + per - 1) / per);   // no nodes: no units
  return s;
}
__device__ __forceinline__ long long weight_of(const Sequence& s) {
  return static_cast<long long>(s.units) * (s.tiles + kUnitTiles);
}

// Where CTA c's range of the line begins, and the sequence that holds a position: by one warp.
struct Line {
  long long total;
  int parts;   // CTAs that take part
};
__device__ __forceinline__ long long range_begin(const Line& line, int c) { return line.total * c / line.parts; }
__device__ __forceinline__ Line measure_line(const TreeArgs& a, int ctas, int lane) {
  long long total = 0, tiles = 0;
  for (int b = lane; b < a.batch; b += 32) {
    const Sequence s = sequence_at(a, b);
    total += weight_of(s);
    tiles += static_cast<long long>(s.units) * s.tiles;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
  }
  return Line{total, static_cast<int>(max(1ll, min(static_cast<long long>(ctas), tiles)))};
}
// Sequence that holds `position` < total, and where it starts on the line.
__device__ __forceinline__ int find_sequence(const TreeArgs& a, long long position, int lane, long long& start) {
  long long before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int b = b0 + lane;
    const long long own = b < a.batch ? weight_of(sequence_at(a, b)) : 0;
    long long up_to = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long other = __shfl_up_sync(0xffffffffu, up_to, o);
      if (lane >= o) up_to += other;
    }
    const unsigned holds = __ballot_sync(0xffffffffu, before + up_to > position);
    if (holds) {
      const int at = __ffs(holds) - 1;
      start = before + __shfl_sync(0xffffffffu, up_to - own, at);
      return b0 + at;
    }
    before += __shfl_sync(0xffffffffu, up_to, 31);
  }
  start = before;
  return a.batch;
}

// A CTA's part of a unit.
struct Segment {
  int b, kv_head, row0, rows;      // rows: live rows of the group from row0 on (0: the range ends)
  int prefix, count, tile0, tile1; // key tiles [tile0, tile1)
  int whole;
  int slot;                        // workspace slot of a partial result: 0 for a unit that began before the range
};
// Walks the segments of a range: one warp, which hands them to the others through a ring in shared memory.
struct Cursor {
  long long begin, end, start;   // of the range; start of the current unit
  int b, unit;
  Sequence s;
  __device__ __forceinline__ bool next(const TreeArgs& a, Segment& out) {
    while (start < end && b < a.batch) {
      if (unit >= s.units) {
        unit = 0;
        if (++b >= a.batch) return false;
        s = sequence_at(a, b);
        continue;
      }
      const long long first = start + kUnitTiles;
      const int tile0 = static_cast<int>(max(0ll, begin - first)), tile1 = static_cast<int>(min(static_cast<long long>(s.tiles), end - first));
      const int own = unit;
      const long long own_start = start;
      ++unit;
      start += s.tiles + kUnitTiles;
      if (tile0 >= tile1) continue;
      const int per = group_rows(a.dim), rows = s.count * (a.q_heads / a.kv_heads), groups = s.units / a.kv_heads;
      out.b = b;
      out.kv_head = own / groups;
      out.row0 = own % groups * per;
      out.rows = min(per, rows - out.row0);
      out.prefix = s.prefix;
      out.count = s.count;
      out.tile0 = tile0;
      out.tile1 = tile1;
      out.whole = tile0 == 0 && tile1 == s.tiles;
      out.slot = own_start < begin ? 0 : 1;
      return true;
    }
    return false;
  }
};

// ---- shared memory -------------------------------------------------------------------------------------------
constexpr int kSegments = 8;         // of the ring
constexpr int kSegmentReaders = 17;  // warps: MMA issue, eight softmax, eight loaders

template <int D>
struct Shared {
  uint64_t seg_full[kSegments], seg_empty[kSegments];
  Segment seg[kSegments];
  uint64_t k_full[kStages<D>], k_empty[kStages<D>], v_full[kStages<D>], v_empty[kStages<D>];
  uint64_t q_full[2], s_full[2], p_full[2], pv_done[2];
  uint64_t ml_full, o_read;   // the two streams' meeting points: sums written, O read
  uint32_t tmem;
  float2 ml[2][128];
};

// The next segment of the range, by every lane of a warp; false at its end (or when a wait ran out).
template <int D>
__device__ __forceinline__ bool next_segment(Shared<D>* sh, int& n, Segment& seg, int lane, uint32_t* status) {
  const int at = n % kSegments;
  if (!__all_sync(0xffffffffu, mbar_wait(&sh->seg_full[at], (n / kSegments) & 1, status, 61))) return false;
  seg = sh->seg[at];
  ++n;
  __syncwarp();
  if (lane == 0) mbar_arrive(&sh->seg_empty[at]);
  return seg.rows > 0;
}

// ---- 8-bit codes to bf16 -------------------------------------------------------------------------------------
// Two codes in the high bytes of x's halves -> sign and magnitude bits of bf16: the value times 2^-120.
__device__ __forceinline__ uint32_t widen_pair(uint32_t x) { return (x & 0x80008000u) | ((x >> 4) & 0x07f007f0u); }
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint2 widen_word(uint32_t w, uint32_t factor) {   // four codes
  return make_uint2(mul_bf16x2(widen_pair(__byte_perm(w, 0u, 0x1404)), factor),
                    mul_bf16x2(widen_pair(__byte_perm(w, 0u, 0x3424)), factor));
}
// A row's factors as bf16 bits: 2^(120 + n) in the low half as far as bf16 holds it (n <= 7), the rest in the
// high half (1 unless the row holds values above 57344).  255 (not finite): NaN.
constexpr uint32_t kOne = 0x3f80u;
__device__ __forceinline__ uint32_t widen_factors(uint32_t byte) {
  if (byte == 255u) return kOne << 16 | 0x7fc0u;
  return (byte > 134u ? (byte - 7u) << 7 : kOne) << 16 | (min(byte, 134u) + 120u) << 7;
}

// ---- loaders -------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ bool not_finite(uint32_t pair) {
  return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u;
}
__device__ __forceinline__ bool not_finite(const uint4& v) {
  return not_finite(v.x) || not_finite(v.y) || not_finite(v.z) || not_finite(v.w);
}

// One warp's sixteen rows of every tile of the keys (or values).  A lane looks after row lane % 16's address and scale
// and copies pieces lane, lane + 32, ... of the sixteen rows.
template <int D, bool kEight, bool kValues>
__device__ __forceinline__ void load_tiles(const TreeArgs& a, Shared<D>* sh, uint32_t ring, int warp, int lane) {
  constexpr int kPieces = kEight ? D / 16 : D / 8;       // 16-byte pieces of a row
  constexpr int kLoads = kPieces / 2;                    // of sixteen rows, per lane
  constexpr int kBuffers = 16 / kLoads;
  constexpr int kElement = kEight ? 1 : 2;
  uint64_t* full = kValues ? sh->v_full : sh->k_full;
  uint64_t* empty = kValues ? sh->v_empty : sh->k_empty;
  const char* base = static_cast<const char*>(kValues ? a.pool.v : a.pool.k);
  const char* other = static_cast<const char*>(a.pool.v);

  uint4 raw[kBuffers][kLoads];
  uint32_t factors[kBuffers];
  Segment seg;
  int tile = 0, issued = 0, stored = 0, seg_n = 0;
  bool more = next_segment(sh, seg_n, seg, lane, a.pool.status);
  if (more) tile = seg.tile0;
  long long row_at = -1;     // byte offset of the lane's row of the next tile, -1: no row there
  size_t scale_at = 0;
  const auto locate = [&]() {
    row_at = -1;
    if (!more) return;
    const int t = tile * kTile + warp * 16 + lane % 16;
    if (t >= seg.prefix + seg.count) return;
    const long long page = draft_page(a.pool, seg.b, t, 48);
    if (page < 0) return;
    row_at = static_cast<long long>((draft_row(a.pool, page, t) + static_cast<size_t>(seg.kv_head) * D) * kElement);
    if (kEight) scale_at = draft_scale(a.pool, page, t) + seg.kv_head;
  };
  // Fetches the next tile of the range into a buffer.  Of drafts that not every node sees, a value row that is
  // not finite must not meet the zero weights of the nodes that do not see it: it is loaded as zeros, and
  // the key row is made NaN, which gives those that see it NaN scores and touches no other node.
  const auto issue = [&](uint4 (&buffer)[kLoads], uint32_t& factor) {
    const int first_draft = seg.count > 1 ? max(0, seg.prefix - tile * kTile) : kTile;   // row of the tile
    const bool drafts = first_draft < kTile;
    if (kEight) {
      factor = kOne << 16;
      if (row_at >= 0) {
        uint32_t byte = (kValues ? a.pool.v_scales : a.pool.k_scales)[scale_at];
        factor = widen_factors(byte);
        if (drafts && warp * 16 + lane % 16 >= first_draft) {
          if (kValues && byte == 255u) factor = kOne << 16;                              // zeros
          if (!kValues && a.pool.v_scales[scale_at] == 255) factor = widen_factors(255u);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int piece = i * 32 + lane, row = piece / kPieces;
      const long long at = __shfl_sync(0xffffffffu, row_at, row);
      buffer[i] = at >= 0 ? load_once(base + at + piece % kPieces * 16) : make_uint4(0u, 0u, 0u, 0u);
    }
    if (!kEight && drafts) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int piece = i * 32 + lane, row = piece / kPieces;
        const long long at = __shfl_sync(0xffffffffu, row_at, row);
        if (at < 0 || warp * 16 + row < first_draft) continue;
        if (kValues) {
          if (not_finite(buffer[i])) buffer[i] = make_uint4(0u, 0u, 0u, 0u);
        } else if (not_finite(load_once(other + at + piece % kPieces * 16))) {
          buffer[i] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
        }
      }
    }
    ++issued;
    if (++tile >= seg.tile1) {
      more = next_segment(sh, seg_n, seg, lane, a.pool.status);
      if (more) tile = seg.tile0;
    }
    locate();
  };
  locate();
#pragma unroll
  for (int u = 0; u < kBuffers; ++u)
    if (more) issue(raw[u], factors[u]);
  bool ok = true;
  while (ok && stored < issued) {
#pragma unroll
    for (int u = 0; u < kBuffers; ++u) {
      if (!ok || stored >= issued) break;
      const int stage = stored % kStages<D>, use = stored / kStages<D>;
      if (use > 0) ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], (use - 1) & 1, a.pool.status, kValues ? 51 : 50));
      if (!ok) break;
      const uint32_t to = ring + stage * kTileBytes<D>;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int piece = i * 32 + lane, row = piece / kPieces, c = piece % kPieces, r = warp * 16 + row;
        const uint4 v = raw[u][i];
        if (!kEight) {
          sts_b32x4(to + (c / 8) * (kTile * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4), v.x, v.y, v.z, v.w);
        } else {
          const uint32_t both = __shfl_sync(0xffffffffu, factors[u], row);
          const uint32_t factor = __byte_perm(both, both, 0x1010);
          uint2 w[4] = {widen_word(v.x, factor), widen_word(v.y, factor), widen_word(v.z, factor), widen_word(v.w, factor)};
          if ((both >> 16) != kOne) {   // values above 57344
            const uint32_t more_factor = __byte_perm(both, both, 0x3232);
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = make_uint2(mul_bf16x2(w[k].x, more_factor), mul_bf16x2(w[k].y, more_factor));
          }
          // pieces 2c and 2c + 1 of the row; odd slabs store the second one first, so that eight lanes hit all banks once
          const uint32_t slab = to + (c / 4) * (kTile * 128) + r * 128;
          const int p0 = (2 * c) & 7, odd = (c / 4) & 1;
          const uint32_t at0 = slab + ((p0 ^ (r & 7)) << 4), at1 = slab + (((p0 + 1) ^ (r & 7)) << 4);
          if (odd) {
            sts_b32x4(at1, w[2].x, w[2].y, w[3].x, w[3].y);
            sts_b32x4(at0, w[0].x, w[0].y, w[1].x, w[1].y);
          } else {
            sts_b32x4(at0, w[0].x, w[0].y, w[1].x, w[1].y);
            sts_b32x4(at1, w[2].x, w[2].y, w[3].x, w[3].y);
          }
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[stage]);
      ++stored;
      if (more) issue(raw[u], factors[u]);
    }
  }
}

// ---- output --------------------------------------------------------------------------------------------------
struct Partials {
  float* acc;   // [slots][rows][D]
  float2* ml;   // [slots][rows]
  int rows;     // rows a slot has room for
};
__host__ __device__ inline int slot_rows(int nodes, int q_heads, int kv_heads, int dim) {
  const int rows = nodes * (q_heads / kv_heads);
  return rows < group_rows(dim) ? rows : group_rows(dim);
}
__device__ __forceinline__ Partials partials_of(const TreeArgs& a) {
  Partials p;
  p.rows = slot_rows(a.nodes, a.q_heads, a.kv_heads, a.dim);
  p.ml = static_cast<float2*>(a.workspace);
  p.acc = reinterpret_cast<float*>(p.ml + static_cast<size_t>((2 * kMaxCtas * p.rows + 1) & ~1));
  return p;
}

// Eight neighbouring channels of one output row.
__device__ __forceinline__ void store_out8(const TreeArgs& a, size_t token, int head, int d, const float (&x)[8], bool gate_pieces) {
  float y[8];
  if (a.gate != nullptr && gate_pieces) {
    const uint4 g = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.gate) + token * a.gate_token +
                                                    static_cast<size_t>(head) * a.gate_head + d);
    const float gate[8] = {bf16_lo(g.x), bf16_hi(g.x), bf16_lo(g.y), bf16_hi(g.y), bf16_lo(g.z), bf16_hi(g.z), bf16_lo(g.w), bf16_hi(g.w)};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float factor = sigmoid(gate[i]);
      y[i] = a.round ? bf16_round(x[i]) * bf16_round(factor) : x[i] * factor;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = tree_output(a, token, head, d + i, x[i]);
  }
  *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + (token * a.q_heads + head) * a.dim + d) =
      make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
}
__device__ __forceinline__ bool gate_in_pieces(const TreeArgs& a) {
  return a.gate_is_bf16 && a.gate_token % 8 == 0 && a.gate_head % 8 == 0 && (reinterpret_cast<uintptr_t>(a.gate) & 15u) == 0;
}

template <int D, bool kEight>
__global__ void __launch_bounds__(kThreads, 1) tree_decode_sm100(TreeArgs a) {
  constexpr bool kOneO = D == 256;                       // one accumulator for both score buffers
  constexpr uint32_t kColO1 = D, kColS = kOneO ? 256 : 2 * D, kColQ = kColS + 128;
  static_assert(kColQ + (kOneO ? D / 2 : D) <= 512, "tensor memory");
  constexpr uint32_t kIdescQK = umma_idesc_bf16(128, kTile, false), kIdescPV = umma_idesc_bf16(128, D, true);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Shared<D>* sh = reinterpret_cast<Shared<D>*>(smem + 2 * kStages<D> * kTileBytes<D>);
  const uint32_t k_ring = smem_u32(smem), v_ring = k_ring + kStages<D> * kTileBytes<D>;
  const int warp = uniform_warp_index(), lane = threadIdx.x % 32;
  pdl_launch_dependents();   // the merge may be placed as SMs free up; it waits for this grid's end

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages<D>; ++s) {
      mbar_init(&sh->k_full[s], 4);
      mbar_init(&sh->v_full[s], 4);
      mbar_init(&sh->k_empty[s], 1);
      mbar_init(&sh->v_empty[s], 1);
    }
    for (int i = 0; i < kSegments; ++i) {
      mbar_init(&sh->seg_full[i], 1);
      mbar_init(&sh->seg_empty[i], kSegmentReaders);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&sh->q_full[x], 4);
      mbar_init(&sh->s_full[x], 1);
      mbar_init(&sh->p_full[x], 4);
      mbar_init(&sh->pv_done[x], 1);
    }
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

  // Register file: 640 threads x 96 at launch; the issuing warpgroup gives 56 x 128 back, of which the softmax ones
  // take 16 x 256 and the loaders 8 x 256.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
      // ---------------------------------------------------------------- MMA issue
      int tile_n = 0, q_n[2] = {0, 0}, p_n[2] = {0, 0};   // tiles, queries and P handed over so far
      bool ok = true;
      int seg_n = 0;
      Segment seg;
      while (ok && next_segment(sh, seg_n, seg, lane, status)) {
        const int tiles = __shfl_sync(0xffffffffu, seg.tile1 - seg.tile0, 0);
        const bool pair = __shfl_sync(0xffffffffu, seg.rows > 128 ? 1 : 0, 0);
        const int items = pair ? 2 * tiles : tiles;
        for (int x = 0; x < (pair ? 2 : 1) && ok; ++x)
          ok = __all_sync(0xffffffffu, mbar_wait(&sh->q_full[x], q_n[x]++ & 1, status, 52));
        if (!ok) break;
        const auto issue_qk = [&](int i) -> bool {
          const int x = i & 1, n = tile_n + (pair ? i >> 1 : i), stage = n % kStages<D>;
          if (!pair || x == 0) {
            if (!__all_sync(0xffffffffu, mbar_wait(&sh->k_full[stage], (n / kStages<D>) & 1, status, 53))) return false;
          }
          tc_fence_after();
          const uint64_t k_desc = umma_desc_sw128(k_ring + stage * kTileBytes<D>, 16, 1024);
          const uint32_t q = tmem + kColQ + (pair && x ? D / 2 : 0);
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              umma_ts(tmem + kColS + x * kTile, q + ks * 8, k_desc + (((ks / 4) * (kTile * 128) + (ks % 4) * 32) >> 4), kIdescQK, ks > 0);
            tc_commit(&sh->s_full[x]);
            if (!pair || x == 1) tc_commit(&sh->k_empty[stage]);
          }
          __syncwarp();
          return true;
        };
        const auto issue_pv = [&](int i) -> bool {
          const int x = i & 1, j = pair ? i >> 1 : i, n = tile_n + j, stage = n % kStages<D>;
          if (!pair || x == 0) {
            if (!__all_sync(0xffffffffu, mbar_wait(&sh->v_full[stage], (n / kStages<D>) & 1, status, 54))) return false;
          }
          if (!__all_sync(0xffffffffu, mbar_wait(&sh->p_full[x], p_n[x]++ & 1, status, 55))) return false;
          tc_fence_after();
          const uint64_t v_desc = umma_desc_sw128(v_ring + stage * kTileBytes<D>, kTile * 128, 1024);
          const bool add = kOneO ? i > 0 : pair ? j > 0 : i > 1;
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < kTile / 16; ++ks)
              umma_ts(tmem + (kOneO ? 0u : x * kColO1), tmem + kColS + x * kTile + ks * 8, v_desc + ks * (2048 >> 4), kIdescPV, add || ks > 0);
            tc_commit(&sh->pv_done[kOneO ? 0 : x]);
            if (!pair || x == 1) tc_commit(&sh->v_empty[stage]);
          }
          __syncwarp();
          return true;
        };
        ok = issue_qk(0) && (items < 2 || issue_qk(1));
        for (int i = 0; i < items && ok; ++i) ok = issue_pv(i) && (i + 2 >= items || issue_qk(i + 2));
        tile_n += tiles;
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- the range's segments
      const Line line = measure_line(a, gridDim.x, lane);
      const int c = blockIdx.x;
      Cursor cursor;
      cursor.begin = cursor.end = cursor.start = 0;
      cursor.b = cursor.unit = 0;
      cursor.s = Sequence{0, 0, 0, 0};
      if (c < line.parts && line.total > 0) {
        cursor.begin = range_begin(line, c);
        cursor.end = range_begin(line, c + 1);
        cursor.b = find_sequence(a, cursor.begin, lane, cursor.start);
        if (cursor.b < a.batch) {   // straight to the unit that holds the range's begin
          cursor.s = sequence_at(a, cursor.b);
          cursor.unit = static_cast<int>((cursor.begin - cursor.start) / (cursor.s.tiles + kUnitTiles));
          cursor.start += static_cast<long long>(cursor.unit) * (cursor.s.tiles + kUnitTiles);
        }
      }
      bool more = true;
      for (int n = 0; more; ++n) {
        const int at = n % kSegments;
        Segment seg{};
        more = cursor.next(a, seg);
        if (n >= kSegments && !__all_sync(0xffffffffu, mbar_wait(&sh->seg_empty[at], (n / kSegments - 1) & 1, status, 62))) break;
        if (lane == 0) {
          if (!more) seg.rows = 0;
          sh->seg[at] = seg;
          mbar_arrive(&sh->seg_full[at]);
        }
        __syncwarp();
      }
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
    // ------------------------------------------------------------------ softmax, one thread per row
    const int x = (warp - 4) / 4, quarter = warp & 3, row = quarter * 32 + lane, group = a.q_heads / a.kv_heads;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const float scale_log2 = a.scale * 1.4426950408889634f;
    const Partials parts = partials_of(a);
    const bool gate_pieces = gate_in_pieces(a);
    int s_n[2] = {0, 0}, pv_n[2] = {0, 0}, met = 0;   // score tiles taken, products into each O, meetings of the streams
    bool ok = true;
    int seg_n = 0;
    Segment seg;
    // (at width 256 the second warpgroup only keeps the ring of segments going)
    while (next_segment(sh, seg_n, seg, lane, status)) {
      if (kOneO && x == 1) continue;
      const bool pair = seg.rows > 128;
      const int tiles = seg.tile1 - seg.tile0, own_row = (pair ? x * 128 : 0) + row;
      const bool live = own_row < seg.rows, warp_live = (pair ? x * 128 : 0) + quarter * 32 < seg.rows;
      const int r = seg.row0 + own_row, node = r / group, head = seg.kv_head * group + r % group;
      const size_t token = static_cast<size_t>(seg.b) * a.nodes + node;
      // ---- the queries, into TMEM
      if (pair || x == 0) {
        if (warp_live) {
          const uint4* q = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + (token * a.q_heads + head) * D);
#pragma unroll 1
          for (int c = 0; c < D / 64; ++c) {
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint4 v = live ? q[c * 8 + i] : make_uint4(0u, 0u, 0u, 0u);
              w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
            }
            tmem_st32(lanes + kColQ + (pair ? x * (D / 2) : 0) + c * 32, w);
          }
          tmem_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->q_full[pair ? x : 0]);
      }
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
      float m_used = -INFINITY, m_true = -INFINITY, l = 0.0f;
      const int step = pair || kOneO ? 1 : 2;
      int done = 0;
      for (int j = pair || kOneO ? 0 : x; j < tiles && ok; j += step, ++done) {
        const int sb = kOneO ? j & 1 : x;
        ok = __all_sync(0xffffffffu, mbar_wait(&sh->s_full[sb], s_n[sb]++ & 1, status, 56));
        if (!ok) break;
        if (warp_live) {
          tc_fence_after();
          uint32_t s[2][32];
          const uint32_t s_at = lanes + kColS + sb * kTile;
          tmem_ld32(s_at, s[0]);
          tmem_ld32(s_at + 32, s[1]);
          tmem_wait_ld();
          const int behind = (seg.tile0 + j) * kTile - seg.prefix;   // of the drafts' first slot
          if (behind > -kTile) {
            const uint64_t seen = behind >= 64  ? seen_hi >> (behind - 64)
                                  : behind > 0  ? seen_lo >> behind | seen_hi << (64 - behind)
                                  : behind == 0 ? seen_lo
                                                : seen_lo << -behind | ((1ull << -behind) - 1);
            const uint32_t bits[2] = {static_cast<uint32_t>(seen), static_cast<uint32_t>(seen >> 32)};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(bits[h] >> i & 1u)) s[h][i] = 0xff800000u;
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(s[h][i]), __uint_as_float(s[h][i + 1]));
          m_true = max3(fmaxf(m_true, mx[0]), mx[1], fmaxf(mx[2], mx[3]));
          const bool grow = (m_true - m_used) * scale_log2 > kRescale;
          if (__any_sync(0xffffffffu, grow)) {
            const float factor = grow ? fast_exp2((m_used - m_true) * scale_log2) : 1.0f;
            if (grow) m_used = m_true;
            l *= factor;
            if (done > 0) {
              // (with its own O the previous product has ended: this tile's scores were committed behind it)
              if (kOneO) ok = __all_sync(0xffffffffu, mbar_wait(&sh->pv_done[0], (pv_n[0] + done - 1) & 1, status, 57));
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 16; ++c) {
                uint32_t o[16];
                const uint32_t o_at = lanes + (kOneO ? 0u : x * kColO1) + c * 16;
                tmem_ld16(o_at, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                tmem_st16(o_at, o);
              }
              tmem_wait_st();
            }
          }
          const float m_safe = m_used == -INFINITY ? 0.0f : m_used;   // nothing seen yet
          const uint64_t scale2 = f2_pack(scale_log2, scale_log2), neg2 = f2_pack(-m_safe * scale_log2, -m_safe * scale_log2);
          uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t packed[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float p0, p1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(s[h][i]), __uint_as_float(s[h][i + 1])), scale2, neg2), p0, p1);
              p0 = fast_exp2(p0);
              p1 = fast_exp2(p1);
              sum2[(i >> 1) & 1] = f2_add(sum2[(i >> 1) & 1], f2_pack(p0, p1));
              packed[i / 2] = pack_bf16(p0, p1);
            }
            tmem_st16(s_at + h * 16, packed);
          }
          float a0, a1, b0, b1;
          f2_unpack(sum2[0], a0, a1);
          f2_unpack(sum2[1], b0, b1);
          l += (a0 + a1) + (b0 + b1);
          tmem_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full[sb]);
      }
      if (!ok) break;
      const bool merged = !pair && !kOneO;
      const int products[2] = {merged ? (tiles + 1) / 2 : tiles, merged ? tiles / 2 : pair ? tiles : 0};
      // A parity tells the phase that is awaited from its neighbours only, so the one before must be known to be over:
      // this stream's last scores were committed behind its last but one product (one O: behind the last but two).
      const int own_o = kOneO ? 0 : x;
      pv_n[0] += products[0];
      pv_n[1] += products[1];
      if (kOneO && tiles > 1) ok = __all_sync(0xffffffffu, mbar_wait(&sh->pv_done[0], (pv_n[0] - 2) & 1, status, 57));
      if (ok && done > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sh->pv_done[own_o], (pv_n[own_o] - 1) & 1, status, 58));
      if (!ok) break;
      tc_fence_after();
      // ---- read-out: rows of one stream, or the two streams' halves of the keys merged, half of the channels each
      float m = m_used, f0 = 1.0f, f1 = 0.0f;
      bool both = false;
      if (merged) {
        sh->ml[x][row] = make_float2(m_used, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->ml_full);
        ok = __all_sync(0xffffffffu, mbar_wait(&sh->ml_full, met & 1, status, 59));
        // (the other stream has seen its last product end before it arrived there: this returns at once)
        if (ok && products[1 - x] > 0)
          ok = __all_sync(0xffffffffu, mbar_wait(&sh->pv_done[1 - x], (pv_n[1 - x] - 1) & 1, status, 58));
        if (!ok) break;
        tc_fence_after();
        const float2 one = sh->ml[0][row], two = sh->ml[1][row];
        both = tiles > 1;
        m = both ? fmaxf(one.x, two.x) : one.x;
        const float m_safe = m == -INFINITY ? 0.0f : m;
        f0 = fast_exp2((one.x - m_safe) * scale_log2);
        f1 = both ? fast_exp2((two.x - m_safe) * scale_log2) : 0.0f;
        l = both ? one.y * f0 + two.y * f1 : one.y * f0;
      }
      if (warp_live) {
        const int slot = 2 * blockIdx.x + seg.slot;
        const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
        float* acc = parts.acc + (static_cast<size_t>(slot) * parts.rows + own_row) * D;
        const int c0 = merged ? x * (D / 32) : 0, c1 = merged ? c0 + D / 32 : D / 16;
#pragma unroll 1
        for (int c = c0; c < c1; ++c) {
          uint32_t o[16];
          tmem_ld16(lanes + (merged || kOneO ? 0u : x * kColO1) + c * 16, o);
          if (both) {
            uint32_t o2[16];
            tmem_ld16(lanes + kColO1 + c * 16, o2);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f0 + __uint_as_float(o2[i]) * f1);
          } else {
            tmem_wait_ld();
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
#pragma unroll
            for (int i = 0; i < 4; ++i)
              reinterpret_cast<uint4*>(acc + c * 16)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
          __syncwarp();
        }
        if (live && (x == 0 || pair)) {
          if (!seg.whole) parts.ml[static_cast<size_t>(slot) * parts.rows + own_row] = make_float2(m * scale_log2, l);
          else if (a.lse) a.lse[token * a.q_heads + head] = (m == -INFINITY ? 0.0f : m * a.scale) + logf(l);
        }
        tc_fence_before();
      }
      if (merged) {   // both have read both accumulators (and sums) before either stream's next product
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->o_read);
        ok = __all_sync(0xffffffffu, mbar_wait(&sh->o_read, met++ & 1, status, 60));
        if (!ok) break;
      }
    }
  } else {
    // ------------------------------------------------------------------ loaders
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    if (warp < 16) load_tiles<D, kEight, false>(a, sh, k_ring, warp - 12, lane);
    else load_tiles<D, kEight, true>(a, sh, v_ring, warp - 16, lane);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// Merges the parts of the units that the line's cuts fall into, in the order of the keys.  Block (j, y): cut j + 1,
// eight rows; it acts if its cut is the first one inside its unit.  One warp per row.
__global__ void __launch_bounds__(256) tree_decode_merge(TreeArgs a, int ctas) {
  __shared__ Line line;
  __shared__ long long found_start;
  __shared__ int found_b;
  __shared__ float weight[8][kMaxCtas];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, cut = blockIdx.x + 1, row = blockIdx.y * 8 + warp;
  if (warp == 0) {   // (prefix and counts were there before the kernel that this one waits for)
    const Line l = measure_line(a, ctas, lane);
    long long start = 0;
    const int b = cut < l.parts ? find_sequence(a, range_begin(l, cut), lane, start) : a.batch;
    if (lane == 0) {
      line = l;
      found_b = b;
      found_start = start;
    }
  }
  __syncthreads();
  pdl_wait();   // the parts are complete and visible from here on
  if (cut >= line.parts || found_b >= a.batch) return;
  const Sequence s = sequence_at(a, found_b);
  const long long span = s.tiles + kUnitTiles;
  const int unit = static_cast<int>((range_begin(line, cut) - found_start) / span);
  const long long start = found_start + unit * span, end = start + span;
  if (range_begin(line, cut) <= start || range_begin(line, cut - 1) > start) return;
  // the CTAs that hold tiles of it
  int first = -1, last = -1;
  for (int c = cut - 1; c < line.parts && range_begin(line, c) < end; ++c) {
    if (min(range_begin(line, c + 1), end) > max(range_begin(line, c), start + kUnitTiles)) {
      if (first < 0) first = c;
      last = c;
    }
  }
  if (first == last) return;   // one CTA holds all of its tiles and has written it out
  const int group = a.q_heads / a.kv_heads, groups = s.units / a.kv_heads, per = group_rows(a.dim);
  const int row0 = unit % groups * per, rows = min(per, s.count * group - row0), kv_head = unit / groups;
  if (row >= rows) return;
  const Partials parts = partials_of(a);
  const auto part_at = [&](int c) {
    return static_cast<size_t>(2 * c + (start < range_begin(line, c) ? 0 : 1)) * parts.rows + row;
  };
  float m = -INFINITY;
  for (int c = first + lane; c <= last; c += 32) m = fmaxf(m, parts.ml[part_at(c)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float m_safe = m == -INFINITY ? 0.0f : m;
  for (int c = first + lane; c <= last; c += 32) weight[warp][c - first] = fast_exp2(parts.ml[part_at(c)].x - m_safe);
  __syncwarp();
  float l = 0.0f, acc[8] = {};
  const int D = a.dim;
#pragma unroll 4
  for (int c = first; c <= last; ++c) {
    const float w = weight[warp][c - first];
    const size_t at = part_at(c);
    l = fmaf(parts.ml[at].y, w, l);
    const float* from = parts.acc + at * D + lane * 8;
    if (lane * 8 < D) {
      const float4 u = reinterpret_cast<const float4*>(from)[0], v = reinterpret_cast<const float4*>(from)[1];
      acc[0] = fmaf(u.x, w, acc[0]); acc[1] = fmaf(u.y, w, acc[1]); acc[2] = fmaf(u.z, w, acc[2]); acc[3] = fmaf(u.w, w, acc[3]);
      acc[4] = fmaf(v.x, w, acc[4]); acc[5] = fmaf(v.y, w, acc[5]); acc[6] = fmaf(v.z, w, acc[6]); acc[7] = fmaf(v.w, w, acc[7]);
    }
  }
  const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
  const int r = row0 + row, node = r / group, head = kv_head * group + r % group;
  const size_t token = static_cast<size_t>(found_b) * a.nodes + node;
  if (lane * 8 < D) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= inverse;
    store_out8(a, token, head, lane * 8, acc, gate_in_pieces(a));
  }
  if (lane == 0 && a.lse) a.lse[token * a.q_heads + head] = m_safe * 0.6931471805599453f + logf(l);
}

template <int D, bool kEight>
cudaError_t launch(cudaStream_t stream, const TreeArgs& a) {
  const int rows = slot_rows(a.nodes, a.q_heads, a.kv_heads, D);
  const long long units = static_cast<long long>(a.batch) * a.kv_heads * ((a.nodes * (a.q_heads / a.kv_heads) + kGroupRows<D> - 1) / kGroupRows<D>);
  const long long tiles = units * ((static_cast<long long>(a.max_prefix) + a.nodes + kTile - 1) / kTile);
  const int ctas = static_cast<int>(tiles < kMaxCtas ? tiles : kMaxCtas);
  constexpr int kBytes = 2 * kStages<D> * kTileBytes<D> + static_cast<int>(sizeof(Shared<D>)) + 1024;
  static_assert(kBytes <= 227 * 1024, "shared memory");
  cudaError_t e = cudaFuncSetAttribute(tree_decode_sm100<D, kEight>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
  if (e != cudaSuccess) return e;
  tree_decode_sm100<D, kEight><<<ctas, kThreads, kBytes, stream>>>(a);
  if ((e = cudaGetLastError()) != cudaSuccess || ctas == 1) return e;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(ctas - 1, (rows + 7) / 8);
  config.blockDim = dim3(256);
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, tree_decode_merge, a, ctas);
}

}  // namespace

bool tree_decode_tc_supported(const TreeArgs& a) {
  const size_t element = a.pool.store == kStoreBf16 ? 2 : 1;
  const auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  return a.q_is_bf16 && a.out_is_bf16 && a.pool.store != kStoreFp32 && (a.dim == 64 || a.dim == 128 || a.dim == 256) &&
         aligned(a.q) && aligned(a.out) && aligned(a.pool.k) && aligned(a.pool.v) && a.pool.page_stride * element % 16 == 0 &&
         a.pool.token_stride * element % 16 == 0;
}

size_t tree_decode_tc_workspace_bytes(int nodes, int q_heads, int kv_heads, int dim) {
  if (dim != 64 && dim != 128 && dim != 256) return 0;
  const size_t rows = slot_rows(nodes, q_heads, kv_heads, dim);
  return ((2 * kMaxCtas * rows + 1) & ~static_cast<size_t>(1)) * sizeof(float2) + 2 * kMaxCtas * rows * dim * sizeof(float);
}

cudaError_t tree_decode_tc(cudaStream_t stream, const TreeArgs& a) {
  const bool eight = a.pool.store == kStoreE4m3;
  if (a.dim == 64) return eight ? launch<64, true>(stream, a) : launch<64, false>(stream, a);
  if (a.dim == 128) return eight ? launch<128, true>(stream, a) : launch<128, false>(stream, a);
  return eight ? launch<256, true>(stream, a) : launch<256, false>(stream, a);
}

}  // namespace pluto
