// How the attention of drafted tokens is cut over the GPU, whatever the sequences' lengths.
//
// A unit is a (sequence, KV head, group of rows); it is a row of key tiles.  All units, each with a few tiles more for what
// it costs besides, form one line that is cut into equal ranges, one per worker (a CTA or a warp).  A worker walks the
// units of its range; a unit that it holds whole it writes out, of the others it leaves (accumulator, maximum, sum) in
// one of its two workspace slots, and tree_decode_merge adds a cut unit's parts in the order of the keys.  Where the
// line is cut follows from the lengths alone, so results repeat bit for bit.
#pragma once

#include "draft_rows.cuh"

namespace pluto {

// Positions are 32-bit: line_fits is asked on the host.  A cache row holds all KV heads of a token, so workers that walk
// the heads side by side read whole rows of it between them.
struct LineShape {
  int tile_shift;   // keys per tile
  int overhead;     // what a unit costs besides its tiles, in tiles
  int rows_shift;   // rows of a unit at most
  int workers;      // at most
  int side;         // KV heads walked side by side, by neighbouring workers over the same range: all of them, or 1
};
inline bool line_fits(const TreeArgs& a, const LineShape& shape) {
  const long long groups = (static_cast<long long>(a.nodes) * a.group + (1 << shape.rows_shift) - 1) >> shape.rows_shift;
  const long long tiles = ((static_cast<long long>(a.max_prefix) + a.nodes) >> shape.tile_shift) + 1 + shape.overhead;
  return tiles < (1ll << 31) / (a.batch * groups * a.kv_heads + 1);
}

struct Sequence {
  int prefix, count, tiles, units;
};
__device__ __forceinline__ Sequence sequence_at(const TreeArgs& a, const LineShape& shape, int b) {
  Sequence s;
  s.count = draft_count(a.counts, b, a.nodes, a.pool.status, 47);
  s.prefix = a.prefix[b];
  if (s.prefix < 0 || s.prefix > a.max_prefix) {
    report_status(a.pool.status, 47, kBadLength);
    s.prefix = s.prefix < 0 ? 0 : a.max_prefix;
  }
  s.tiles = (s.prefix + s.count + (1 << shape.tile_shift) - 1) >> shape.tile_shift;
  s.units = a.kv_heads / shape.side * ((s.count * a.group + (1 << shape.rows_shift) - 1) >> shape.rows_shift);   // no nodes: no units
  return s;
}
__device__ __forceinline__ unsigned weight_of(const LineShape& shape, const Sequence& s) {
  return static_cast<unsigned>(s.units) * (s.tiles + shape.overhead);
}

struct Line {
  unsigned total, base;
  unsigned parts, longer;   // ranges, no more than there are tiles; the first `longer` hold base + 1, the others base
};
__device__ __forceinline__ unsigned range_begin(const Line& line, unsigned c) { return line.base * c + min(c, line.longer); }
__device__ __forceinline__ unsigned holder_of(const Line& line, unsigned position) {   // range it falls into
  const unsigned from = line.longer * (line.base + 1);
  return position < from ? position / (line.base + 1) : line.longer + (position - from) / line.base;
}
__device__ __forceinline__ Line cut_line(const LineShape& shape, unsigned total, unsigned tiles) {
  Line line;
  line.total = total;
  line.parts = max(1u, min(static_cast<unsigned>(shape.workers / shape.side), tiles));
  line.base = total / line.parts;
  line.longer = total - line.base * line.parts;
  return line;
}

// The whole line, by one warp; `before`: the weight of the sequences below `upto`.
__device__ __forceinline__ Line measure_line(const TreeArgs& a, const LineShape& shape, int lane, int upto, unsigned& before) {
  unsigned total = 0, tiles = 0, below = 0;
  for (int b = lane; b < a.batch; b += 32) {
    const Sequence s = sequence_at(a, shape, b);
    const unsigned weight = weight_of(shape, s);
    total += weight;
    tiles += s.units * s.tiles;
    if (b < upto) below += weight;
  }
  total = __reduce_add_sync(0xffffffffu, total);
  tiles = __reduce_add_sync(0xffffffffu, tiles);
  before = __reduce_add_sync(0xffffffffu, below);
  return cut_line(shape, total, tiles);
}

// A worker's part of a unit.
struct Segment {
  int b, kv_head, row0, rows;      // rows: live rows of the group from row0 on (0: the range ends)
  int prefix, count, tile0, tile1; // key tiles [tile0, tile1)
  int whole;
  int slot;                        // workspace slot of a partial result: 0 for a unit that began before the range
};
// Walks the segments of a range.
struct Cursor {
  unsigned begin, end, start;   // of the range; start of the current unit
  int b, unit, head;             // head: the worker's, where they are walked side by side
  Sequence s;
  // by a whole warp
  __device__ __forceinline__ void seek(const TreeArgs& a, const LineShape& shape, unsigned worker, int lane) {
    unsigned none;
    const Line line = measure_line(a, shape, lane, 0, none);
    begin = end = start = 0;
    b = unit = 0;
    s = Sequence{0, 0, 0, 0};
    const unsigned range = worker / shape.side;
    head = worker % shape.side;
    if (range >= line.parts || line.total == 0) return;
    begin = range_begin(line, range);
    end = range_begin(line, range + 1);
    // the sequence that holds the begin
    unsigned before = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
      const int own_b = min(b0 + lane, a.batch - 1);
      const Sequence own = sequence_at(a, shape, own_b);
      const unsigned weight = b0 + lane < a.batch ? weight_of(shape, own) : 0u;
      unsigned up_to = weight;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned other = __shfl_up_sync(0xffffffffu, up_to, o);
        if (lane >= o) up_to += other;
      }
      const unsigned holds = __ballot_sync(0xffffffffu, before + up_to > begin);
      if (holds) {
        const int at = __ffs(holds) - 1;
        b = b0 + at;
        start = before + __shfl_sync(0xffffffffu, up_to - weight, at);
        s.prefix = __shfl_sync(0xffffffffu, own.prefix, at);
        s.count = __shfl_sync(0xffffffffu, own.count, at);
        s.tiles = __shfl_sync(0xffffffffu, own.tiles, at);
        s.units = __shfl_sync(0xffffffffu, own.units, at);
        break;
      }
      before += __shfl_sync(0xffffffffu, up_to, 31);
    }
    unit = (begin - start) / (s.tiles + shape.overhead);   // straight to the unit that holds the begin
    start += unit * (s.tiles + shape.overhead);
  }
  __device__ __forceinline__ bool next(const TreeArgs& a, const LineShape& shape, Segment& out) {
    while (start < end && b < a.batch) {
      if (unit >= s.units) {
        unit = 0;
        if (++b >= a.batch) return false;
        s = sequence_at(a, shape, b);
        continue;
      }
      const unsigned first = start + shape.overhead;
      const int tile0 = begin > first ? begin - first : 0, tile1 = end > first ? min(static_cast<unsigned>(s.tiles), end - first) : 0u;
      const int own = unit;
      const unsigned own_start = start;
      ++unit;
      start += s.tiles + shape.overhead;
      if (tile0 >= tile1) continue;
      const int rows = s.count * a.group, groups = (rows + (1 << shape.rows_shift) - 1) >> shape.rows_shift;
      out.b = b;
      out.kv_head = shape.side > 1 ? head : groups == 1 ? own : own / groups;
      out.row0 = (groups == 1 ? 0 : own % groups) << shape.rows_shift;
      out.rows = min(1 << shape.rows_shift, rows - out.row0);
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

// ---- the workspace: two slots per worker --------------------------------------------------------------------
struct Partials {
  float* acc;   // [slots][rows][D], relative to the maximum
  float2* ml;   // [slots][rows]: maximum in powers of two, sum of the weights
  int rows;     // rows a slot has room for
};
__host__ __device__ inline int slot_rows(const LineShape& shape, int nodes, int q_heads, int kv_heads) {
  const int rows = nodes * (q_heads / kv_heads);
  return rows < (1 << shape.rows_shift) ? rows : 1 << shape.rows_shift;
}
__host__ __device__ inline size_t ml_pairs(const LineShape& shape, int rows) {   // even: the accumulators stay 16-byte aligned
  return (2 * static_cast<size_t>(shape.workers) * rows + 1) & ~static_cast<size_t>(1);
}
inline size_t line_workspace_bytes(const LineShape& shape, int nodes, int q_heads, int kv_heads, int dim) {
  const int rows = slot_rows(shape, nodes, q_heads, kv_heads);
  return ml_pairs(shape, rows) * sizeof(float2) + 2 * static_cast<size_t>(shape.workers) * rows * dim * sizeof(float);
}
__device__ __forceinline__ Partials partials_of(const TreeArgs& a, const LineShape& shape) {
  Partials p;
  p.rows = slot_rows(shape, a.nodes, a.q_heads, a.kv_heads);
  p.ml = static_cast<float2*>(a.workspace);
  p.acc = reinterpret_cast<float*>(p.ml + ml_pairs(shape, p.rows));
  return p;
}

__device__ __forceinline__ float power_of_two(float n) {   // n whole, -126 to 127
  return __uint_as_float(static_cast<uint32_t>(static_cast<int>(n) + 127) << 23);
}
// Parts over 8-bit caches leave in the unit of the values, which all parts share, and times 2^-drop, so that a part's weights
// sum to less than 2^-11: sums over parts are finite wherever the values are.
__device__ __forceinline__ float part_drop(float l) {
  return l > 0.0f ? fminf(static_cast<float>(static_cast<int>(__float_as_uint(l) >> 23) - 127 + 12), 126.0f) : 0.0f;
}

// Bounded wait on a phase parity, as mbar_wait, that gives up for a wait that ran out and for nothing else: what a call
// reports about its data stays in the status word until it is read, and the next calls are right all the same.
__device__ __forceinline__ bool tree_wait(uint64_t* bar, uint32_t parity, uint32_t* status, uint32_t site) {
  if (mbar_test(bar, parity)) return true;
  const uint64_t start = global_timer_ns();
  uint32_t spins = 0;
  while (!mbar_test(bar, parity)) {
    if ((++spins & 0x3ffu) == 0) {
      if ((*reinterpret_cast<volatile uint32_t*>(status) & 0xffu) == kWaitTimeout) return false;   // someone else gave up
      if (global_timer_ns() - start > kWaitLimitNs) {
        atomicExch(status, (site << 8) | kWaitTimeout);
        return false;
      }
    }
  }
  return true;
}

// ---- output ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ bool gate_in_pieces(const TreeArgs& a) {   // of eight channels, 16-byte aligned
  return a.gate_is_bf16 && a.gate_token % 8 == 0 && a.gate_head % 8 == 0 && (reinterpret_cast<uintptr_t>(a.gate) & 15u) == 0;
}
// Eight neighbouring channels of one output row (bf16).
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

// tree_decode_merge.cu: 4-D map of a page pool (column, KV head, token in page, page); a box is `tokens` tokens of `columns`
// channels of one KV head, swizzled over 128 or 64 bytes or not (0); zeros outside the pool.  It takes pools whose
// pages `tokens` divides, or one page per sequence, with strides that a map can hold.
bool tree_pool_fits(const TreeArgs& a, int tokens);
bool tree_pool_map(CUtensorMap* map, const void* base, const TreeArgs& a, int tokens, int columns, int swizzle);

// tree_decode_merge.cu: launched behind the kernel that leaves the parts, by programmatic dependent launch
cudaError_t tree_decode_merge(cudaStream_t stream, const TreeArgs& a, const LineShape& shape);

}  // namespace pluto
