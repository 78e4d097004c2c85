// Merges the parts of the units that the cuts of the line (tree_line.cuh) fall into, in the order of the keys:
//   out = sum_c 2^(m_c - m) acc_c / sum_c 2^(m_c - m) l_c,   m = max_c m_c.
// A CTA per unit and eight rows, a warp per row; the parts' weights are computed by the lanes, 32 parts at a
// time, and the sums run over the parts in order with a lane owning eight channels.
#include "tree_line.cuh"

namespace pluto {
namespace {

__global__ void __launch_bounds__(256) tree_decode_merge_kernel(TreeArgs a, LineShape shape, int groups_at_most) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, row = blockIdx.y * 8 + warp;
  const int per_sequence = a.kv_heads * groups_at_most, b = blockIdx.x / per_sequence;
  // (lengths and counts were there before the kernel that this one waits for)
  long long start;
  const Line line = measure_line(a, shape, lane, b, start);
  const Sequence s = sequence_at(a, shape, b);
  pdl_wait();   // the parts are complete and visible from here on
  // the sequence's units in their order, kv_head * groups + group; this block's may not exist
  const int unit = blockIdx.x % per_sequence;
  if (unit >= s.units || line.total == 0) return;
  start += static_cast<long long>(unit) * (s.tiles + shape.overhead);
  const long long end = start + s.tiles + shape.overhead;
  const int group = a.q_heads / a.kv_heads, groups = s.units / a.kv_heads, kv_head = unit / groups;
  const int row0 = unit % groups * shape.rows, rows = min(shape.rows, s.count * group - row0);
  if (row >= rows) return;
  // the workers that hold tiles of it
  int guess = static_cast<int>(start * line.parts / line.total);
  while (guess > 0 && range_begin(line, guess) > start) --guess;
  while (guess + 1 < line.parts && range_begin(line, guess + 1) <= start) ++guess;
  int first = -1, last = -1;
  for (int c = guess; c < line.parts && range_begin(line, c) < end; ++c)
    if (min(range_begin(line, c + 1), end) > max(range_begin(line, c), start + shape.overhead)) {
      if (first < 0) first = c;
      last = c;
    }
  if (first == last) return;   // one worker holds all of its tiles and has written it out
  const Partials parts = partials_of(a, shape);
  const auto part_at = [&](int c) {
    return static_cast<size_t>(2 * c + (start < range_begin(line, c) ? 0 : 1)) * parts.rows + row;
  };
  float m = -INFINITY;
  for (int c = first + lane; c <= last; c += 32) m = fmaxf(m, parts.ml[part_at(c)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float m_safe = m == -INFINITY ? 0.0f : m;
  float l = 0.0f, acc[8] = {};
  const int D = a.dim;
  for (int c0 = first; c0 <= last; c0 += 32) {
    const int c = c0 + lane;
    const float2 own = c <= last ? parts.ml[part_at(c)] : make_float2(-INFINITY, 0.0f);
    const float weight = fast_exp2(own.x - m_safe);
    const int n = min(32, last - c0 + 1);
#pragma unroll 8
    for (int u = 0; u < n; ++u) {
      const float w = __shfl_sync(0xffffffffu, weight, u);
      l = fmaf(__shfl_sync(0xffffffffu, own.y, u), w, l);
      if (lane * 8 < D) {
        const float4* from = reinterpret_cast<const float4*>(parts.acc + part_at(c0 + u) * D + lane * 8);
        const float4 x = from[0], y = from[1];
        acc[0] = fmaf(x.x, w, acc[0]); acc[1] = fmaf(x.y, w, acc[1]); acc[2] = fmaf(x.z, w, acc[2]); acc[3] = fmaf(x.w, w, acc[3]);
        acc[4] = fmaf(y.x, w, acc[4]); acc[5] = fmaf(y.y, w, acc[5]); acc[6] = fmaf(y.z, w, acc[6]); acc[7] = fmaf(y.w, w, acc[7]);
      }
    }
  }
  const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
  const int r = row0 + row, node = r / group, head = kv_head * group + r % group;
  const size_t token = static_cast<size_t>(b) * a.nodes + node;
  if (lane * 8 < D) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= inverse;
    store_out8(a, token, head, lane * 8, acc, gate_in_pieces(a));
  }
  if (lane == 0 && a.lse) a.lse[token * a.q_heads + head] = m_safe * 0.6931471805599453f + logf(l);
}

}  // namespace

cudaError_t tree_decode_merge(cudaStream_t stream, const TreeArgs& a, const LineShape& shape) {
  const int groups = (a.nodes * (a.q_heads / a.kv_heads) + shape.rows - 1) / shape.rows;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(a.batch) * a.kv_heads * groups, (slot_rows(shape, a.nodes, a.q_heads, a.kv_heads) + 7) / 8);
  config.blockDim = dim3(256);
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, tree_decode_merge_kernel, a, shape, groups);
}

}  // namespace pluto
