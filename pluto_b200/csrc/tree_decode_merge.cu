// Merges the parts of the units that the cuts of the line (tree_line.cuh) fall into, in the order of the keys:
//   out = sum_c 2^(m_c - m) acc_c / sum_c 2^(m_c - m) l_c,   m = max_c m_c.
// A lane owns eight channels; the order of the additions is fixed.  Few units, of up to a few hundred parts (a short
// batch): a CTA per row, its eight warps take every eighth part each and their sums meet in shared memory (one
// sequence of 777 tokens, 46 parts: 7 us, 35 with a warp per row).  Many units: a warp per row, eight parts in flight
// (192 units of 9 parts, 5 rows: 7 us, 11 with four); units of a part or two: two in flight, for more warps per SM, and
// no more CTAs than fit, as a CTA's look-ups take longer than a row (39040 rows: 26 us, 55 with a warp for every row and
// eight parts).
#include "tree_line.cuh"

namespace pluto {
namespace {

constexpr int kWarps = 8;

template <bool kSplit, int kAhead>   // kAhead: parts in flight
__global__ void __launch_bounds__(kWarps * 32) tree_decode_merge_kernel(TreeArgs a, LineShape shape, int groups_at_most) {
  __shared__ float sums[kSplit ? kWarps : 1][256];
  __shared__ float sum_of_weights[kSplit ? kWarps : 1];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int per_sequence = a.kv_heads * groups_at_most, b = blockIdx.x / per_sequence, unit = blockIdx.x % per_sequence;
  // (lengths and counts were there before the kernel that this one waits for)
  unsigned start;
  const Line line = measure_line(a, shape, lane, b, start);
  const Sequence s = sequence_at(a, shape, b);
  pdl_wait();   // the parts are complete and visible from here on
  // the sequence's units in their order, kv_head * groups + group; this block's may not exist
  const int group = a.group, groups = (s.count * group + (1 << shape.rows_shift) - 1) >> shape.rows_shift;
  if (unit >= a.kv_heads * groups || line.total == 0) return;
  const int kv_head = unit / groups;
  start += (shape.side > 1 ? unit % groups : unit) * (s.tiles + shape.overhead);
  const unsigned end = start + s.tiles + shape.overhead;
  const int row0 = unit % groups << shape.rows_shift, rows = min(1 << shape.rows_shift, s.count * group - row0);
  // the ranges that hold tiles of it
  const int first = static_cast<int>(holder_of(line, start + shape.overhead)), last = static_cast<int>(holder_of(line, end - 1));
  if (first == last) return;   // one worker holds all of its tiles and has written it out
  const Partials parts = partials_of(a, shape);
  // (the whole CTA has a row, or none, where its warps share it)
  for (int row = kSplit ? blockIdx.y : blockIdx.y * kWarps + warp; row < rows; row += kSplit ? rows : gridDim.y * kWarps) {
    const auto part_at = [&](int c) {
      return static_cast<size_t>(2 * (c * shape.side + (shape.side > 1 ? kv_head : 0)) + (start < range_begin(line, c) ? 0 : 1)) * parts.rows + row;
    };
    const int D = a.dim, step = kSplit ? kWarps : 1;
    const bool owns = lane * 8 < D;
    float4 x[kAhead][2];
    float2 ml[kAhead];
    const auto load = [&](int c0) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int c = c0 + u * step;
        if (c > last) break;
        const size_t at = part_at(c);
        ml[u] = parts.ml[at];
        const float4* from = reinterpret_cast<const float4*>(parts.acc + at * D + (owns ? lane * 8 : 0));
        x[u][0] = from[0];
        x[u][1] = from[1];
      }
    };
    int c0 = first + (kSplit ? warp : 0);
    load(c0);   // (before the maximum is known, which takes as long)
    float m = -INFINITY;
    for (int c = first + lane; c <= last; c += 32) m = fmaxf(m, parts.ml[part_at(c)].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float m_safe = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, acc[8] = {};
    while (c0 <= last) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (c0 + u * step > last) break;   // (a weight of zero would not do: nothing was read)
        const float w = fast_exp2(ml[u].x - m_safe);
        l = fmaf(ml[u].y, w, l);
        acc[0] = fmaf(x[u][0].x, w, acc[0]); acc[1] = fmaf(x[u][0].y, w, acc[1]);
        acc[2] = fmaf(x[u][0].z, w, acc[2]); acc[3] = fmaf(x[u][0].w, w, acc[3]);
        acc[4] = fmaf(x[u][1].x, w, acc[4]); acc[5] = fmaf(x[u][1].y, w, acc[5]);
        acc[6] = fmaf(x[u][1].z, w, acc[6]); acc[7] = fmaf(x[u][1].w, w, acc[7]);
      }
      c0 += kAhead * step;
      load(c0);
    }
    const int r = row0 + row, node = r / group, head = kv_head * group + r % group;
    const size_t token = static_cast<size_t>(b) * a.nodes + node;
    if (kSplit) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (owns) sums[warp][lane * 8 + i] = acc[i];
      if (lane == 0) sum_of_weights[warp] = l;
      __syncthreads();
      if (warp > 0) return;
      l = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
      for (int w = 0; w < kWarps; ++w) {
        l += sum_of_weights[w];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += owns ? sums[w][lane * 8 + i] : 0.0f;
      }
    }
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
    if (owns) {
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] *= inverse;
      store_out8(a, token, head, lane * 8, acc, gate_in_pieces(a));
    }
    if (lane == 0 && a.lse) a.lse[token * a.q_heads + head] = m_safe * 0.6931471805599453f + logf(l);
  }
}

}  // namespace

bool tree_pool_fits(const TreeArgs& a, int tokens) {
  const size_t element = a.pool.store == kStoreBf16 ? 2 : 1;
  return (a.pool.table == nullptr || a.pool.max_blocks == 1 || a.pool.page_size % tokens == 0) &&
         a.pool.page_stride * element < (1ull << 40) && a.pool.token_stride * element < (1ull << 40);
}

bool tree_pool_map(CUtensorMap* map, const void* base, const TreeArgs& a, int tokens, int columns, int swizzle) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = [] {
    void* symbol = nullptr;
    cudaDriverEntryPointQueryResult result;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &symbol, cudaEnableDefault, &result) != cudaSuccess ||
        result != cudaDriverEntryPointSuccess)
      return static_cast<Encode>(nullptr);
    return reinterpret_cast<Encode>(symbol);
  }();
  if (encode == nullptr) return false;
  const bool eight = a.pool.store == kStoreE4m3;
  const cuuint64_t element = eight ? 1 : 2;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.dim), static_cast<cuuint64_t>(a.kv_heads), static_cast<cuuint64_t>(a.pool.page_size),
                              static_cast<cuuint64_t>(a.pool.table ? a.pool.num_pages : a.batch)};
  const cuuint64_t strides[3] = {a.dim * element, a.pool.token_stride * element, a.pool.page_stride * element};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(columns), 1, static_cast<cuuint32_t>(tokens), 1}, steps[4] = {1, 1, 1, 1};
  return encode(map, eight ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box,
                steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                swizzle == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : swizzle == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t tree_decode_merge(cudaStream_t stream, const TreeArgs& a, const LineShape& shape) {
  const int groups = (a.nodes * a.group + (1 << shape.rows_shift) - 1) >> shape.rows_shift;
  const int rows = slot_rows(shape, a.nodes, a.q_heads, a.kv_heads);
  const long long units = static_cast<long long>(a.batch) * a.kv_heads * groups;
  // parts of a unit, when the line is long enough for all workers
  const bool many_parts = shape.workers >= 16 * units, few_parts = shape.workers < 2 * units;
  const int row_groups = (rows + kWarps - 1) / kWarps, resident = static_cast<int>(148 * 16 / units) + 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(units), many_parts ? rows : row_groups < resident ? row_groups : resident);
  config.blockDim = dim3(kWarps * 32);
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return many_parts  ? cudaLaunchKernelEx(&config, tree_decode_merge_kernel<true, 8>, a, shape, groups)
         : few_parts ? cudaLaunchKernelEx(&config, tree_decode_merge_kernel<false, 2>, a, shape, groups)
                     : cudaLaunchKernelEx(&config, tree_decode_merge_kernel<false, 8>, a, shape, groups);
}

}  // namespace pluto
