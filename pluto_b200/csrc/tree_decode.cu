// Attention of drafted tokens over a cache, in fp32 arithmetic for every shape, storage type and alignment.
//
// Node i of sequence b holds slot prefix[b] + i and sees the cached slots [0, prefix[b]), its ancestors and itself:
//   out(i, h) = sum_t softmax_t(q(i, h) . k(t) / sqrt(D)) v(t),   t over what i sees.
// A tree of one node is the reference's cached step (src/llm/layers/util/cached_attention_ops.cc:83-126).
//
// A CTA owns a (node, query head).  Its warps take every eighth key, a lane owns up to eight channels, the
// running maximum, sum and accumulator of a warp stay in registers, and the warps' states are merged in
// order.  Keys that a node does not see are skipped, so nothing they hold can reach it.  Nodes from counts[b]
// on are left as they were.  Shapes of the tensor cores take tree_decode_mma.cu or tree_decode_sm100.cu.
#include "draft_rows.cuh"

namespace pluto {
namespace {

constexpr int kWarps = 8;
constexpr int kAhead = 4;   // keys of a warp in flight

__device__ __forceinline__ float stored(const void* p, size_t at, int store) {
  return store == kStoreBf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at])
         : store == kStoreFp32 ? static_cast<const float*>(p)[at]
                               : e4m3_value(static_cast<const uint8_t*>(p)[at]);
}

__global__ void __launch_bounds__(kWarps * 32) tree_decode_exact_kernel(TreeArgs a) {
  __shared__ int parents[kMaxDraftNodes];
  __shared__ int seen[kMaxDraftNodes], seen_count;   // the node's ancestors and itself, rising
  __shared__ float acc_of[kWarps][256], ml_of[kWarps][2];
  const int head = blockIdx.y, b = blockIdx.x / a.nodes, node = blockIdx.x % a.nodes;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, D = a.dim, kv_head = head / (a.q_heads / a.kv_heads);
  if (node >= draft_count(a.counts, b, a.nodes, a.pool.status, 44)) return;
  int prefix = a.prefix[b];
  if (prefix < 0 || prefix > a.max_prefix) {
    if (threadIdx.x == 0) report_status(a.pool.status, 44, kBadLength);
    prefix = prefix < 0 ? 0 : a.max_prefix;
  }
  for (int i = threadIdx.x; i <= node; i += kWarps * 32)
    parents[i] = a.parents ? a.parents[static_cast<size_t>(b) * a.nodes + i] : i - 1;
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = 0;
    for (int i = node; i >= 0;) {
      seen[n++] = i;
      const int up = parents[i];
      if (up < -1 || up >= i) report_status(a.pool.status, 44, kBadDraft);   // taken as a first token's
      i = up < i ? up : -1;
    }
    for (int i = 0; i < n / 2; ++i) {
      const int t = seen[i];
      seen[i] = seen[n - 1 - i];
      seen[n - 1 - i] = t;
    }
    seen_count = n;
  }
  __syncthreads();
  const int keys = prefix + seen_count;
  const size_t row = (static_cast<size_t>(b) * a.nodes + node) * a.q_heads + head;
  float q[8], acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    q[i] = d < D ? stored(a.q, row * D + d, a.q_is_bf16 ? kStoreBf16 : kStoreFp32) : 0.0f;
    acc[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int t0 = warp * kAhead; t0 < keys; t0 += kWarps * kAhead) {
    float k[kAhead][8], v[kAhead][8], factor[kAhead];
    bool live[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int key = t0 + j;
      live[j] = key < keys;
      const int slot = !live[j] ? 0 : key < prefix ? key : prefix + seen[key - prefix];
      const long long page = live[j] ? draft_page(a.pool, b, slot, 45) : -1;
      const bool there = page >= 0;   // a slot without a page reads as zeros
      const size_t at = there ? draft_row(a.pool, page, slot) + static_cast<size_t>(kv_head) * D : 0;
      float kf = 1.0f, vf = 1.0f;
      if (there && a.pool.store == kStoreE4m3) {
        const size_t s = draft_scale(a.pool, page, slot) + kv_head;
        kf = e8m0_value(a.pool.k_scales[s]);
        vf = e8m0_value(a.pool.v_scales[s]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        k[j][i] = there && d < D ? stored(a.pool.k, at + d, a.pool.store) * kf : 0.0f;
        v[j][i] = there && d < D ? stored(a.pool.v, at + d, a.pool.store) * vf : 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) dot = fmaf(k[j][i], q[i], dot);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      factor[j] = live[j] ? dot * a.scale : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (!live[j]) continue;   // (uniform over the warp)
      const float m_new = fmaxf(m, factor[j]);
      const float m_safe = m_new == -INFINITY ? 0.0f : m_new;
      const float correction = expf(m - m_safe), p = expf(factor[j] - m_safe);
      l = l * correction + p;
      m = m_new;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = fmaf(p, v[j][i], acc[i] * correction);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) acc_of[warp][lane + 32 * i] = acc[i];
  if (lane == 0) {
    ml_of[warp][0] = m;
    ml_of[warp][1] = l;
  }
  __syncthreads();
  float m_all = -INFINITY;
  for (int w = 0; w < kWarps; ++w) m_all = fmaxf(m_all, ml_of[w][0]);
  const float m_safe = m_all == -INFINITY ? 0.0f : m_all;
  float l_all = 0.0f;
  for (int w = 0; w < kWarps; ++w) l_all += ml_of[w][1] * expf(ml_of[w][0] - m_safe);
  for (int d = threadIdx.x; d < D; d += kWarps * 32) {
    float sum = 0.0f;
    for (int w = 0; w < kWarps; ++w) sum += acc_of[w][d] * expf(ml_of[w][0] - m_safe);
    float value = l_all == 0.0f ? 0.0f : sum / l_all;   // (nothing but scores of -infinity)
    value = tree_output(a, static_cast<size_t>(b) * a.nodes + node, head, d, value);
    if (a.out_is_bf16) static_cast<__nv_bfloat16*>(a.out)[row * D + d] = __float2bfloat16_rn(value);
    else static_cast<float*>(a.out)[row * D + d] = value;
  }
  if (threadIdx.x == 0 && a.lse) a.lse[row] = m_safe + logf(l_all);
}

}  // namespace

cudaError_t tree_decode_exact(cudaStream_t stream, const TreeArgs& a) {
  tree_decode_exact_kernel<<<dim3(a.batch * a.nodes, a.q_heads), kWarps * 32, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace pluto
