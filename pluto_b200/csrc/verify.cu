// Verification of drafted tokens against the target model's probabilities, from given random numbers.  The
// reference decodes greedily one token at a time (src/llm/generate_greedy_continuation.*) and has no
// counterpart.
//
// Row r of `target` is the target's distribution after node r - 1 (row 0: after the last cached token).
//   chain (no parents): node i was drawn from row i of `draft`; it is accepted, if all before it were, when
//     u_i * q(x_i) < p(x_i).  The first one refused leaves max(p - q, 0) to draw the last token from.  Without
//     `draft` the drafts were given, not drawn: q is one at the drafted token.
//   tree: given drafts.  The children of the last accepted node are tried in order; child c is accepted when
//     u_c * (1 - sum of the p of the siblings tried before) < p(x_c), a token tried before never.  When none is
//     left, the last token is drawn from p without the tried tokens.
// The last token is the smallest x with p'(0) + ... + p'(x) > u * (sum of p'), p' the distribution it is drawn
// from; where nothing is left of it, the target's row itself; -1 where that row's sum is not positive and finite.
//
// Comparisons and sums are in double: products of two fp32 numbers are exact there, and sums of a row agree
// to 1e-16 in any order, so the token does not depend on how the row was cut (by the batch) unless a running sum comes that
// close to the threshold.
//
// The tests of all nodes are independent given the p of the drafted tokens, so a thread takes a node and only
// the walk along the accepted path is serial.  What costs is the one row the last token is drawn from (two with
// `draft`): a cluster of CTAs shares it, a warp per contiguous chunk, and the chunks' sums meet in distributed shared
// memory.  The CTA whose chunk holds the threshold cuts that chunk over its threads and looks for the token, by sums
// over threads first.  A pass of the serial parts (tests, walk, scans, two barriers of the cluster) takes longer than
// the row, so eight CTAs share it only while all clusters are resident at once, else four.  Chains of 8, 131071 tokens, us with
// eight against four: 1 chain 8.6 : 11.7, 32 chains 12.4 : 12.8, 38 17.6 : 17.3, 64 25 : 20, 128 53 : 42.  64 chains are 3.3 TB/s of
// the two rows; one chain of 5, 50257 tokens: 7.0 us.
#include "common.cuh"
#include "engine.h"

namespace pluto {
namespace {

constexpr int kMaxParts = 8, kThreads = 512, kWarps = kThreads / 32;
constexpr int kUnroll = 8;

template <bool kBf16>
__device__ __forceinline__ float prob(const void* p, size_t at) {
  return kBf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]) : static_cast<const float*>(p)[at];
}

__device__ __forceinline__ double lds_cluster_f64(const double* own, uint32_t rank) {
  uint64_t v;
  asm volatile(
      "{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.b64 %0, [a];\n\t}"
      : "=l"(v)
      : "r"(smem_u32(own)), "r"(rank)
      : "memory");
  return __longlong_as_double(static_cast<long long>(v));
}

// What of the row is left at token x: 0 for a tried token, p - q, or p.
template <bool kBf16>
__device__ __forceinline__ double left_at(const void* p, size_t p0, const void* q, size_t q0, const uint32_t* tried,
                                          int first, int x) {
  const double value = prob<kBf16>(p, p0 + x);
  if (q != nullptr) {
    const double rest = value - static_cast<double>(prob<kBf16>(q, q0 + x));
    return rest < 0.0 ? 0.0 : rest;   // (NaN stays)
  }
  return tried != nullptr && (tried[(x - first) >> 5] >> ((x - first) & 31) & 1u) ? 0.0 : value;
}

// Inclusive sums over the lanes of a warp.
__device__ __forceinline__ double warp_scan(double x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double other = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += other;
  }
  return x;
}

// One cluster per sequence, `parts` CTAs; chunk: tokens of a warp, a multiple of 32.
template <bool kBf16>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(VerifyArgs a, int parts, int chunk) {
  extern __shared__ uint32_t tried[];      // one bit per token of this CTA's slice
  __shared__ double p_of[kMaxDraftNodes], sums[2][kWarps], all[kMaxParts * kWarps];
  __shared__ int token_of[kMaxDraftNodes], parent_of[kMaxDraftNodes], child_of[kMaxDraftNodes + 1];
  __shared__ uint8_t good[kMaxDraftNodes], repeated[kMaxDraftNodes];
  __shared__ int path[kMaxDraftNodes], accepted, last, any_tried, first_over, last_some;
  const int b = blockIdx.y, part = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32, i = threadIdx.x;
  const size_t node0 = static_cast<size_t>(b) * a.nodes, row0 = static_cast<size_t>(b) * (a.nodes + 1);
  int count = a.nodes;
  if (a.counts != nullptr) {
    count = a.counts[b];
    if (count < 0 || count > a.nodes) {
      report_status(a.status, 43, kBadLength);
      count = count < 0 ? 0 : a.nodes;
    }
  }
  const bool tree = a.parents != nullptr;
  if (i <= kMaxDraftNodes) child_of[i] = -1;
  bool fits = false;
  double u = 0.0;
  int token = 0, parent = 0;
  if (i < a.nodes) {   // (beside the count)
    token = a.tokens[node0 + i];
    parent = tree ? a.parents[node0 + i] : i - 1;
    u = a.accept[node0 + i];
  }
  if (i < count) {
    fits = token >= 0 && token < a.vocab && parent >= -1 && parent < i;
    if (!fits) report_status(a.status, 43, kBadDraft);
    const double p = fits ? static_cast<double>(prob<kBf16>(a.target, (row0 + parent + 1) * a.vocab + token)) : 0.0;
    token_of[i] = fits ? token : -1;
    parent_of[i] = fits ? parent : -2;   // never anybody's child
    p_of[i] = p;
    if (!tree) {
      const double q = a.draft == nullptr ? 1.0 : fits ? static_cast<double>(prob<kBf16>(a.draft, (node0 + i) * a.vocab + token)) : 0.0;
      good[i] = fits && u * q < p;
    }
  }
  __syncthreads();
  if (tree) {
    bool again = false;   // a token that an earlier sibling had already carries no probability any more
    if (i < count) {
      for (int j = 0; j < i; ++j) again = again || (parent_of[j] == parent_of[i] && token_of[j] == token_of[i]);
      repeated[i] = again;
    }
    __syncthreads();
    if (i < count) {
      double left = 1.0;
      for (int j = 0; j < i; ++j)
        if (parent_of[j] == parent_of[i] && !repeated[j]) left -= p_of[j];
      good[i] = fits && !again && u * left < p_of[i];
    }
    __syncthreads();
    if (i < count && good[i]) {
      bool first = true;   // the siblings before it are tried first
      for (int j = 0; j < i; ++j) first = first && !(parent_of[j] == parent_of[i] && good[j]);
      if (first) child_of[parent_of[i] + 1] = i;
    }
  } else if (i < count && good[i]) {
    child_of[i] = i;
  }
  __syncthreads();
  if (i == 0) {
    int n = 0, node = -1;
    for (int next = child_of[0]; next >= 0; next = child_of[next + 1]) path[n++] = node = next;
    accepted = n;
    last = node;
    any_tried = 0;
    first_over = kThreads;
    last_some = -1;
  }
  const int first_token = part * kWarps * chunk;
  const bool drop = tree || a.draft == nullptr;
  if (drop)
    for (int w = i; w < kWarps * chunk / 32; w += kThreads) tried[w] = 0u;
  __syncthreads();
  if (drop && i < count && parent_of[i] == last) {
    const int x = token_of[i] - first_token;
    if (tree || i == accepted) {
      any_tried = 1;
      if (x >= 0 && x < kWarps * chunk) atomicOr(&tried[x >> 5], 1u << (x & 31));
    }
  }
  if (part == 0) {
    for (int n = i; n < a.nodes; n += kThreads) a.path[node0 + n] = n < accepted ? path[n] : -1;
    for (int n = i; n <= a.nodes; n += kThreads)
      if (n != accepted) a.out[static_cast<size_t>(b) * (a.nodes + 1) + n] = n < accepted ? token_of[path[n]] : -1;
    if (i == 0) a.accepted[b] = accepted;
  }
  __syncthreads();

  const size_t p0 = (row0 + last + 1) * a.vocab, q0 = (node0 + accepted) * a.vocab;
  const int begin = min(a.vocab, first_token + warp * chunk), end = min(a.vocab, begin + chunk);
  // what is left after the refusals, or the row itself; then the row itself where nothing is left
  const void* q = !tree && accepted < count ? a.draft : nullptr;
  const uint32_t* gone = drop && any_tried ? tried : nullptr;
  // Sums of the chunks: lane's chunks lane * 4 to + 3 (unused ones hold 0)
  const int chunks = parts * kWarps;
  double total = 0.0, own[4], upto = 0.0;
  for (int attempt = 0; attempt < 2; ++attempt) {
    double sum = 0.0;
    for (int x0 = begin + lane; x0 < end; x0 += 32 * kUnroll) {
      float v[kUnroll], w[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int x = x0 + 32 * k;
        v[k] = x < end ? prob<kBf16>(a.target, p0 + x) : 0.0f;
        w[k] = q != nullptr && x < end ? prob<kBf16>(q, q0 + x) : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int x = x0 + 32 * k;
        if (gone != nullptr && x < end && (gone[(x - first_token) >> 5] >> ((x - first_token) & 31) & 1u)) v[k] = 0.0f;
        const double rest = static_cast<double>(v[k]) - static_cast<double>(w[k]);
        sum += q != nullptr && rest < 0.0 ? 0.0 : rest;   // (NaN stays)
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sums[attempt][warp] = sum;
    cluster_sync();
    if (i < kMaxParts * kWarps) all[i] = i < chunks ? lds_cluster_f64(&sums[attempt][i % kWarps], i / kWarps) : 0.0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) own[k] = all[lane * 4 + k];
    upto = warp_scan((own[0] + own[1]) + (own[2] + own[3]), lane);
    total = __shfl_sync(0xffffffffu, upto, 31);
    if (total > 0.0 || (q == nullptr && gone == nullptr)) break;
    q = nullptr;
    gone = nullptr;
    __syncthreads();   // all[] is written again
  }
  cluster_arrive();   // this CTA has read the others' sums; it leaves when they have read its own
  int32_t* out = a.out + static_cast<size_t>(b) * (a.nodes + 1) + accepted;
  if (!(total > 0.0) || isinf(total)) {
    if (part == 0 && i == 0) *out = -1;
    cluster_wait();
    return;
  }
  // the chunk that holds the threshold (the last one with anything in it where rounding leaves none)
  const double threshold = static_cast<double>(a.sample[b]) * total;
  double cum = __shfl_up_sync(0xffffffffu, upto, 1), before = 0.0, before_some = 0.0;   // (kept exactly: no difference of sums)
  int over = -1, some = -1;
  if (lane == 0) cum = 0.0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (own[k] > 0.0) {
      some = lane * 4 + k;
      before_some = cum;
      if (over < 0 && cum + own[k] > threshold) {
        over = some;
        before = cum;
      }
    }
    cum += own[k];
  }
  const unsigned overs = __ballot_sync(0xffffffffu, over >= 0), somes = __ballot_sync(0xffffffffu, some >= 0);
  const int from = overs ? __ffs(overs) - 1 : 31 - __clz(somes);
  const int holder = __shfl_sync(0xffffffffu, overs ? over : some, from);
  before = __shfl_sync(0xffffffffu, overs ? before : before_some, from);
  if (holder / kWarps == part) {
    // a few neighbouring tokens per thread
    const int per = (chunk + kThreads - 1) / kThreads;
    const int stop = min(a.vocab, first_token + (holder % kWarps + 1) * chunk);
    const int at = min(stop, first_token + holder % kWarps * chunk + i * per), to = min(stop, at + per);
    double sum = 0.0;
#pragma unroll 4
    for (int x = at; x < to; ++x) sum += left_at<kBf16>(a.target, p0, q, q0, gone, first_token, x);
    const double scanned = warp_scan(sum, lane);
    double below = __shfl_up_sync(0xffffffffu, scanned, 1);
    if (lane == 0) below = 0.0;
    __syncthreads();   // all[] was read by every warp
    if (lane == 31) all[warp] = scanned;
    __syncthreads();
    for (int w = 0; w < warp; ++w) before += all[w];
    below += before;
    if (sum > 0.0) {
      atomicMax(&last_some, i);
      if (below + sum > threshold) atomicMin(&first_over, i);
    }
    __syncthreads();
    if (i == (first_over < kThreads ? first_over : last_some)) {
      int found = -1;
      for (int x = at; x < to; ++x) {
        const double value = left_at<kBf16>(a.target, p0, q, q0, gone, first_token, x);
        below += value;
        if (value > 0.0) {
          found = x;
          if (below > threshold) break;
        }
      }
      *out = found;
    }
  }
  cluster_wait();
}

}  // namespace

cudaError_t verify_drafts(cudaStream_t stream, const VerifyArgs& a) {
  const int parts = a.batch * kMaxParts <= 2 * 148 ? kMaxParts : kMaxParts / 2;
  const int per_warp = (a.vocab + parts * kWarps - 1) / (parts * kWarps), chunk = (per_warp + 31) / 32 * 32;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(parts, a.batch);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = static_cast<size_t>(kWarps) * chunk / 8;
  config.stream = stream;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim = {static_cast<unsigned>(parts), 1, 1};
  config.attrs = &cluster;
  config.numAttrs = 1;
  const cudaError_t e = a.is_bf16 ? cudaLaunchKernelEx(&config, verify_kernel<true>, a, parts, chunk)
                                  : cudaLaunchKernelEx(&config, verify_kernel<false>, a, parts, chunk);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace pluto
