// extern "C" entry points of decoding with drafted tokens and of the 8-bit cache: argument validation and
// dispatch.  Nothing is queued before every check has passed.
#include <math.h>

#include "../../include/pluto_b200.h"
#include "engine.h"

namespace pluto {
int report(int code, const char* message);
int report_cuda(cudaError_t e, const char* what);
}  // namespace pluto

namespace {

using pluto::report;

bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
size_t bytes_of(int dtype) { return dtype == PLUTO_FP32 ? 4 : 2; }   // of an activation type
bool activation(int dtype) { return dtype == PLUTO_FP32 || dtype == PLUTO_BF16; }
bool fits_int(long long a, long long b, long long c) { return a * b <= 0x7fffffff && a * b * c <= 0x7fffffff; }

int fill_pool(pluto::DraftPool* p, const pluto_kv_cache* cache, const pluto_kv_scales* scales, int kv_heads,
              int head_dim) {
  if (!cache) return report(PLUTO_E_INVALID, "attention requires non-null device pointers");
  if (cache->k_bases || cache->v_bases)
    return report(PLUTO_E_UNIMPLEMENTED, "drafted tokens and 8-bit caches take one pool, not separate caches");
  if (!cache->k_base || !cache->v_base) return report(PLUTO_E_INVALID, "attention requires non-null device pointers");
  if (!activation(cache->dtype) && cache->dtype != PLUTO_E4M3)
    return report(PLUTO_E_INVALID, "attention cache has an unknown dtype");
  const size_t element = cache->dtype == PLUTO_FP32 ? 4 : cache->dtype == PLUTO_BF16 ? 2 : 1;
  if (cache->page_size <= 0 || (cache->block_table && (cache->max_blocks <= 0 || cache->num_pages <= 0)) ||
      cache->token_stride < static_cast<size_t>(kv_heads) * head_dim || cache->page_stride < cache->token_stride ||
      !aligned_to(cache->k_base, element) || !aligned_to(cache->v_base, element) || !aligned_to(cache->block_table, 4))
    return report(PLUTO_E_INVALID, "attention cache shape or capacity does not match parameters");
  if ((cache->dtype == PLUTO_E4M3) != (scales != nullptr))
    return report(PLUTO_E_INVALID, "an 8-bit cache needs its scales, and only that");
  if (scales && (!scales->k || !scales->v)) return report(PLUTO_E_INVALID, "attention requires non-null device pointers");
  if (scales && (scales->token_stride < static_cast<size_t>(kv_heads) || scales->page_stride < scales->token_stride))
    return report(PLUTO_E_INVALID, "attention cache shape or capacity does not match parameters");
  *p = pluto::DraftPool{};
  p->k = cache->k_base; p->v = cache->v_base;
  p->table = cache->block_table;
  p->max_blocks = cache->max_blocks; p->page_size = cache->page_size; p->num_pages = cache->num_pages;
  p->store = cache->dtype == PLUTO_FP32 ? pluto::kStoreFp32 : cache->dtype == PLUTO_BF16 ? pluto::kStoreBf16 : pluto::kStoreE4m3;
  p->page_stride = cache->page_stride; p->token_stride = cache->token_stride;
  if (scales) {
    p->k_scales = scales->k; p->v_scales = scales->v;
    p->scale_page = scales->page_stride; p->scale_token = scales->token_stride;
  }
  return PLUTO_OK;
}

// The last step before a launch: every argument has been checked.
int take_status(uint32_t** status) {
  *status = pluto::kernel_status_word();
  return *status ? PLUTO_OK : report(PLUTO_E_INTERNAL, "kernel status word unavailable");
}

int fill_kv8(pluto::Kv8Args* a, const void* k, const void* v, int dtype, size_t batch_stride, size_t token_stride,
             size_t head_stride, const pluto_kv_cache* cache, const pluto_kv_scales* scales, const int32_t* positions,
             const int32_t* counts, int batch, int tokens, int kv_heads, int head_dim) {
  if (batch <= 0 || tokens <= 0 || kv_heads <= 0 || head_dim <= 0 || head_dim > 256 || !activation(dtype) ||
      !fits_int(batch, tokens, kv_heads))
    return report(PLUTO_E_INVALID, "invalid 8-bit cache dimensions or parameters");
  if (cache && cache->dtype != PLUTO_E4M3) return report(PLUTO_E_INVALID, "the cache is not an 8-bit one");
  if (!k || !v) return report(PLUTO_E_INVALID, "attention requires non-null device pointers");
  const size_t element = dtype == PLUTO_BF16 ? 2 : 4;
  if (!aligned_to(k, element) || !aligned_to(v, element) || !aligned_to(positions, 4) || !aligned_to(counts, 4) || (kv_heads > 1 && head_stride < static_cast<size_t>(head_dim)))
    return report(PLUTO_E_INVALID, "invalid 8-bit cache dimensions or parameters");
  *a = pluto::Kv8Args{};
  if (int c = fill_pool(&a->pool, cache, scales, kv_heads, head_dim)) return c;
  a->k = const_cast<void*>(k); a->v = const_cast<void*>(v);
  a->batch_stride = batch_stride; a->token_stride = token_stride; a->head_stride = head_stride;
  a->is_bf16 = dtype == PLUTO_BF16;
  a->positions = positions; a->counts = counts;
  a->batch = batch; a->tokens = tokens; a->heads = kv_heads; a->dim = head_dim;
  return take_status(&a->pool.status);
}

bool draft_shape(int batch, int nodes, int q_heads, int kv_heads, int head_dim) {
  return batch > 0 && nodes > 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 && q_heads <= 65535 && head_dim > 0 &&
         head_dim <= 256 && batch <= 65535 && fits_int(batch, nodes, q_heads);
}

bool tensor_core_shape(const pluto::TreeArgs& a) {
  const size_t element = a.pool.store == pluto::kStoreBf16 ? 2 : 1;
  return a.q_is_bf16 && a.out_is_bf16 && a.pool.store != pluto::kStoreFp32 && (a.dim == 64 || a.dim == 128 || a.dim == 256) &&
         aligned_to(a.q, 16) && aligned_to(a.out, 16) && aligned_to(a.pool.k, 16) && aligned_to(a.pool.v, 16) &&
         a.pool.page_stride * element % 16 == 0 && a.pool.token_stride * element % 16 == 0;
}

}  // namespace

extern "C" {

int pluto_kv8_append(pluto_stream_t stream, const void* k, const void* v, int dtype, size_t batch_stride,
                     size_t token_stride, size_t head_stride, const pluto_kv_cache* cache, const pluto_kv_scales* scales,
                     const int32_t* positions, const int32_t* counts, int batch, int tokens, int kv_heads, int head_dim) {
  pluto::Kv8Args a;
  if (int c = fill_kv8(&a, k, v, dtype, batch_stride, token_stride, head_stride, cache, scales, positions, counts, batch,
                       tokens, kv_heads, head_dim))
    return c;
  return pluto::report_cuda(pluto::kv8_append(stream, a), "8-bit cache append");
}

int pluto_kv8_read(pluto_stream_t stream, void* k, void* v, int dtype, size_t batch_stride, size_t token_stride,
                   size_t head_stride, const pluto_kv_cache* cache, const pluto_kv_scales* scales, const int32_t* positions,
                   const int32_t* counts, int batch, int tokens, int kv_heads, int head_dim) {
  pluto::Kv8Args a;
  if (int c = fill_kv8(&a, k, v, dtype, batch_stride, token_stride, head_stride, cache, scales, positions, counts, batch,
                       tokens, kv_heads, head_dim))
    return c;
  return pluto::report_cuda(pluto::kv8_read(stream, a), "8-bit cache read");
}

int pluto_kv_keep(pluto_stream_t stream, const pluto_kv_cache* cache, const pluto_kv_scales* scales, const int32_t* prefix_lens,
                  const int32_t* path, const int32_t* accepted, int batch, int nodes, int kv_heads, int head_dim) {
  if (!draft_shape(batch, nodes, kv_heads, kv_heads, head_dim) || nodes > pluto::kMaxDraftNodes)
    return report(PLUTO_E_INVALID, "invalid draft dimensions or parameters");
  pluto::KeepArgs a{};
  if (int c = fill_pool(&a.pool, cache, scales, kv_heads, head_dim)) return c;
  if (!prefix_lens || !path || !accepted) return report(PLUTO_E_INVALID, "attention requires non-null device pointers");
  if (!aligned_to(prefix_lens, 4) || !aligned_to(path, 4) || !aligned_to(accepted, 4))
    return report(PLUTO_E_INVALID, "attention tensors are not aligned to their elements");
  a.prefix = prefix_lens; a.path = path; a.accepted = accepted;
  a.batch = batch; a.nodes = nodes; a.heads = kv_heads; a.dim = head_dim;
  if (int c = take_status(&a.pool.status)) return c;
  return pluto::report_cuda(pluto::kv_keep(stream, a), "cache rows of the accepted path");
}

int pluto_draft_prepare(pluto_stream_t stream, const void* q_in, const void* k_in, const void* v_in, int in_dtype,
                        size_t q_token_stride, size_t q_head_stride, const float* q_norm, const float* k_norm,
                        const int32_t* prefix_lens, const int32_t* parents, const int32_t* counts, void* q_out,
                        int q_out_dtype, const pluto_kv_cache* cache, const pluto_kv_scales* scales, int batch, int nodes,
                        int q_heads, int kv_heads, int head_dim, int rotary_dim, float rms_norm_epsilon, float rope_theta,
                        int round_to_bf16) {
  if (!draft_shape(batch, nodes, q_heads, kv_heads, head_dim) || (parents && nodes > pluto::kMaxDraftNodes) || rotary_dim <= 0 ||
      rotary_dim > head_dim || rotary_dim % 2 != 0 || !isfinite(rope_theta) || rope_theta <= 0.0f ||
      !isfinite(rms_norm_epsilon) || rms_norm_epsilon <= 0.0f || !activation(in_dtype) || !activation(q_out_dtype))
    return report(PLUTO_E_INVALID, "invalid full-attention dimensions or parameters");
  pluto::DraftPrepareArgs d{};
  if (int c = fill_pool(&d.pool, cache, scales, kv_heads, head_dim)) return c;
  if (!q_in || !k_in || !v_in || !q_norm || !k_norm || !q_out)
    return report(PLUTO_E_INVALID, "attention requires non-null device pointers");
  if (!aligned_to(q_in, bytes_of(in_dtype)) || !aligned_to(k_in, bytes_of(in_dtype)) || !aligned_to(v_in, bytes_of(in_dtype)) ||
      !aligned_to(q_out, bytes_of(q_out_dtype)) || !aligned_to(q_norm, 4) || !aligned_to(k_norm, 4) || !aligned_to(prefix_lens, 4) ||
      !aligned_to(parents, 4) || !aligned_to(counts, 4))
    return report(PLUTO_E_INVALID, "attention tensors are not aligned to their elements");
  pluto::PrepareArgs& a = d.p;
  a.q_in = q_in; a.k_in = k_in; a.v_in = v_in; a.in_is_bf16 = in_dtype == PLUTO_BF16;
  a.q_token = q_token_stride; a.q_head = q_head_stride;
  a.q_norm = q_norm; a.k_norm = k_norm; a.positions = prefix_lens;
  a.q_out = q_out; a.q_out_is_bf16 = q_out_dtype == PLUTO_BF16;
  a.batch = batch; a.tokens = nodes; a.q_heads = q_heads; a.kv_heads = kv_heads;
  a.head_dim = head_dim; a.rotary = rotary_dim;
  a.epsilon = rms_norm_epsilon; a.log_theta = logf(rope_theta); a.round = round_to_bf16;
  d.parents = parents; d.counts = counts;
  if (int c = take_status(&d.pool.status)) return c;
  return pluto::report_cuda(pluto::draft_prepare(stream, d), "prepare drafted tokens");
}

size_t pluto_gqa_tree_decode_workspace_bytes(int batch, int nodes, int q_heads, int kv_heads, int head_dim) {
  if (!draft_shape(batch, nodes, q_heads, kv_heads, head_dim) || nodes > pluto::kMaxDraftNodes) return 0;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 16;
  // which kernel runs goes by the cache as well, which is not asked for here
  const size_t few = pluto::tree_decode_mma_workspace_bytes(nodes, q_heads, kv_heads, head_dim);
  const size_t many = pluto::tree_decode_tc_workspace_bytes(nodes, q_heads, kv_heads, head_dim);
  return few > many ? few : many;
}

int pluto_gqa_tree_decode(pluto_stream_t stream, const void* q, int q_dtype, const void* gate, int gate_dtype,
                          size_t gate_token_stride, size_t gate_head_stride, const pluto_kv_cache* cache,
                          const pluto_kv_scales* scales, const int32_t* prefix_lens, int max_prefix_len, const int32_t* parents,
                          const int32_t* counts, void* out, int out_dtype, float* lse, void* workspace,
                          size_t workspace_bytes, int batch, int nodes, int q_heads, int kv_heads, int head_dim,
                          int round_to_bf16) {
  if (!draft_shape(batch, nodes, q_heads, kv_heads, head_dim) || nodes > pluto::kMaxDraftNodes || max_prefix_len < 0 ||
      max_prefix_len > 0x7fffffff - 1024 ||   // (slots rounded up to whole tiles stay 32-bit)
       !activation(q_dtype) || !activation(out_dtype) ||
      (gate && !activation(gate_dtype)))
    return report(PLUTO_E_INVALID, "invalid full-attention dimensions or parameters");
  pluto::TreeArgs a{};
  if (int c = fill_pool(&a.pool, cache, scales, kv_heads, head_dim)) return c;
  if (!q || !prefix_lens || !out || !workspace) return report(PLUTO_E_INVALID, "attention requires non-null device pointers");
  if (!aligned_to(q, bytes_of(q_dtype)) || !aligned_to(out, bytes_of(out_dtype)) || (gate && !aligned_to(gate, bytes_of(gate_dtype))) ||
      !aligned_to(lse, 4) || !aligned_to(prefix_lens, 4) || !aligned_to(parents, 4) || !aligned_to(counts, 4))
    return report(PLUTO_E_INVALID, "attention tensors are not aligned to their elements");
  if (workspace_bytes < pluto_gqa_tree_decode_workspace_bytes(batch, nodes, q_heads, kv_heads, head_dim) ||
      !aligned_to(workspace, 16))
    return report(PLUTO_E_INVALID, "attention decode workspace is too small or misaligned");
  a.q = q; a.q_is_bf16 = q_dtype == PLUTO_BF16;
  a.gate = gate; a.gate_is_bf16 = gate_dtype == PLUTO_BF16;
  a.gate_token = gate_token_stride; a.gate_head = gate_head_stride;
  a.prefix = prefix_lens; a.max_prefix = max_prefix_len;
  a.parents = parents; a.counts = counts;
  a.out = out; a.out_is_bf16 = out_dtype == PLUTO_BF16; a.lse = lse;
  a.workspace = workspace;
  a.batch = batch; a.nodes = nodes; a.q_heads = q_heads; a.kv_heads = kv_heads; a.dim = head_dim;
  a.round = round_to_bf16;
  a.group = q_heads / kv_heads;
  a.scale = 1.0f / sqrtf(static_cast<float>(head_dim));
  if (int c = take_status(&a.pool.status)) return c;
  const bool tensor_cores = tensor_core_shape(a);
  return pluto::report_cuda(tensor_cores && pluto::tree_decode_mma_supported(a)  ? pluto::tree_decode_mma(stream, a)
                            : tensor_cores && pluto::tree_decode_tc_supported(a) ? pluto::tree_decode_tc(stream, a)
                                                                                 : pluto::tree_decode_exact(stream, a),
                            "attention of drafted tokens");
}

int pluto_verify_drafts(pluto_stream_t stream, const void* target_probs, const void* draft_probs, int dtype,
                        const int32_t* tokens, const float* accept_uniforms, const float* sample_uniforms,
                        const int32_t* parents, const int32_t* counts, int32_t* accepted, int32_t* path, int32_t* out_tokens,
                        int batch, int nodes, int vocab) {
  if (batch <= 0 || batch > 65535 || nodes <= 0 || nodes > pluto::kMaxDraftNodes || vocab <= 0 || vocab > 1048576 ||
      !activation(dtype))
    return report(PLUTO_E_INVALID, "invalid draft dimensions or parameters");
  if (parents && draft_probs)
    return report(PLUTO_E_UNIMPLEMENTED, "draft probabilities are taken for chains, not for trees");
  if (!target_probs || !tokens || !accept_uniforms || !sample_uniforms || !accepted || !path || !out_tokens)
    return report(PLUTO_E_INVALID, "draft verification requires non-null device pointers");
  if (!aligned_to(target_probs, bytes_of(dtype)) || !aligned_to(draft_probs, bytes_of(dtype)) || !aligned_to(tokens, 4) ||
      !aligned_to(accept_uniforms, 4) || !aligned_to(sample_uniforms, 4) || !aligned_to(parents, 4) || !aligned_to(counts, 4) ||
      !aligned_to(accepted, 4) || !aligned_to(path, 4) || !aligned_to(out_tokens, 4))
    return report(PLUTO_E_INVALID, "draft verification tensors are not aligned to their elements");
  pluto::VerifyArgs a{};
  a.target = target_probs; a.draft = draft_probs; a.is_bf16 = dtype == PLUTO_BF16;
  a.tokens = tokens; a.parents = parents; a.counts = counts;
  a.accept = accept_uniforms; a.sample = sample_uniforms;
  a.accepted = accepted; a.path = path; a.out = out_tokens;
  a.batch = batch; a.nodes = nodes; a.vocab = vocab;
  if (int c = take_status(&a.status)) return c;
  return pluto::report_cuda(pluto::verify_drafts(stream, a), "verify drafted tokens");
}

}  // extern "C"
