// The 8-bit key/value cache: rows quantised as they are written, read back as the values they hold, and the
// rows of an accepted path moved to the front of the drafts' slots.  The reference keeps its cache in fp32
// (src/llm/key_value_cache.h:25-57) and has none of the three.
//
// Append and read are streams.  A row's channels are dealt to the lanes of a sub-warp, eight consecutive
// ones each (16 bytes of bf16 in, 8 of codes out), so the row maximum is a butterfly over at most 32 lanes
// and no shared memory is used; a sub-warp takes the key and the value row of kRows (token, head) pairs at
// a time, which keeps 2 * kRows loads per lane in flight.  Widths that 8 does not divide and rows off the
// 16-byte boundary take single channels, a warp per row.  Measured (B200, 16 x 8191 tokens, 8 heads of 128, bf16): append
// 154 us, 5.2 TB/s, bound by the issue of its instructions; read 126 us, 6.4 TB/s.  Scale bytes gathered into words
// took longer (177), four rows at a time no less.
#include "draft_rows.cuh"

namespace pluto {
namespace {

constexpr int kRows = 2;

struct RowAt {
  bool live;
  size_t data, pool, scale;   // element offsets: activation row, pool row, scale byte
};

__device__ __forceinline__ RowAt row_at(const Kv8Args& a, unsigned row, uint32_t site) {
  RowAt r{};
  const unsigned h = row % a.heads, token = row / a.heads, t = token % a.tokens, b = token / a.tokens;
  if (b >= static_cast<unsigned>(a.batch) || static_cast<int>(t) >= draft_count(a.counts, b, a.tokens, a.pool.status, site)) return r;
  const long long slot = static_cast<long long>(a.positions ? a.positions[b] : 0) + t;
  const long long page = draft_page(a.pool, b, slot > 0x7fffffff ? -1 : static_cast<int>(slot), site);
  if (page < 0) return r;
  r.live = true;
  r.data = b * a.batch_stride + t * a.token_stride + h * a.head_stride;
  r.pool = draft_row(a.pool, page, static_cast<int>(slot)) + static_cast<size_t>(h) * a.dim;
  r.scale = draft_scale(a.pool, page, static_cast<int>(slot)) + h;
  return r;
}

// The rows of a sub-warp: usually neighbouring heads of one token, which share the look-ups.
__device__ __forceinline__ void rows_at(const Kv8Args& a, unsigned row, uint32_t site, RowAt (&at)[kRows]) {
  at[0] = row_at(a, row, site);
  unsigned h = row % a.heads;
#pragma unroll
  for (int i = 1; i < kRows; ++i) {
    if (++h < static_cast<unsigned>(a.heads)) {
      at[i] = at[i - 1];
      at[i].data += a.head_stride;
      at[i].pool += a.dim;
      at[i].scale += 1;
    } else {
      at[i] = row_at(a, row + i, site);
      h = 0;
    }
  }
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Eight channels as they lie in memory.
template <bool kBf16>
struct Raw8 {
  uint4 w[kBf16 ? 1 : 2];
  __device__ __forceinline__ void load(const void* p, size_t at) {
    const char* from = static_cast<const char*>(p) + at * (kBf16 ? 2 : 4);
#pragma unroll
    for (int i = 0; i < (kBf16 ? 1 : 2); ++i) w[i] = __ldcs(reinterpret_cast<const uint4*>(from) + i);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (kBf16 ? 1 : 2); ++i) w[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void values(float (&x)[8]) const {
    const uint32_t words[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[kBf16 ? 0 : 1].x, w[kBf16 ? 0 : 1].y, w[kBf16 ? 0 : 1].z, w[kBf16 ? 0 : 1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = !kBf16 ? __uint_as_float(words[i]) : i & 1 ? bf16_hi(words[i / 2]) : bf16_lo(words[i / 2]);
  }
};

// Largest magnitude of a row as the bits of an fp32 value (its lanes each hold eight channels).  Magnitudes order as
// integers; bf16 ones are compared two at a time.
template <bool kBf16, int kLanes>
__device__ __forceinline__ uint32_t row_largest(const Raw8<kBf16>& x) {
  if constexpr (kBf16) {
    constexpr uint32_t kAbs = 0x7fff7fffu;
    uint32_t m = max_u16x2(max_u16x2(x.w[0].x & kAbs, x.w[0].y & kAbs), max_u16x2(x.w[0].z & kAbs, x.w[0].w & kAbs));
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) m = max_u16x2(m, __shfl_xor_sync(0xffffffffu, m, o));
    return max(m & 0xffff0000u, m << 16);
  } else {
    float v[8];
    x.values(v);
    uint32_t m = 0u;
#pragma unroll
    for (int u = 0; u < 8; ++u) m = max(m, __float_as_uint(v[u]) & 0x7fffffffu);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
  }
}

// The codes of eight channels; a row that is not finite gets NaN codes.
template <bool kBf16>
__device__ __forceinline__ uint2 codes8(const Raw8<kBf16>& in, uint32_t byte) {
  if (byte == 255u) return make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
  const float f = e8m0_inverse(byte);
  float x[8];
  in.values(x);
  return make_uint2(e4m3_pair(x[0] * f, x[1] * f) | e4m3_pair(x[2] * f, x[3] * f) << 16,
                    e4m3_pair(x[4] * f, x[5] * f) | e4m3_pair(x[6] * f, x[7] * f) << 16);
}

template <bool kBf16, int kLanes>   // lanes per row: dim <= 8 * kLanes
__global__ void __launch_bounds__(256) kv8_append_vec(Kv8Args a) {
  const unsigned group = blockIdx.x * (256u / kLanes) + threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const int c = lane * 8;
  Raw8<kBf16> in[kRows][2];
  RowAt at[kRows];
  rows_at(a, group * kRows, 40, at);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    in[i][0].zero();
    in[i][1].zero();
    if (at[i].live && c < a.dim) {
      in[i][0].load(a.k, at[i].data + c);
      in[i][1].load(a.v, at[i].data + c);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i)
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const uint32_t byte = e8m0_of(row_largest<kBf16, kLanes>(in[i][side]));
      if (!at[i].live) continue;
      if (c < a.dim) *reinterpret_cast<uint2*>(static_cast<uint8_t*>(side ? a.pool.v : a.pool.k) + at[i].pool + c) = codes8(in[i][side], byte);
      if (lane == 0) (side ? a.pool.v_scales : a.pool.k_scales)[at[i].scale] = static_cast<uint8_t>(byte);
    }
}

__device__ __forceinline__ float load1(const void* p, size_t at, int is_bf16) {
  return is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]) : static_cast<const float*>(p)[at];
}
__device__ __forceinline__ void store1(void* p, size_t at, int is_bf16, float x) {
  if (is_bf16) static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(x);
  else static_cast<float*>(p)[at] = x;
}

__global__ void __launch_bounds__(256) kv8_append_any(Kv8Args a) {
  const int lane = threadIdx.x % 32;
  const RowAt at = row_at(a, blockIdx.x * 8u + threadIdx.x / 32, 40);
  if (!at.live) return;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const void* in = side ? a.v : a.k;
    uint8_t* pool = static_cast<uint8_t*>(side ? a.pool.v : a.pool.k) + at.pool;
    uint32_t m = 0u;
    for (int c = lane; c < a.dim; c += 32) m = max(m, __float_as_uint(load1(in, at.data + c, a.is_bf16)) & 0x7fffffffu);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t byte = e8m0_of(m);
    for (int c = lane; c < a.dim; c += 32)
      pool[c] = byte == 255u ? 0x7f : static_cast<uint8_t>(e4m3_pair(load1(in, at.data + c, a.is_bf16) * e8m0_inverse(byte), 0.0f));
    if (lane == 0) (side ? a.pool.v_scales : a.pool.k_scales)[at.scale] = static_cast<uint8_t>(byte);
  }
}

template <bool kBf16>
__device__ __forceinline__ void store8(void* p, size_t at, uint2 codes, float f) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 pair = e4m3_values((i < 2 ? codes.x : codes.y) >> (16 * (i & 1)));
    x[2 * i] = pair.x * f;
    x[2 * i + 1] = pair.y * f;
  }
  if (kBf16) {
    __stcs(reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p) + at),
           make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])));
  } else {
    float4* out = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
    __stcs(out, make_float4(x[0], x[1], x[2], x[3]));
    __stcs(out + 1, make_float4(x[4], x[5], x[6], x[7]));
  }
}

template <bool kBf16, int kLanes>
__global__ void __launch_bounds__(256) kv8_read_vec(Kv8Args a) {
  const unsigned group = blockIdx.x * (256u / kLanes) + threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const int c = lane * 8;
  if (c >= a.dim) return;
  uint2 k[kRows], v[kRows];
  uint32_t kb[kRows], vb[kRows];
  RowAt at[kRows];
  rows_at(a, group * kRows, 41, at);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (at[i].live) {
      k[i] = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.pool.k) + at[i].pool + c);
      v[i] = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.pool.v) + at[i].pool + c);
      kb[i] = a.pool.k_scales[at[i].scale];
      vb[i] = a.pool.v_scales[at[i].scale];
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (at[i].live) {
      store8<kBf16>(a.k, at[i].data + c, k[i], e8m0_value(kb[i]));
      store8<kBf16>(a.v, at[i].data + c, v[i], e8m0_value(vb[i]));
    }
}

__global__ void __launch_bounds__(256) kv8_read_any(Kv8Args a) {
  const int lane = threadIdx.x % 32;
  const RowAt at = row_at(a, blockIdx.x * 8u + threadIdx.x / 32, 41);
  if (!at.live) return;
  const float kf = e8m0_value(a.pool.k_scales[at.scale]), vf = e8m0_value(a.pool.v_scales[at.scale]);
  for (int c = lane; c < a.dim; c += 32) {
    store1(a.k, at.data + c, a.is_bf16, e4m3_value(static_cast<const uint8_t*>(a.pool.k)[at.pool + c]) * kf);
    store1(a.v, at.data + c, a.is_bf16, e4m3_value(static_cast<const uint8_t*>(a.pool.v)[at.pool + c]) * vf);
  }
}

// Eight channels at a time: rows and strides on 16-byte boundaries (8 bytes of codes).
bool vector_rows(const Kv8Args& a) {
  const size_t step = a.is_bf16 ? 8 : 4;
  const auto aligned = [](const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  return a.dim % 8 == 0 && a.batch_stride % step == 0 && a.token_stride % step == 0 && a.head_stride % step == 0 &&
         aligned(a.k, 16) && aligned(a.v, 16) && aligned(a.pool.k, 8) && aligned(a.pool.v, 8) &&
         a.pool.page_stride % 8 == 0 && a.pool.token_stride % 8 == 0;
}

unsigned blocks_for(const Kv8Args& a, int lanes, int rows) {
  const unsigned total = static_cast<unsigned>(a.batch) * a.tokens * a.heads, per_block = 256 / lanes * rows;
  return (total + per_block - 1) / per_block;
}

// Moves the rows of an accepted path to the first slots of the drafts, in place.  A thread owns one piece
// (16 bytes where the rows allow it, and one scale byte of E4M3 storage) of the key or value row and takes
// the path in order, eight rows at a time, loads before stores: entry j comes from slot path[j] >= j, which
// no earlier entry has written, so no barrier is needed.  A path that is not strictly increasing inside
// [0, nodes) is reported and nothing of that sequence moves.
template <typename Piece>
__device__ __forceinline__ void move_rows(char* base, const size_t* rows, const int* path, int count, size_t at) {
  for (int i0 = 0; i0 < count; i0 += 8) {
    Piece x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u < count && path[i0 + u] != i0 + u) x[u] = *reinterpret_cast<const Piece*>(base + rows[path[i0 + u]] + at);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u < count && path[i0 + u] != i0 + u) *reinterpret_cast<Piece*>(base + rows[i0 + u] + at) = x[u];
  }
}

template <typename Piece>
__global__ void __launch_bounds__(128) kv_keep_kernel(KeepArgs a, size_t row_bytes, int element) {
  __shared__ int path[kMaxDraftNodes], bad;
  __shared__ size_t rows[kMaxDraftNodes], scales[kMaxDraftNodes];
  const int b = blockIdx.y;
  int count = a.accepted[b];
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  if (count < 0 || count > a.nodes) {
    if (threadIdx.x == 0) report_status(a.pool.status, 42, kBadDraft);
    return;
  }
  const int prefix = a.prefix[b];
  for (int i = threadIdx.x; i < count; i += 128) {
    const int node = a.path[static_cast<size_t>(b) * a.nodes + i];
    path[i] = node;
    if (node < i || node >= a.nodes || (i > 0 && node <= a.path[static_cast<size_t>(b) * a.nodes + i - 1])) bad = 1;
  }
  __syncthreads();
  if (bad) {
    if (threadIdx.x == 0) report_status(a.pool.status, 42, kBadDraft);
    return;
  }
  const int last = count > 0 ? path[count - 1] : -1;   // the slots beyond it are not touched
  for (int i = threadIdx.x; i <= last; i += 128) {
    const long long slot = static_cast<long long>(prefix) + i;
    const long long page = prefix < 0 || slot > 0x7fffffff ? draft_page(a.pool, b, -1, 42) : draft_page(a.pool, b, static_cast<int>(slot), 42);
    if (page < 0) {
      bad = 1;
    } else {
      rows[i] = draft_row(a.pool, page, static_cast<int>(slot)) * element;
      if (a.pool.store == kStoreE4m3) scales[i] = draft_scale(a.pool, page, static_cast<int>(slot));
    }
  }
  __syncthreads();
  if (bad) return;
  const size_t at = (static_cast<size_t>(blockIdx.x) * 128 + threadIdx.x) * sizeof(Piece);
  if (at < row_bytes) {
    move_rows<Piece>(static_cast<char*>(blockIdx.z ? a.pool.v : a.pool.k), rows, path, count, at);
  } else if (a.pool.store == kStoreE4m3) {
    const size_t head = at / sizeof(Piece) - (row_bytes + sizeof(Piece) - 1) / sizeof(Piece);
    if (head < static_cast<size_t>(a.heads))
      move_rows<uint8_t>(reinterpret_cast<char*>(blockIdx.z ? a.pool.v_scales : a.pool.k_scales), scales, path, count, head);
  }
}

template <bool kBf16, int kLanes>
void launch_vec(cudaStream_t stream, const Kv8Args& a, bool append) {
  const unsigned blocks = blocks_for(a, kLanes, kRows);
  if (append) kv8_append_vec<kBf16, kLanes><<<blocks, 256, 0, stream>>>(a);
  else kv8_read_vec<kBf16, kLanes><<<blocks, 256, 0, stream>>>(a);
}
template <bool kBf16>
void launch_vec(cudaStream_t stream, const Kv8Args& a, bool append) {
  if (a.dim <= 64) launch_vec<kBf16, 8>(stream, a, append);
  else if (a.dim <= 128) launch_vec<kBf16, 16>(stream, a, append);
  else launch_vec<kBf16, 32>(stream, a, append);
}
cudaError_t launch_rows(cudaStream_t stream, const Kv8Args& a, bool append) {
  if (vector_rows(a)) {
    if (a.is_bf16) launch_vec<true>(stream, a, append);
    else launch_vec<false>(stream, a, append);
  } else if (append) {
    kv8_append_any<<<blocks_for(a, 32, 1), 256, 0, stream>>>(a);
  } else {
    kv8_read_any<<<blocks_for(a, 32, 1), 256, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t kv8_append(cudaStream_t stream, const Kv8Args& a) { return launch_rows(stream, a, true); }
cudaError_t kv8_read(cudaStream_t stream, const Kv8Args& a) { return launch_rows(stream, a, false); }

cudaError_t kv_keep(cudaStream_t stream, const KeepArgs& a) {
  const int element = a.pool.store == kStoreE4m3 ? 1 : a.pool.store == kStoreBf16 ? 2 : 4;
  const size_t row = static_cast<size_t>(a.heads) * a.dim * element;
  const auto fits = [&](size_t n) {
    return row % n == 0 && a.pool.page_stride * element % n == 0 && a.pool.token_stride * element % n == 0 &&
           reinterpret_cast<uintptr_t>(a.pool.k) % n == 0 && reinterpret_cast<uintptr_t>(a.pool.v) % n == 0;
  };
  const size_t piece = fits(16) ? 16 : fits(4) ? 4 : 1;
  const size_t pieces = row / piece + (a.pool.store == kStoreE4m3 ? a.heads : 0);
  const dim3 grid(static_cast<unsigned>((pieces + 127) / 128), a.batch, 2);
  if (piece == 16) kv_keep_kernel<uint4><<<grid, 128, 0, stream>>>(a, row, element);
  else if (piece == 4) kv_keep_kernel<uint32_t><<<grid, 128, 0, stream>>>(a, row, element);
  else kv_keep_kernel<uint8_t><<<grid, 128, 0, stream>>>(a, row, element);
  return cudaGetLastError();
}

}  // namespace pluto
