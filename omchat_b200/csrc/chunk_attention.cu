// Attention of a chunk of new tokens over the paged cache, which holds the new tokens' keys and values already.
//
// Sequence s has the rows cu[s] .. cu[s + 1] - 1 of q, at the positions ctx[s] - n .. ctx[s] - 1 of its cache (n rows):
//   o[t, h] = sum_{j <= p(t)} softmax_j(scale q[t, h] . k[j, g]) v[j, g],  g = h / (Hq / Hkv)
#include <math.h>
#include <stdint.h>

#include "omc_internal.h"
#include "ptx.cuh"

namespace omc {

typedef __nv_bfloat16 bf16;

struct ChunkArgs {
  const bf16* q;
  long long ldq;
  const bf16* pool;        // [n_pages][2][Hkv][page_size][D]
  const int32_t* table;    // [n_seq][max_pages]
  const int32_t* cu;       // [n_seq + 1]
  const int32_t* ctx;      // [n_seq]
  bf16* out;
  long long ldo;
  int n_seq, T, max_new, max_ctx, n_pages, max_pages, page_size, Hq, Hkv;
  float scale_log2;
};

// One warp per (row, query head): lanes over the head's dimensions, keys one after the other.
template <int D>
__global__ void __launch_bounds__(128) chunk_attn_rows_kernel(const ChunkArgs a) {
  constexpr int E = D / 32;
  const int s = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 31, i = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int first = max(0, a.cu[s]), n = a.cu[s + 1] - a.cu[s];
  if (i >= n || i >= a.max_new || first + i >= a.T) return;
  const int end = min(min(a.ctx[s], a.max_ctx), a.max_pages * a.page_size) - n + i + 1;
  const bf16* q = a.q + (long long)(first + i) * a.ldq + h * D + lane * E;
  float qv[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) qv[e] = __bfloat162float(q[e]) * a.scale_log2, o[e] = 0.f;
  const int g = h / (a.Hq / a.Hkv);
  for (int j = 0; j < end; ++j) {
    const int page = a.table[(long long)s * a.max_pages + j / a.page_size];
    const bool there = page >= 0 && page < a.n_pages;
    const bf16* k = a.pool + (((long long)(there ? page : 0) * 2 * a.Hkv + g) * a.page_size + j % a.page_size) * D + lane * E;
    const bf16* v = k + (long long)a.Hkv * a.page_size * D;
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) dot += qv[e] * (there ? __bfloat162float(k[e]) : 0.f);
    dot = warp_sum(dot);
    const float top = fmaxf(m, dot), f = exp2f(m - top), p = exp2f(dot - top);
    l = l * f + p;
    m = top;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * f + p * (there ? __bfloat162float(v[e]) : 0.f);
  }
  bf16* out = a.out + (long long)(first + i) * a.ldo + h * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = __float2bfloat16(l > 0.f ? o[e] / l : (l == 0.f ? 0.f : l));
}

}  // namespace omc

using namespace omc;

extern "C" long long omc_paged_chunk_attn_workspace_bytes(int n_seq, int max_new, int max_ctx, int Hq, int Hkv, int head_dim) {
  (void)n_seq; (void)max_new; (void)max_ctx; (void)Hq; (void)Hkv; (void)head_dim;
  return 0;
}

extern "C" int omc_paged_chunk_attn(const void* q, long long ldq, const void* kv_pool, int n_pages, const int32_t* block_table, int max_pages, int page_size,
                                    const int32_t* cu_new, const int32_t* ctx_lens, int n_seq, int T, int max_new, int max_ctx, int Hq, int Hkv, int head_dim,
                                    float scale, void* out, long long ldo, void* workspace, long long workspace_bytes, void* stream) {
  if (head_dim != 64 && head_dim != 128) return set_error(OMC_ERR_SHAPE, "omc_paged_chunk_attn: heads of 64 or 128");
  if (Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0) return set_error(OMC_ERR_SHAPE, "omc_paged_chunk_attn: query heads must be a multiple of the key/value heads");
  if (n_pages <= 0 || max_pages <= 0 || page_size <= 0) return set_error(OMC_ERR_ARG, "omc_paged_chunk_attn: bad paging parameters");
  if ((long long)n_pages * 2 * Hkv * page_size >= (1ll << 31)) return set_error(OMC_ERR_SHAPE, "omc_paged_chunk_attn: a pool of 2^31 rows or more");
  if (n_seq < 0 || T < 0 || max_new < 0 || max_ctx < 0) return set_error(OMC_ERR_SHAPE, "omc_paged_chunk_attn: negative size");
  if (!(scale > 0.f) || isinf(scale)) return set_error(OMC_ERR_ARG, "omc_paged_chunk_attn: the scale has to be a positive number");
  if (ldq % 8 != 0 || ldo % 8 != 0 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kv_pool) | reinterpret_cast<uintptr_t>(out)) & 15) != 0)
    return set_error(OMC_ERR_ALIGN, "omc_paged_chunk_attn: q, pool and out on 16-byte boundaries, row strides multiples of 8");
  if (T > 1 && (ldq < (long long)Hq * head_dim || ldo < (long long)Hq * head_dim)) return set_error(OMC_ERR_SHAPE, "omc_paged_chunk_attn: rows overlap");
  if (n_seq == 0 || T == 0 || max_new == 0) return OMC_OK;
  if (q == nullptr || kv_pool == nullptr || out == nullptr || block_table == nullptr || cu_new == nullptr || ctx_lens == nullptr)
    return set_error(OMC_ERR_ARG, "omc_paged_chunk_attn: null pointer");
  (void)workspace; (void)workspace_bytes;
  ChunkArgs a{static_cast<const bf16*>(q), ldq, static_cast<const bf16*>(kv_pool), block_table, cu_new, ctx_lens, static_cast<bf16*>(out), ldo,
              n_seq, T, max_new, max_ctx, n_pages, max_pages, page_size, Hq, Hkv, scale * 1.4426950408889634f};
  const dim3 grid((max_new + 3) / 4, Hq, n_seq);
  if (head_dim == 64) chunk_attn_rows_kernel<64><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
  else chunk_attn_rows_kernel<128><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
  return check_launch("omc_paged_chunk_attn");
}
