// Attention of packed sequences and over a paged cache:
//   out = softmax(scale * q k^T) v,  lse = ln sum exp(scale * q k),
// in one pass over the keys with the running maximum m and sum l of the softmax:
//   m' = max(m, s), l' = l e^(m - m') + sum e^(s - m'), o' = o e^(m - m') + sum e^(s - m') v.
//
// One wavefront per query row and head.  64 keys at a time: a lane forms the score of one
// key (the query lies in LDS), then the lanes share out the head's values and add the 64
// rows of v, each weighted by a score fetched from its lane.
#include "rows_of_heads.h"

#include <cmath>

namespace mchip {
namespace {

struct AttentionArgs {
  int heads, group, head_dim, causal;
  float scale;
  mcHeads q, k, v, out;  // k, v: packed only
  mcPagedCache cache;    // paged only
  const int* q_starts;
  const int* k_starts;      // packed only
  const int* block_table;   // paged only
  const int* context_lens;  // paged only
  int table_width, num, total_q, total_k, max_q, max_context;
  float* lse;
};

// The sequence of a packed row: last s with starts[s] <= row.
__device__ __forceinline__ int sequence_of(const int* __restrict__ starts, int num, int row) {
  int lo = 0, hi = num;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <typename T, bool PAGED>
__global__ __launch_bounds__(64) void attention_rows_kernel(AttentionArgs a) {
  __shared__ float ql[kMaxHeadDim];
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  const int seq = sequence_of(a.q_starts, a.num, row);
  const int q0 = a.q_starts[seq], q1 = min(a.q_starts[seq + 1], a.total_q);
  if (row < q0 || row >= q1 || q0 < 0) return;
  const int hk = h / a.group, D = a.head_dim;
  int k0 = 0, keys;
  if (PAGED) {
    if (row - q0 >= a.max_q) return;
    keys = min(a.context_lens[seq], a.max_context);
  } else {
    k0 = max(a.k_starts[seq], 0);
    keys = min(a.k_starts[seq + 1], a.total_k) - k0;
  }
  if (a.causal) keys = min(keys, (PAGED ? a.context_lens[seq] : keys) - (q1 - q0) + (row - q0) + 1);
  const T* q = static_cast<const T*>(a.q.data) + row * a.q.token_stride + h * a.q.head_stride;
  for (int d = lane; d < D; d += 64) ql[d] = static_cast<float>(q[d]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[kMaxHeadDim / 64] = {};
  for (int base = 0; base < keys; base += 64) {
    const int key = base + lane;
    float s = -INFINITY;
    long at = -1;
    if (key < keys) {
      if (PAGED) {
        const int b = key / a.cache.block_size;
        const int number = b < a.table_width ? a.block_table[(long)seq * a.table_width + b] : -1;
        if (number >= 0 && number < a.cache.num_blocks)
          at = number * a.cache.block_stride + (key % a.cache.block_size) * a.cache.token_stride +
               hk * a.cache.head_stride;
      } else {
        at = (long)(k0 + key) * a.k.token_stride + hk * a.k.head_stride;
      }
    }
    if (at >= 0) {
      const T* k = static_cast<const T*>(PAGED ? a.cache.keys : a.k.data) + at;
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot += ql[d] * static_cast<float>(k[d]);
      s = dot * a.scale;
    }
    float top = s;
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor(top, w, 64));
    const float next = fmaxf(m, top), base_m = next == -INFINITY ? 0.f : next;
    const float keep = expf(m - base_m), p = at >= 0 ? expf(s - base_m) : 0.f;
    float sum = p;
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) sum += __shfl_xor(sum, w, 64);
    l = l * keep + sum;
    m = next;
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 64; ++i) o[i] *= keep;
    for (int j = 0; j < 64; ++j) {
      const long row_at = __shfl(at, j, 64);
      if (row_at < 0) continue;
      const float w = __shfl(p, j, 64);
      const T* v = PAGED ? static_cast<const T*>(a.cache.values) + row_at
                         : static_cast<const T*>(a.v.data) + (long)(k0 + base + j) * a.v.token_stride +
                               hk * a.v.head_stride;
#pragma unroll
      for (int i = 0; i < kMaxHeadDim / 64; ++i)
        if (lane + 64 * i < D) o[i] += w * static_cast<float>(v[lane + 64 * i]);
    }
  }
  T* out = static_cast<T*>(a.out.data) + row * a.out.token_stride + h * a.out.head_stride;
#pragma unroll
  for (int i = 0; i < kMaxHeadDim / 64; ++i)
    if (lane + 64 * i < D) out[lane + 64 * i] = static_cast<T>(l == 0.f ? 0.f : o[i] / l);
  if (a.lse && lane == 0) a.lse[(long)h * a.total_q + row] = m + logf(l);  // no key: -inf
}

template <bool PAGED>
int launch(const AttentionArgs& a, int type, hipStream_t st) {
  const dim3 grid(a.total_q, a.heads);
  if (type == MC_TYPE_F32) attention_rows_kernel<float, PAGED><<<grid, 64, 0, st>>>(a);
  else if (type == MC_TYPE_F16) attention_rows_kernel<half_t, PAGED><<<grid, 64, 0, st>>>(a);
  else attention_rows_kernel<bf16_t, PAGED><<<grid, 64, 0, st>>>(a);
  MC_LAUNCH_CHECK();
  return 0;
}

int check_geom(const char* who, const mcAttentionGeom* g, AttentionArgs* a) {
  MC_REQUIRE(g, "%s: null geometry", who);
  if (check_type(who, g->type, g->head_dim)) return -1;
  MC_REQUIRE(g->heads > 0 && g->heads_kv > 0 && g->heads % g->heads_kv == 0,
             "%s: %d query heads do not share %d key heads evenly", who, g->heads, g->heads_kv);
  MC_REQUIRE(g->heads <= 65535, "%s: more than 65535 heads", who);
  MC_REQUIRE(g->scale > 0.f && std::isfinite(g->scale), "%s: scale %g is not positive and finite", who, g->scale);
  a->heads = g->heads;
  a->group = g->heads / g->heads_kv;
  a->head_dim = g->head_dim;
  a->causal = g->causal != 0;
  a->scale = g->scale;
  return 0;
}

}  // namespace
}  // namespace mchip

using namespace mchip;

extern "C" int mcAttentionPacked(const mcAttentionGeom* geom, const mcHeads* q, const mcHeads* k,
                                 const mcHeads* v, const int* q_starts, const int* k_starts,
                                 int num_sequences, int total_q, int total_k, const mcHeads* out,
                                 float* lse, void* stream) {
  static const char who[] = "mcAttentionPacked";
  AttentionArgs a = {};
  if (check_geom(who, geom, &a)) return -1;
  MC_REQUIRE(num_sequences >= 0 && total_q >= 0 && total_k >= 0, "%s: bad extents", who);
  if (num_sequences == 0 || total_q == 0) return 0;
  MC_REQUIRE(q_starts && k_starts, "%s: null argument", who);
  if (check_heads(who, "q", q, geom->type) || check_heads(who, "out", out, geom->type)) return -1;
  if (total_k > 0) {
    if (check_heads(who, "k", k, geom->type) || check_heads(who, "v", v, geom->type)) return -1;
    a.k = *k;
    a.v = *v;
  }
  a.q = *q;
  a.out = *out;
  a.q_starts = q_starts;
  a.k_starts = k_starts;
  a.num = num_sequences;
  a.total_q = total_q;
  a.total_k = total_k;
  a.lse = lse;
  return launch<false>(a, geom->type, static_cast<hipStream_t>(stream));
}

extern "C" int mcAttentionPaged(const mcAttentionGeom* geom, const mcHeads* q, const mcPagedCache* cache,
                                const int* block_table, int table_width, const int* q_starts,
                                const int* context_lens, int num_requests, int total_q, int max_q,
                                int max_context, const mcHeads* out, float* lse, void* stream) {
  static const char who[] = "mcAttentionPaged";
  AttentionArgs a = {};
  if (check_geom(who, geom, &a)) return -1;
  MC_REQUIRE(num_requests >= 0 && total_q >= 0 && max_q >= 0 && max_context >= 0 && table_width > 0,
             "%s: bad extents", who);
  if (num_requests == 0 || total_q == 0 || max_q == 0) return 0;
  MC_REQUIRE(block_table && q_starts && context_lens, "%s: null argument", who);
  if (check_heads(who, "q", q, geom->type) || check_heads(who, "out", out, geom->type) ||
      check_cache(who, cache, geom->type))
    return -1;
  a.q = *q;
  a.out = *out;
  a.cache = *cache;
  a.block_table = block_table;
  a.table_width = table_width;
  a.q_starts = q_starts;
  a.context_lens = context_lens;
  a.num = num_requests;
  a.total_q = total_q;
  a.max_q = max_q;
  a.max_context = max_context;
  a.lse = lse;
  return launch<true>(a, geom->type, static_cast<hipStream_t>(stream));
}
