// What the attention kernels are launched with, and how they find their rows and keys.
#ifndef MCHIP_ATTENTION_ARGS_H_
#define MCHIP_ATTENTION_ARGS_H_

#include "rows_of_heads.h"

namespace mchip {

// n / d for 0 <= n < 2^32 by a product: the round-up method for invariant divisors
// (Granlund and Montgomery, 1994).
struct FastDivision {
  unsigned d, factor;
  int shift;
  void set(unsigned divisor) {
    d = divisor;
    int log = 0;
    while ((1ull << log) < divisor) ++log;  // ceil(log2 d)
    factor = static_cast<unsigned>((((1ull << log) - divisor) << 32) / divisor + 1);
    shift = log;
  }
  __device__ __forceinline__ unsigned quotient(unsigned n) const {
    const unsigned t = __umulhi(factor, n);
    return shift == 0 ? n : (t + ((n - t) >> 1)) >> (shift - 1);
  }
};

struct AttentionArgs {
  int heads, heads_kv, head_dim, causal;
  FastDivision group;  // query heads of a key head
  float scale_log2;    // scale * log2(e): the softmax is formed with powers of two
  mcHeads q, k, v, out;  // k, v: packed only
  mcPagedCache cache;    // paged only
  FastDivision block;    // its block size
  const int* q_starts;
  const int* k_starts;      // packed only
  const int* block_table;   // paged only
  const int* context_lens;  // paged only
  int table_width, num, total_q, total_k, max_q, max_context;
  float* lse;
  // keys cut into pieces (paged only): piece p holds keys p * piece .. (p + 1) * piece
  int pieces, piece;
  float* partial;  // [pieces][total_q * heads][DP]: sums over a piece's keys, not divided
  float* stats;    // [pieces][total_q * heads][2]: largest score, sum of weights
  int tiles;       // row tiles of one key head
};

constexpr int kTileRows = 128;

// Sequence s starts at starts[s] * group / rows + s * gap on a scale of tiles (gap 1 leaves
// room for its ragged end), or of rows (group = rows = 1, gap 0).  The last s that starts
// at `at` or before.
__device__ __forceinline__ int sequence_of_tile(const int* __restrict__ starts, int num, int group,
                                                int rows, int at, int gap) {
  int lo = 0, hi = num;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (static_cast<long>(starts[mid]) * group / rows + mid * gap <= at) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The keys of a sequence, and what its rows see of them.
struct Keys {
  int first;   // packed: row of the first key
  int count;   // keys there are
  int offset;  // row i (of the sequence's queries) sees min(count, offset + i) keys
};

template <bool PAGED>
__device__ __forceinline__ Keys keys_of(const AttentionArgs& a, int seq, int queries) {
  Keys k;
  if (PAGED) {
    const int context = max(a.context_lens[seq], 0);
    k.first = 0;
    k.count = static_cast<int>(min(static_cast<long>(min(context, a.max_context)),
                                   static_cast<long>(a.table_width) * a.cache.block_size));
    k.offset = context - queries + 1;
  } else {
    k.first = max(a.k_starts[seq], 0);
    k.count = max(min(a.k_starts[seq + 1], a.total_k) - k.first, 0);
    k.offset = k.count - queries + 1;
  }
  if (!a.causal) k.offset = k.count;
  return k;
}

// Keys that some row of a row's tile sees (tiles start at multiples of kTileRows in a
// sequence's rows, token by token and head by head of the group; the last row sees most).
template <bool PAGED>
__device__ __forceinline__ int keys_of_tile(const AttentionArgs& a, const Keys& k, int row, int rows) {
  const int last = min(row / kTileRows * kTileRows + kTileRows - 1, rows - 1);
  return max(min(k.count, a.causal ? k.offset + static_cast<int>(a.group.quotient(last)) : k.count), 0);
}

// Element offset of a key's row in the cache, -1 if its block does not exist.
__device__ __forceinline__ long cache_row(const AttentionArgs& a, const int* __restrict__ table, int key) {
  const unsigned b = a.block.quotient(key);
  const int number = table[b];
  if (static_cast<unsigned>(number) >= static_cast<unsigned>(a.cache.num_blocks)) return -1;
  return number * a.cache.block_stride +
         static_cast<long>(static_cast<unsigned>(key) - b * a.block.d) * a.cache.token_stride;
}

// One source file per element type.
int attention_f32(const AttentionArgs& a, bool paged, hipStream_t st);
int attention_f16(const AttentionArgs& a, bool paged, hipStream_t st);
int attention_bf16(const AttentionArgs& a, bool paged, hipStream_t st);

}  // namespace mchip

#endif  // MCHIP_ATTENTION_ARGS_H_
