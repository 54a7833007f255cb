// Attention of many query rows: a workgroup of four wavefronts holds a tile of rows in
// registers and passes over the keys, a tile at a time through LDS.
//
// Rows: the query heads of one key head lie behind each other (row = token * group + head
// of the group), so a tile reads the keys of its one key head, whatever the group.  A
// wavefront has 32 rows.  Both products are formed transposed, so that a lane owns one
// row in all of them and the softmax needs no exchange but the one between the lane's two
// halves of the wavefront:
//
//   S^T [keys, rows] = K [keys, d] Q^T [d, rows]     32 x 32 blocks: lane l has row l % 32,
//                                                    keys 8 (i / 4) + 4 (l / 32) + i % 4, i < 16
//   O^T [d, rows]   += V^T [d, keys] P^T [keys, rows]
//
// P never leaves the registers: the keys that a lane holds after the first product are, in
// the order of its registers, taken as the ones it supplies to the second, and V's rows
// are fetched in that order.  16-bit V is transposed on its way out of LDS
// (ds_read_b64_tr_b16: of 16 lanes that address 4 rows of 16 values, each gets a column).
#ifndef MCHIP_ATTENTION_TILE_H_
#define MCHIP_ATTENTION_TILE_H_

#include "attention_args.h"

#include <type_traits>

namespace mchip {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));

// What differs by element type: the operand registers and the products.
template <typename T>
struct Product {  // fp16, bf16
  typedef T vec8 __attribute__((ext_vector_type(8)));
  typedef vec8 Operand;               // 8 values of d, or of keys: 16 per product
  static constexpr int kDepth = 16;
  static __device__ __forceinline__ floatx16 mma(vec8 a, vec8 b, floatx16 c) {
    if constexpr (__is_same(T, bf16_t)) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

template <typename T, int DP>
struct TileShape {
  static constexpr int kRowBytes = DP * static_cast<int>(sizeof(T));
  static constexpr int kKeys = kRowBytes <= 256 ? 64 : 32;     // keys of a tile
  static constexpr int kChunks = kRowBytes / 16;               // 16-byte chunks of a row
  // LDS rows: an odd number of chunks apart for K, so that 16 lanes that read one chunk of
  // 16 rows meet all banks; V's rows so that the 4 (16 bits) or 2 (32 bits, four rows
  // apart) row pieces of a read lie side by side modulo 256 bytes.
  static constexpr int kKStride = (kChunks | 1) * 16;
  static constexpr int kVStride = sizeof(T) == 2 ? ((kRowBytes / 32) | 1) * 32 : kRowBytes + 32;
  // Staging: a thread carries one chunk (of a power of two, the last ones idle) of kStage rows.
  static constexpr int kLanes = kChunks <= 8 ? 8 : kChunks <= 16 ? 16 : kChunks <= 32 ? 32 : 64;
  static constexpr int kPass = 256 / kLanes;                   // rows that the workgroup loads at once
  static constexpr int kStage = kKeys / kPass;
};

// Where the keys are.
enum class Source {
  kPacked,  // rows of one tensor
  kRuns,    // a paged cache whose block size is a multiple of kPass: the rows loaded at once
            // lie in one block, so addresses are scalars plus a fixed offset per thread
  kPaged    // any block size: a lane looks a key up
};

// Scores of 32 keys (rows `base` on of the K tile) against the wavefront's rows.
template <typename T, int DP>
__device__ __forceinline__ floatx16 scores(const char* lds_k, int base, const floatx4* q, int lane) {
  using S = TileShape<T, DP>;
  const char* at = lds_k + (base + (lane & 31)) * S::kKStride + (lane >> 5) * 16;
  floatx16 c = {};
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const floatx4 a = *reinterpret_cast<const floatx4*>(at + s * 32);
      c = Product<T>::mma(__builtin_bit_cast(typename Product<T>::vec8, a),
                          __builtin_bit_cast(typename Product<T>::vec8, q[s]), c);
    }
  } else {
#pragma unroll
    for (int s = 0; s < DP / 8; ++s) {  // 8 values of d: four products of two (half 0's and half 1's)
      const floatx4 a = *reinterpret_cast<const floatx4*>(at + s * 32);
#pragma unroll
      for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], q[s][e], c, 0, 0, 0);
    }
  }
  return c;
}

typedef __attribute__((address_space(3))) shortx4 lds_shortx4;

// Four keys (rows `key` on) of the 16 columns that a group of 16 lanes shares.
__device__ __forceinline__ shortx4 column_of_4(const char* at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)const_cast<char*>(at));
}

__device__ __forceinline__ bool finite16(short x, unsigned short exponent) {
  return (static_cast<unsigned short>(x) & exponent) != exponent;
}

// O^T += V^T P^T for 32 keys (rows `base` on of the V tile), p: the lane's 16 weights.
// SAFE: infinities and NaN of V count as 0 here.
template <typename T, int DP, bool SAFE>
__device__ __forceinline__ void weighted_sum(const char* lds_v, int base, const floatx16& p, floatx16* o,
                                             int lane) {
  using S = TileShape<T, DP>;
  if constexpr (sizeof(T) == 2) {
    constexpr unsigned short kExponent = __is_same(T, bf16_t) ? 0x7f80 : 0x7c00;
    typename Product<T>::vec8 w[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i >> 3][i & 7] = static_cast<T>(p[i]);
    const char* at = lds_v + (base + 4 * (lane >> 5) + ((lane & 15) >> 2)) * S::kVStride +
                     (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const shortx4 lo = column_of_4(at + 16 * s * S::kVStride + 64 * t);
        const shortx4 hi = column_of_4(at + (16 * s + 8) * S::kVStride + 64 * t);
        shortx8 a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        if constexpr (SAFE) {
#pragma unroll
          for (int e = 0; e < 8; ++e) a[e] = finite16(a[e], kExponent) ? a[e] : short(0);
        }
        o[t] = Product<T>::mma(__builtin_bit_cast(typename Product<T>::vec8, a), w[s], o[t]);
      }
  } else {
    const char* at = lds_v + (base + 4 * (lane >> 5)) * S::kVStride + (lane & 31) * 4;
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int t = 0; t < DP / 32; ++t) {
        float a = *reinterpret_cast<const float*>(at + (8 * (i >> 2) + (i & 3)) * S::kVStride + 128 * t);
        if constexpr (SAFE) a = __builtin_isfinite(a) ? a : 0.f;
        o[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[i], o[t], 0, 0, 0);
      }
  }
}

// What weighted_sum<SAFE> left out, for the rows that see it: a weight of a key that is
// seen is positive, so the sum gets the infinity or NaN itself.  seen: the lane's keys of
// the tile, valid: those that exist.
template <typename T, int DP>
__device__ __forceinline__ void add_not_finite(const char* lds_v, int seen, unsigned long valid,
                                               floatx16* o, int lane) {
  using S = TileShape<T, DP>;
  for (int key = 0; key < seen; ++key) {
    if (!(valid >> key & 1)) continue;
    const T* row = reinterpret_cast<const T*>(lds_v + key * S::kVStride);
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float v = static_cast<float>(row[32 * t + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3)]);
        if (!__builtin_isfinite(v)) o[t][i] += v;
        __builtin_amdgcn_sched_barrier(0);  // rare and slow: takes no registers from the rest
      }
  }
}

// The larger of the lane's value and that of lane ^ 32.  (The two results of the builtin
// for this instruction are taken as equal when its operands are, so it is written out; a
// vector result needs two wait states before a lane exchange reads it.)
__device__ __forceinline__ float larger_of_halves(float x) {
  float y = x;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));  // {low, low}, {high, high}
  return fmaxf(x, y);
}

// The running softmax of one row: powers of two of the scores times scale * log2(e).  The
// sum is the lane's own half of the keys until the end.
struct Running {
  float m = -INFINITY, l = 0.f;
};

// The weights of fp16 are kept this many powers of two larger than those of the largest
// score, so that small ones stay out of fp16's subnormal range.
template <typename T>
constexpr float kLift = __is_same(T, half_t) ? 10.f : 0.f;
// m moves only when a score is this much above it (in powers of two): the sums are then
// rescaled for a few tiles of a pass instead of most, and weights reach 2^8 (fp16: 2^15,
// just within its range).  The quotient at the end does not depend on m.
template <typename T>
constexpr float kSlack = __is_same(T, half_t) ? 5.f : 8.f;

// Takes a tile's scores into the running softmax: s becomes the weights, o is rescaled
// where some row's m moves.
template <typename T, int DP, int SUB>
__device__ __forceinline__ void softmax_step(floatx16* s, floatx16* o, Running& r, float scale_log2) {
  float top = s[0][0];
#pragma unroll
  for (int u = 0; u < SUB; ++u)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
  top = larger_of_halves(top) * scale_log2;
  if (__any(top > r.m + kSlack<T>)) {
    const float m = fmaxf(r.m, top);
    const float keep = m == -INFINITY ? 1.f : exp2f(r.m - m);
    r.m = m;
    r.l *= keep;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) o[t] *= keep;
  }
  const float shift = (r.m == -INFINITY ? 0.f : r.m) - kLift<T>;
#pragma unroll
  for (int u = 0; u < SUB; ++u)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[u][i] = __builtin_amdgcn_exp2f(fmaf(s[u][i], scale_log2, -shift));
      r.l += s[u][i];
    }
}

// The lane's row: out and lse, or its partial sums where the keys are cut into pieces.
template <typename T, int DP, bool PAGED>
__device__ __forceinline__ void store_rows(const AttentionArgs& a, const floatx16* o, Running r, int token,
                                           int head, int piece, bool whole, bool real, int lane) {
  r.l += __shfl_xor(r.l, 32, 64);
  if (!real) return;
  if (PAGED && !whole) {
    const long at = (static_cast<long>(piece) * a.total_q + token) * a.heads + head;
    float* to = a.partial + at * DP + 4 * (lane >> 5);
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<floatx4*>(to + 32 * t + 8 * i) =
            floatx4{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
    if (lane < 32) {
      a.stats[2 * at] = r.m;
      a.stats[2 * at + 1] = r.l;
    }
    return;
  }
  const float inverse = r.l == 0.f ? 0.f : 1.f / r.l;
  T* out = static_cast<T*>(a.out.data) + token * a.out.token_stride + head * a.out.head_stride + 4 * (lane >> 5);
#pragma unroll
  for (int t = 0; t < DP / 32; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (32 * t + 8 * i < a.head_dim) {  // (head_dim is a multiple of 8)
        typedef T vec4 __attribute__((ext_vector_type(4)));
        vec4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = static_cast<T>(o[t][4 * i + e] * inverse);
        *reinterpret_cast<vec4*>(out + 32 * t + 8 * i) = x;
      }
  if (a.lse && lane < 32)
    a.lse[static_cast<long>(head) * a.total_q + token] =
        r.l == 0.f ? -INFINITY : (r.m - kLift<T> + log2f(r.l)) * 0.69314718f;
}

template <typename T, int DP, Source SRC>
__global__ __launch_bounds__(256, DP * sizeof(T) <= 256 ? 2 : 1) void attention_tile_kernel(
    const AttentionArgs a) {
  using S = TileShape<T, DP>;
  constexpr bool PAGED = SRC != Source::kPacked;
  constexpr int KT = S::kKeys, SUB = KT / 32;
  __shared__ __attribute__((aligned(16))) char lds_k[2][KT * S::kKStride];
  __shared__ __attribute__((aligned(16))) char lds_v[2][KT * S::kVStride];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = a.group.d, D = a.head_dim;
  // key heads vary fastest: with workgroups dealt to the XCDs in turn, eight key heads (or
  // a divisor or multiple of eight) put each one's keys into one XCD's L2.  Tiles run from
  // the last, which sees most keys, to the first.
  const int hk = blockIdx.x % a.heads_kv;
  const int rest = blockIdx.x / a.heads_kv;
  const int piece = rest / a.tiles, tile = a.tiles - 1 - rest % a.tiles;
  const int seq = sequence_of_tile(a.q_starts, a.num, group, kTileRows, tile, 1);
  const int q0 = max(a.q_starts[seq], 0), q1 = min(a.q_starts[seq + 1], a.total_q);
  const int queries = PAGED ? min(q1 - q0, a.max_q) : q1 - q0;
  const int first = (tile - static_cast<int>(static_cast<long>(a.q_starts[seq]) * group / kTileRows + seq)) * kTileRows;
  const int rows = queries * group;
  if (first < 0 || first >= rows) return;  // (tiles are counted generously)
  const Keys keys = keys_of<PAGED>(a, seq, q1 - q0);

  // the lane's row; those past the last repeat it and are not stored
  const int row = min(first + 32 * wave + (lane & 31), rows - 1);
  const bool real = first + 32 * wave + (lane & 31) < rows;
  const int token = a.group.quotient(row), head = hk * group + (row - token * group);
  const int limit = max(min(keys.count, a.causal ? keys.offset + token : keys.count), 0);
  // rows see more from the first to the last of a wavefront
  const int low = __builtin_amdgcn_readfirstlane(limit);
  const int high = __builtin_amdgcn_readlane(limit, 31);
  const int all = keys_of_tile<PAGED>(a, keys, first, rows);  // over the workgroup's
  const int begin = PAGED ? min(piece * a.piece, all) : 0;
  const int end = PAGED ? static_cast<int>(min(static_cast<long>(begin) + a.piece, static_cast<long>(all))) : all;
  if (PAGED && piece > 0 && begin >= all) return;

  // queries: 16 bytes per 16 (fp32: 8) values of d, the lane's half of them
  floatx4 q[S::kChunks / 2];
  {
    const char* at = reinterpret_cast<const char*>(static_cast<const T*>(a.q.data) +
                                                   (q0 + token) * a.q.token_stride + head * a.q.head_stride);
#pragma unroll
    for (int s = 0; s < S::kChunks / 2; ++s) {
      const int chunk = 2 * s + (lane >> 5);
      q[s] = floatx4{};
      if (chunk * static_cast<int>(16 / sizeof(T)) < D) q[s] = *reinterpret_cast<const floatx4*>(at + chunk * 16);
    }
  }

  // Staging.  Chunks past head_dim are zeroed in LDS once and not written again.
  const int chunk = tid % S::kLanes, pass_row = tid / S::kLanes;
  const bool there = chunk * static_cast<int>(16 / sizeof(T)) < D;
  const long k_stride = (PAGED ? a.cache.token_stride : a.k.token_stride) * static_cast<long>(sizeof(T));
  const long v_stride = (PAGED ? a.cache.token_stride : a.v.token_stride) * static_cast<long>(sizeof(T));
  const char* kbase = reinterpret_cast<const char*>(
      static_cast<const T*>(PAGED ? a.cache.keys : a.k.data) +
      hk * (PAGED ? a.cache.head_stride : a.k.head_stride) + (PAGED ? 0 : keys.first * a.k.token_stride));
  const char* vbase = reinterpret_cast<const char*>(
      static_cast<const T*>(PAGED ? a.cache.values : a.v.data) +
      hk * (PAGED ? a.cache.head_stride : a.v.head_stride) + (PAGED ? 0 : keys.first * a.v.token_stride));
  const unsigned chunk_at = there ? chunk * 16 : 0;
  const unsigned k_off = pass_row * static_cast<unsigned>(k_stride) + chunk_at;
  const unsigned v_off = pass_row * static_cast<unsigned>(v_stride) + chunk_at;
  const int* table = PAGED ? a.block_table + static_cast<long>(seq) * a.table_width : nullptr;
  char* const put_k = lds_k[0] + pass_row * S::kKStride + chunk * 16;
  char* const put_v = lds_v[0] + pass_row * S::kVStride + chunk * 16;
  if (S::kLanes != S::kChunks || DP != D) {
    if (!there && chunk < S::kChunks)
#pragma unroll
      for (int i = 0; i < 2 * S::kStage; ++i) {
        const int b = i / S::kStage, r = i % S::kStage * S::kPass;
        *reinterpret_cast<floatx4*>(put_k + b * KT * S::kKStride + r * S::kKStride) = floatx4{};
        *reinterpret_cast<floatx4*>(put_v + b * KT * S::kVStride + r * S::kVStride) = floatx4{};
      }
  }
  floatx4 stage_k[S::kStage], stage_v[S::kStage];
  constexpr unsigned long kAllValid = KT == 64 ? ~0ul : (1ul << KT) - 1;
  unsigned long stage_valid = kAllValid;
  int number[S::kStage];  // kRuns: the next tile's blocks
  auto look_up = [&](int tile_begin) {
    if constexpr (SRC == Source::kRuns)
#pragma unroll
      for (int i = 0; i < S::kStage; ++i)
        number[i] = table[a.block.quotient(min(tile_begin + i * S::kPass, end - 1))];
  };
  auto fetch = [&](int tile_begin) {  // keys past the end repeat the last one
    if constexpr (SRC == Source::kPacked) {
      const char* kt = kbase + tile_begin * k_stride;
      const char* vt = vbase + tile_begin * v_stride;
      if (tile_begin + KT <= end) {
#pragma unroll
        for (int i = 0; i < S::kStage; ++i) {
          stage_k[i] = *reinterpret_cast<const floatx4*>(kt + i * S::kPass * k_stride + k_off);
          stage_v[i] = *reinterpret_cast<const floatx4*>(vt + i * S::kPass * v_stride + v_off);
        }
      } else {
        const int last = end - 1 - tile_begin;
#pragma unroll
        for (int i = 0; i < S::kStage; ++i) {
          const unsigned r = min(pass_row + i * S::kPass, last);
          stage_k[i] = *reinterpret_cast<const floatx4*>(kt + (r * static_cast<unsigned>(k_stride) + chunk_at));
          stage_v[i] = *reinterpret_cast<const floatx4*>(vt + (r * static_cast<unsigned>(v_stride) + chunk_at));
        }
      }
    } else if constexpr (SRC == Source::kRuns) {
      stage_valid = kAllValid;
#pragma unroll
      for (int i = 0; i < S::kStage; ++i) {
        // (rows past the end lie in the last key's block)
        const unsigned key = min(tile_begin + i * S::kPass, (end - 1) / S::kPass * S::kPass);
        int n = number[i];
        if (static_cast<unsigned>(n) >= static_cast<unsigned>(a.cache.num_blocks)) {
          n = 0;
          stage_valid &= ~(((1ul << S::kPass) - 1) << (i * S::kPass));
        }
        const long at = (n * a.cache.block_stride) * static_cast<long>(sizeof(T)) +
                        (key - a.block.quotient(key) * a.block.d) * k_stride;
        unsigned off = k_off;
        if (tile_begin + KT > end)
          off = min(pass_row, end - 1 - static_cast<int>(key)) * static_cast<unsigned>(k_stride) + chunk_at;
        stage_k[i] = *reinterpret_cast<const floatx4*>(kbase + at + off);
        stage_v[i] = *reinterpret_cast<const floatx4*>(vbase + at + off);
      }
      if (tile_begin + KT < end) look_up(tile_begin + KT);
    } else {
      const int key = tile_begin + (lane % KT);
      long at = cache_row(a, table, min(key, end - 1));
      stage_valid = __ballot(at >= 0 && key < end) & kAllValid;
      at = max(at, 0l) * static_cast<long>(sizeof(T)) ;
#pragma unroll
      for (int i = 0; i < S::kStage; ++i) {
        const long from = __shfl(at, pass_row + i * S::kPass, 64) + chunk_at;
        stage_k[i] = *reinterpret_cast<const floatx4*>(kbase + from);
        stage_v[i] = *reinterpret_cast<const floatx4*>(vbase + from);
      }
    }
  };
  auto put = [&](int buffer) {
    if (there)
#pragma unroll
      for (int i = 0; i < S::kStage; ++i) {
        *reinterpret_cast<floatx4*>(put_k + buffer * (KT * S::kKStride) + i * S::kPass * S::kKStride) = stage_k[i];
        *reinterpret_cast<floatx4*>(put_v + buffer * (KT * S::kVStride) + i * S::kPass * S::kVStride) = stage_v[i];
      }
  };

  floatx16 o[DP / 32];
  Running run;
  // SAFE: what V's infinities and NaN do to a row is decided by what the row sees.
  auto pass = [&](auto safe) {
    constexpr bool SAFE = decltype(safe)::value;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) o[t] = floatx16{};
    run = Running();
    if (begin >= end) return;
    look_up(begin);
    fetch(begin);
    put(0);
    unsigned long valid = stage_valid;
    if (begin + KT < end) fetch(begin + KT);
    __syncthreads();
    int buffer = 0;
    for (int at = begin; at < end; at += KT) {
      const bool work = at < high;
      const char* const now_k = lds_k[0] + buffer * (KT * S::kKStride);
      const char* const now_v = lds_v[0] + buffer * (KT * S::kVStride);
      floatx16 s[SUB];
      if (work) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) s[u] = scores<T, DP>(now_k, 32 * u, q, lane);
      }
      const unsigned long next_valid = stage_valid;
      if (at + KT < end) {
        put(buffer ^ 1);
        if (at + 2 * KT < end) fetch(at + 2 * KT);
      }
      if (work) {
        const bool masked = at + KT > low || (PAGED && valid != kAllValid);
        if (masked) {
          const int seen = min(limit, end) - at;
#pragma unroll
          for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int key = 32 * u + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
              if (key >= seen || (PAGED && !(valid >> key & 1))) s[u][i] = -INFINITY;
            }
        }
        softmax_step<T, DP, SUB>(s, o, run, a.scale_log2);
#pragma unroll
        for (int u = 0; u < SUB; ++u) weighted_sum<T, DP, SAFE>(now_v, 32 * u, s[u], o, lane);
        if (SAFE) add_not_finite<T, DP>(now_v, min(min(limit, end) - at, KT), valid, o, lane);
      }
      valid = next_valid;
      buffer ^= 1;
      __syncthreads();
    }
  };
  pass(std::false_type());
  // A weight of zero does not keep an infinity or NaN in V's row out of the products.  If
  // some row's sums are not finite, everything is done once more, the safe way.
  float check = 0.f;
#pragma unroll
  for (int t = 0; t < DP / 32; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) check += 0.f * o[t][i];
  if (__syncthreads_or(check != 0.f)) pass(std::true_type());  // (0 * inf and 0 * NaN are NaN, which is not 0)
  store_rows<T, DP, PAGED>(a, o, run, q0 + token, head, piece, all <= a.piece, real, lane);
}

}  // namespace mchip

#endif  // MCHIP_ATTENTION_TILE_H_
