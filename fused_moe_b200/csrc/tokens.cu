// Tokens sorted by expert and back, with weights applied, and the gradients; weights of the selected experts and theirs.
//
// A pair p = t * K + k is token t's k-th selected expert.  Its row is offset[e] + (pairs of expert e before p in flat order): a
// stable counting sort, whose segments start at multiples of `align`.  Pairs of other shards' experts, negative ids, and pairs
// whose row would lie at or behind the capacity `rows` have none (-1).  Unlike the layer's own sort (sort.cu), a token may name
// an expert twice.
//   gather    out[row(t,k)] = x[t]                    backward: grad_x[t] = sum_k grad[row(t,k)]    (= combine, weights 1)
//   combine   out[t] = sum_k w[t,k] * in[row(t,k)]    backward: grad_in[row(t,k)] = w[t,k] * grad[t]
//                                                               grad_w[t,k] = sum over columns of grad[t] * in[row(t,k)]
// Rows without a pair, and rows whose pair the map sends elsewhere, are written as zeros.  The kernels walk tokens, not rows: a
// token's row is read once and written to (or summed from) its at most eight rows.  No atomics on values, every sum in a fixed
// order; sums are float32.
#include "route_token.cuh"
#include "row_vec.cuh"

namespace b200moe {

constexpr int SORT_THREADS = 1024;   // pairs ranked at once by a CTA
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_MAX_CTAS = B200MOE_TOKEN_SORT_MAX_CTAS;
// Up to here every CTA counts the whole batch itself and k_token_count is not launched.  us with it / without, 256 experts,
// align 128: 1 token 4.8 / 3.8, 128 tokens (one CTA) 8.9 / 7.8, 1024 (8) 6.9 / 6.1, 2048 (16) 7.1 / 7.0, 8192 (64) 9.9 / 16.7.
constexpr unsigned SORT_ONE_LAUNCH_CTAS = 16;

// Index of the pair's local expert, or -1.  Unsigned: a negative id is a large one.
__device__ __forceinline__ int local_expert(const int* topk_idx, long long p, long long n_pairs, int offset, int E_local) {
  if (p >= n_pairs) return -1;
  const uint32_t e = static_cast<uint32_t>(ld_dep(topk_idx + p)) - static_cast<uint32_t>(offset);
  return e < static_cast<uint32_t>(E_local) ? static_cast<int>(e) : -1;
}

// hist[b][e] = pairs of local expert e among the `per` pairs of CTA b.
__global__ void __launch_bounds__(SORT_THREADS)
k_token_count(const int* topk_idx, long long n_pairs, long long per, int offset, int E_local, int* hist) {
  __shared__ int s_count[E_GLOBAL];
  pdl_launch_dependents();
  if (threadIdx.x < E_GLOBAL) s_count[threadIdx.x] = 0;
  pdl_wait();
  __syncthreads();
  const long long first = blockIdx.x * per;
  for (long long i = threadIdx.x; i < per; i += SORT_THREADS) {
    const int e = local_expert(topk_idx, first + i, n_pairs, offset, E_local);
    if (e >= 0) atomicAdd(&s_count[e], 1);
  }
  __syncthreads();
  if (threadIdx.x < E_local) hist[blockIdx.x * E_local + threadIdx.x] = s_count[threadIdx.x];
}

// The rows: every CTA derives the layout from the counts of all CTAs (`hist`, or for a small batch, hist == nullptr, by
// counting the whole batch itself, which saves the launch of k_token_count), then ranks its pairs SORT_THREADS at a time.
// Inside a warp the rank is the number of lower lanes with the same expert, and the warps' counts are prefixed per expert.
// Bound by latency: barriers, and the counts of up to 256 CTAs one after the other (8.6 us with the count kernel at 4096
// tokens x 8, 12.5 at 16384; batches of 8 to 32 such loads 9.8 to 8.6 and 17.6 to 13.9, a quarter of the CTAs per quarter of
// the threads 10.0 and 14.6).
__global__ void __launch_bounds__(SORT_THREADS)
k_token_place(const int* topk_idx, long long n_pairs, long long per, int offset, int E_local, int align, int rows,
              const int* hist, int* counts, int* offsets, int* row_pairs, int* scatter_map) {
  __shared__ int s_next[E_GLOBAL];                  // row of the next pair of this expert in this CTA
  __shared__ int s_begin[E_GLOBAL + 1];             // first row of each segment (may exceed `rows`)
  __shared__ int s_total[E_GLOBAL];
  __shared__ int s_scan[E_GLOBAL / 32];
  __shared__ uint16_t s_warp[SORT_WARPS][E_GLOBAL];   // pairs of the warp, then of the warps before it
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  int total = 0, before = 0;
  if (!hist) {
    int* s_before = &s_next[0];
    if (threadIdx.x < E_GLOBAL) s_total[threadIdx.x] = s_before[threadIdx.x] = 0;
    __syncthreads();
    const long long mine = blockIdx.x * per;
    for (long long p = threadIdx.x; p < n_pairs; p += SORT_THREADS) {
      const int e = local_expert(topk_idx, p, n_pairs, offset, E_local);
      if (e < 0) continue;
      atomicAdd(&s_total[e], 1);
      if (p < mine) atomicAdd(&s_before[e], 1);
    }
    __syncthreads();
    if (threadIdx.x < E_local) {
      total = s_total[threadIdx.x];
      before = s_before[threadIdx.x];
    }
  } else if (threadIdx.x < E_local) {
    for (int b = 0; b < static_cast<int>(gridDim.x); ++b) {
      if (b == static_cast<int>(blockIdx.x)) before = total;
      total += ld_dep(hist + b * E_local + threadIdx.x);
    }
    s_total[threadIdx.x] = total;
  }
  const long long padded = threadIdx.x < E_local ? (static_cast<long long>(total) + align - 1) / align * align : 0;
  int incl = static_cast<int>(padded);   // a sum of padded segments fits: checked by the host
  if (threadIdx.x < E_GLOBAL) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += o;
    }
    if (lane == 31) s_scan[warp] = incl;
  }
  __syncthreads();
  if (threadIdx.x < E_GLOBAL) {
    for (int w = 0; w < warp; ++w) incl += s_scan[w];
    s_begin[threadIdx.x + 1] = incl;
    s_next[threadIdx.x] = incl - static_cast<int>(padded) + before;
    if (threadIdx.x == 0) s_begin[0] = 0;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    if (threadIdx.x < E_local) counts[threadIdx.x] = s_total[threadIdx.x];
    if (threadIdx.x <= E_local) offsets[threadIdx.x] = min(s_begin[threadIdx.x], rows);
  }
  // rows without a pair: the ends of the segments and what lies behind the last
  for (int e = blockIdx.x * SORT_WARPS + warp; e < E_local; e += gridDim.x * SORT_WARPS)
    for (int r = s_begin[e] + s_total[e] + lane; r < min(s_begin[e + 1], rows); r += 32) row_pairs[r] = -1;
  for (long long r = s_begin[E_local] + static_cast<long long>(blockIdx.x) * SORT_THREADS + threadIdx.x; r < rows;
       r += static_cast<long long>(gridDim.x) * SORT_THREADS)
    row_pairs[r] = -1;

  const long long first = blockIdx.x * per;
  if (first >= n_pairs) return;   // this CTA is there for the rows without a pair
  for (long long i = 0; i < per; i += SORT_THREADS) {
    for (int j = threadIdx.x; j < SORT_WARPS * E_GLOBAL; j += SORT_THREADS) (&s_warp[0][0])[j] = 0;
    __syncthreads();
    const long long p = first + i + threadIdx.x;
    const int e = i + threadIdx.x < per ? local_expert(topk_idx, p, n_pairs, offset, E_local) : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1u));
    if (e >= 0 && rank == 0) s_warp[warp][e] = static_cast<uint16_t>(__popc(same));
    __syncthreads();
    if (threadIdx.x < E_local) {
      int run = 0;
      for (int w = 0; w < SORT_WARPS; ++w) {
        const int c = s_warp[w][threadIdx.x];
        s_warp[w][threadIdx.x] = static_cast<uint16_t>(run);
        run += c;
      }
      s_total[threadIdx.x] = run;   // of this round
    }
    __syncthreads();
    if (p < n_pairs && i + threadIdx.x < per) {
      int row = -1;
      if (e >= 0) {
        row = s_next[e] + s_warp[warp][e] + rank;
        if (row >= rows) row = -1;
      }
      scatter_map[p] = row;
      if (row >= 0) row_pairs[row] = static_cast<int>(p);
    }
    __syncthreads();
    if (threadIdx.x < E_local) s_next[threadIdx.x] += s_total[threadIdx.x];
  }
}

// A token's pairs, one per lane of every warp: lane k < K holds the row (-1: none; an entry outside 0 .. rows - 1 is none, so
// that a map of another batch cannot lead a store out of the buffer) and the weight of pair (t, k).  `mask`: the lanes with a
// row.
struct TokenPairs {
  int row;
  float weight;
  uint32_t mask;
};
__device__ __forceinline__ TokenPairs token_pairs(const int* scatter_map, const float* weights, long long t, int K, int rows) {
  const int lane = threadIdx.x & 31;
  TokenPairs p;
  p.row = lane < K ? ld_dep(scatter_map + t * K + lane) : -1;
  p.weight = lane < K && weights ? ld_dep(weights + t * K + lane) : 1.f;
  if (static_cast<uint32_t>(p.row) >= static_cast<uint32_t>(rows)) p.row = -1;
  p.mask = __ballot_sync(0xffffffffu, p.row >= 0);
  return p;
}

// CTA i's share of the rows are the `per` rows from i * per on (at most 32: rows_per_cta()), one per lane of every warp; -1:
// none.
__device__ __forceinline__ int share_row(int per, int rows) {
  const int lane = threadIdx.x & 31, row = blockIdx.x * per + lane;
  return lane < per && row < rows ? row : -1;
}
__device__ __forceinline__ int share_pair(const int* row_pairs, int per, int rows) {
  const int row = share_row(per, rows);
  return row >= 0 ? ld_dep(row_pairs + row) : -1;
}
// The row that the map names for a pair, -1 for what is none of the batch's pairs.  Where that is not the row that names the
// pair, no token writes the row.
__device__ __forceinline__ int named_row(const int* scatter_map, int pair, int n_pairs) {
  return static_cast<uint32_t>(pair) < static_cast<uint32_t>(n_pairs) ? ld_dep(scatter_map + pair) : -1;
}
// The rows of the share that no token writes become zeros in the pieces [begin, end).
__device__ __forceinline__ void zero_unused_rows(int named, int per, int rows, uint8_t* out, int pieces, int begin, int end) {
  const int mine = share_row(per, rows);
  for (uint32_t unused = __ballot_sync(0xffffffffu, mine >= 0 && named != mine); unused; unused &= unused - 1) {
    const int row = blockIdx.x * per + __ffs(unused) - 1;
    uint4* dst = reinterpret_cast<uint4*>(out) + static_cast<long long>(row) * pieces;
    for (int p = begin + threadIdx.x; p < end; p += blockDim.x) dst[p] = make_uint4(0u, 0u, 0u, 0u);
  }
}

// out[row(t,k)] = x[t]; CTA (t, y) copies the y-th part of the token's row, and zeroes its share of the unused rows.  Bound
// by its stores, which do not stay in L2 (streaming: 171 -> 169 us): 8192 tokens x 8 rows of 7168 bf16 are 1.06 GB in 170 us,
// 6.2 TB/s.
constexpr int TOKEN_UNROLL = 4;   // pieces of a row in flight per thread
__global__ void __launch_bounds__(256)
k_token_gather(const uint8_t* x, long long x_pitch, int T, int K, int rows, int per, int pieces, const int* row_pairs,
               const int* scatter_map, uint8_t* out) {
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x;
  const int part = (pieces + gridDim.y - 1) / gridDim.y, begin = blockIdx.y * part, end = min(begin + part, pieces);
  // the share's two loads depend on one another: one ahead of those of the token's pairs and one behind, so that nothing
  // waits for either (1 token 2.2 us, 64 tokens 4.2; both behind the token's work 2.3 and 4.5)
  const int pair = share_pair(row_pairs, per, rows);
  TokenPairs pairs = {-1, 1.f, 0u};
  if (t < T) pairs = token_pairs(scatter_map, nullptr, t, K, rows);
  const int named = named_row(scatter_map, pair, T * K);
  if (t < T) {
    const uint4* src = reinterpret_cast<const uint4*>(x + t * x_pitch);
    for (int p0 = begin + threadIdx.x; pairs.mask && p0 - static_cast<int>(threadIdx.x) < end; p0 += TOKEN_UNROLL * blockDim.x) {
      uint4 v[TOKEN_UNROLL];
#pragma unroll
      for (int i = 0; i < TOKEN_UNROLL; ++i)
        if (p0 + i * blockDim.x < end) v[i] = ld_dep(src + p0 + i * blockDim.x);
      for (uint32_t m = pairs.mask; m; m &= m - 1) {
        const int row = __shfl_sync(0xffffffffu, pairs.row, __ffs(m) - 1);
        uint4* dst = reinterpret_cast<uint4*>(out) + static_cast<long long>(row) * pieces;
#pragma unroll
        for (int i = 0; i < TOKEN_UNROLL; ++i)
          if (p0 + i * blockDim.x < end) __stcs(dst + p0 + i * blockDim.x, v[i]);
      }
    }
  }
  zero_unused_rows(named, per, rows, out, pieces, begin, end);
}

// The rows of up to N pairs of a token, in the order of k: the lowest N bits of the mask.
template <int N>
__device__ __forceinline__ void take_pairs(const TokenPairs& pairs, int (&row)[N], float (&w)[N]) {
  uint32_t m = pairs.mask;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int k = m ? __ffs(m) - 1 : 0;
    const int r = __shfl_sync(0xffffffffu, pairs.row, k);
    w[j] = __shfl_sync(0xffffffffu, pairs.weight, k);
    row[j] = m ? r : -1;
    m &= m - 1;
  }
}

// Bound by its loads: 8192 tokens x 8 rows of 7168 bf16 are 1.06 GB in 151 us, 7.0 TB/s.
//
// out[t] = sum_k w[t,k] * in[row(t,k)], k ascending (weights == nullptr: 1), over the pieces [begin, end) of the rows.  N: most
// rows of the token; U: pieces of each in flight per thread (a token with one or two rows would have too few bytes under way
// otherwise: a shard of 32 experts at 14107 tokens 94 us with one piece, 69 with two).  Five CTAs of 256 threads per SM.
template <typename X, int N, int U>
__device__ __forceinline__ void combine_rows(const uint8_t* in, long long in_pitch, const TokenPairs& pairs, int begin,
                                             int end, uint4* out) {
  constexpr int P = PIECE_PAIRS<X>;
  int row[N];
  float w[N];
  take_pairs(pairs, row, w);
  for (int p0 = begin + threadIdx.x; p0 < end; p0 += U * blockDim.x) {
    uint4 raw[U][N];
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (row[k] >= 0 && p0 + i * blockDim.x < end)
          raw[i][k] = ld_dep(reinterpret_cast<const uint4*>(in + row[k] * in_pitch) + p0 + i * blockDim.x);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (p0 + i * blockDim.x >= end) break;
      float2 acc[P];
#pragma unroll
      for (int j = 0; j < P; ++j) acc[j] = both(0.f);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if (row[k] < 0) continue;
        float2 f[P];
        unpack_piece<X>(raw[i][k], f);
#pragma unroll
        for (int j = 0; j < P; ++j) acc[j] = fma2(both(w[k]), f[j], acc[j]);
      }
      out[p0 + i * blockDim.x] = pack_piece<X>(acc);
    }
  }
}
template <typename X>
__global__ void __launch_bounds__(256, 5)
k_token_combine(const uint8_t* in, long long in_pitch, const float* weights, int K, int rows, int pieces,
                const int* scatter_map, uint8_t* out) {
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x;
  const int part = (pieces + gridDim.y - 1) / gridDim.y, begin = blockIdx.y * part, end = min(begin + part, pieces);
  const TokenPairs pairs = token_pairs(scatter_map, weights, t, K, rows);
  uint4* dst = reinterpret_cast<uint4*>(out) + static_cast<long long>(t) * pieces;
  if (__popc(pairs.mask) <= 2)
    combine_rows<X, 2, 2>(in, in_pitch, pairs, begin, end, dst);
  else
    combine_rows<X, TOP_K, 1>(in, in_pitch, pairs, begin, end, dst);
}

// One pass over the rows gives both gradients: 8192 tokens x 8 rows of 7168 bf16 are 2.0 GB in 305 us, 6.5 TB/s.
//
// grad_in[row(t,k)] = w[t,k] * grad[t] and the token's dot products <grad[t], in[row(t,k)]>, summed over the CTA into
// s_dot[j][warp] for the j-th pair with a row; N and U as for combine_rows.
template <typename X, int N, int U>
__device__ __forceinline__ void combine_rows_backward(const uint4* grad, const uint8_t* in, long long in_pitch,
                                                      const TokenPairs& pairs, int pieces, uint8_t* grad_in,
                                                      float (*s_dot)[16]) {
  constexpr int P = PIECE_PAIRS<X>;
  int row[N];
  float w[N];
  float2 dot2[N];
  take_pairs(pairs, row, w);
#pragma unroll
  for (int k = 0; k < N; ++k) dot2[k] = both(0.f);
  for (int p0 = threadIdx.x; p0 < pieces; p0 += U * blockDim.x) {
    uint4 raw_g[U], raw[U][N];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int p = p0 + i * blockDim.x;
      if (p >= pieces) break;
      raw_g[i] = ld_dep(grad + p);
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (s_dot && row[k] >= 0) raw[i][k] = ld_dep(reinterpret_cast<const uint4*>(in + row[k] * in_pitch) + p);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int p = p0 + i * blockDim.x;
      if (p >= pieces) break;
      float2 g[P];
      unpack_piece<X>(raw_g[i], g);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if (row[k] < 0) continue;
        if (s_dot) {
          float2 f[P];
          unpack_piece<X>(raw[i][k], f);
#pragma unroll
          for (int j = 0; j < P; ++j) dot2[k] = fma2(g[j], f[j], dot2[k]);
        }
        if (grad_in) {
          float2 d[P];
#pragma unroll
          for (int j = 0; j < P; ++j) d[j] = mul2(both(w[k]), g[j]);
          reinterpret_cast<uint4*>(grad_in)[static_cast<long long>(row[k]) * pieces + p] = pack_piece<X>(d);
        }
      }
    }
  }
  if (!s_dot) return;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    float dot = dot2[k].x + dot2[k].y;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    if ((threadIdx.x & 31) == 0) s_dot[k][threadIdx.x >> 5] = dot;
  }
}
// One CTA per token (the dot products are sums over the whole row); either output may be absent.  THREADS: 256, three CTAs per
// SM (110 registers and two: 320 us instead of 303 at 8192 tokens x 8 rows of 7168 bf16), or 512 for fewer tokens than SMs (64
// tokens 5.1 us instead of 6.2).
template <typename X, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 3 : 1)
k_token_combine_backward(const uint8_t* grad, long long grad_pitch, const uint8_t* in, long long in_pitch,
                         const float* weights, int T, int K, int rows, int per, int pieces, const int* row_pairs,
                         const int* scatter_map, uint8_t* grad_in, float* grad_w) {
  __shared__ float s_dot[TOP_K][16];
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x;
  if (t < T) {
    const TokenPairs pairs = token_pairs(scatter_map, weights, t, K, rows);
    const uint4* grad_row = reinterpret_cast<const uint4*>(grad + t * grad_pitch);
    if (pairs.mask && __popc(pairs.mask) <= 2)
      combine_rows_backward<X, 2, 2>(grad_row, in, in_pitch, pairs, pieces, grad_in, grad_w ? s_dot : nullptr);
    else if (pairs.mask)
      combine_rows_backward<X, TOP_K, 1>(grad_row, in, in_pitch, pairs, pieces, grad_in, grad_w ? s_dot : nullptr);
    if (grad_w) {
      __syncthreads();
      if (threadIdx.x < K) {
        const uint32_t below = pairs.mask & ((1u << threadIdx.x) - 1u);
        float sum = 0.f;
        if (pairs.mask >> threadIdx.x & 1u)
          for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) sum += s_dot[__popc(below)][i];
        grad_w[static_cast<long long>(t) * K + threadIdx.x] = sum;
      }
    }
  }
  if (grad_in) {
    // behind the token's work: registers are what this kernel is short of (loaded ahead of it 311 us at 8192 tokens x 8 rows of
    // 7168 bf16, here 305.5; f16, which spills 20 bytes, 310)
    const int named = named_row(scatter_map, share_pair(row_pairs, per, rows), T * K);
    zero_unused_rows(named, per, rows, grad_in, pieces, 0, pieces);
  }
}

// w[t,k] = scale * s_k / (sum_j s_j + 1e-20) over the token's K selected experts, s = sigmoid(logit): the operations, and their
// order, of route_token, so that the weights of a selection made by b200moe_route_topk are its bits.  Eight lanes per token.
// An id outside 0 .. 255 has weight 0 and takes no part; a NaN logit makes its token's weights NaN (the sigmoid's clamp would
// take it for a large one, as the routing kernels do).
__device__ __forceinline__ float selected_sigmoid(const float* logits, long long t, int id, float sign) {
  if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(E_GLOBAL)) return 0.f;
  const float x = sign * ld_dep(logits + t * E_GLOBAL + id);
  return isnan(x) ? x : sigmoid_exact_ops(x);
}
__global__ void __launch_bounds__(256)
k_route_weights(const float* logits, const int* topk_idx, int T, int K, float scale, float* weights) {
  pdl_launch_dependents();
  pdl_wait();
  const long long t = static_cast<long long>(blockIdx.x) * (blockDim.x / TOP_K) + threadIdx.x / TOP_K;
  const int k = threadIdx.x % TOP_K;
  const bool live = t < T && k < K;
  const int id = live ? ld_dep(topk_idx + t * K + k) : -1;
  const float s = live ? selected_sigmoid(logits, t, id, 1.f) : 0.f;
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < TOP_K; ++j) sum = __fadd_rn(sum, __shfl_sync(0xffffffffu, s, j, TOP_K));
  if (live) weights[t * K + k] = __fmul_rn(__fdiv_rn(s, __fadd_rn(sum, 1e-20f)), scale);
}

// With S = sum_j s_j + 1e-20 and g = the weights' gradient:
//   grad_logit_k = s_k * (1 - s_k) * scale / S * (g_k - sum_j g_j s_j / S),  every other column 0.
// 1 - sigmoid(x) is taken as sigmoid(-x), which loses nothing where s is near 1.  A warp works on four tokens, eight lanes
// each, and puts their rows together in shared memory; an expert named twice gets both terms, added in the order of k by the
// first lane that names it.  (A warp per token with the columns in registers: 16384 tokens 7.7 us, now 6.5.)
constexpr int ROUTE_GRAD_WARPS = 8, ROUTE_GRAD_TOKENS = 4;
__global__ void __launch_bounds__(ROUTE_GRAD_WARPS * 32)
k_route_weights_backward(const float* logits, const int* topk_idx, const float* grad, int T, int K, float scale,
                         float* grad_logits) {
  __shared__ float4 s_rows[ROUTE_GRAD_WARPS][ROUTE_GRAD_TOKENS * E_GLOBAL / 4];
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, k = lane % TOP_K;
  constexpr int PIECES = ROUTE_GRAD_TOKENS * E_GLOBAL / 4 / 32;   // of the four rows, per lane
  float4* rows = s_rows[warp];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) rows[i * 32 + lane] = make_float4(0.f, 0.f, 0.f, 0.f);
  pdl_wait();
  const long long t0 = (static_cast<long long>(blockIdx.x) * ROUTE_GRAD_WARPS + warp) * ROUTE_GRAD_TOKENS;
  const long long t = t0 + lane / TOP_K;
  const bool live = t < T && k < K;
  const int id = live ? ld_dep(topk_idx + t * K + k) : -1;
  const bool valid = static_cast<uint32_t>(id) < static_cast<uint32_t>(E_GLOBAL);
  const float g = live ? ld_dep(grad + t * K + k) : 0.f;
  const float s = selected_sigmoid(logits, t, id, 1.f), c = selected_sigmoid(logits, t, id, -1.f);
  float total = s, mix = valid ? g * s : 0.f;
#pragma unroll
  for (int d = TOP_K / 2; d > 0; d >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, d);
    mix += __shfl_xor_sync(0xffffffffu, mix, d);
  }
  total += 1e-20f;
  const float grad_k = s * c * (scale / total) * (g - mix / total);
  const uint32_t same = __match_any_sync(0xffffffffu, valid ? (lane / TOP_K) * E_GLOBAL + id : -1 - lane);
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < TOP_K; ++j) {
    const float v = __shfl_sync(0xffffffffu, grad_k, j, TOP_K);
    if (same >> ((lane & ~(TOP_K - 1)) + j) & 1u) sum += v;
  }
  __syncwarp();
  if (valid && __ffs(same) - 1 == lane) reinterpret_cast<float*>(rows)[(lane / TOP_K) * E_GLOBAL + id] = sum;
  __syncwarp();
  float4* dst = reinterpret_cast<float4*>(grad_logits + t0 * E_GLOBAL);
#pragma unroll
  for (int i = 0; i < PIECES; ++i)   // piece i * 32 + lane is of token i * 32 / 64
    if (t0 + i * 32 / (E_GLOBAL / 4) < T) dst[i * 32 + lane] = rows[i * 32 + lane];
}

// Pairs per CTA and CTAs of the sort: whole rounds of SORT_THREADS pairs, at most SORT_MAX_CTAS CTAs.
static long long sort_pairs_per_cta(long long n_pairs) {
  const long long rounds = (n_pairs + SORT_THREADS - 1) / SORT_THREADS;
  const long long per = (rounds + SORT_MAX_CTAS - 1) / SORT_MAX_CTAS;
  return (per < 1 ? 1 : per) * SORT_THREADS;
}

size_t token_sort_scratch_bytes(int T, int K, int E_local) {
  const long long n_pairs = static_cast<long long>(T) * K;
  const long long per = sort_pairs_per_cta(n_pairs), ctas = (n_pairs + per - 1) / per;
  return ctas <= SORT_ONE_LAUNCH_CTAS ? 0 : static_cast<size_t>(ctas) * E_local * sizeof(int);
}

int launch_token_sort(const int* topk_idx, int T, int K, int E_local, int offset, int align, int rows, int* hist,
                      int* counts, int* offsets, int* row_pairs, int* scatter_map, cudaStream_t st) {
  const long long n_pairs = static_cast<long long>(T) * K;
  const long long per = sort_pairs_per_cta(n_pairs);
  unsigned ctas = n_pairs == 0 ? 1u : static_cast<unsigned>((n_pairs + per - 1) / per);
  if (ctas <= SORT_ONE_LAUNCH_CTAS) {
    // few pairs in many rows (segments padded to 128): more CTAs mark the unused rows (64 tokens, 33280 rows
    // 6.6 us, now 4.4)
    hist = nullptr;
    const unsigned marking = (static_cast<unsigned>(rows) + 4 * SORT_THREADS - 1) / (4 * SORT_THREADS);
    if (marking > ctas) ctas = marking < SORT_ONE_LAUNCH_CTAS ? marking : SORT_ONE_LAUNCH_CTAS;
  } else {
    B200MOE_CUDA_TRY(launch_pdl(k_token_count, dim3(ctas), dim3(SORT_THREADS), 0, st, topk_idx, n_pairs, per, offset,
                                E_local, hist));
  }
  B200MOE_CUDA_TRY(launch_pdl(k_token_place, dim3(ctas), dim3(SORT_THREADS), 0, st, topk_idx, n_pairs, per, offset, E_local,
                              align, rows, static_cast<const int*>(hist), counts, offsets, row_pairs, scatter_map));
  return B200MOE_OK;
}

// One CTA per token, more where the capacity has many rows per token.
static unsigned token_ctas(int T, int rows) {
  const int by_rows = (rows + TOP_K - 1) / TOP_K;
  return static_cast<unsigned>(T > by_rows ? T : by_rows);
}
// Rows that each of them looks through: at most nine.
static int rows_per_cta(int rows, unsigned ctas) { return static_cast<int>((rows + static_cast<long long>(ctas) - 1) / ctas); }
static unsigned token_threads(int pieces, int most) {
  const int threads = (pieces + 31) / 32 * 32;
  return static_cast<unsigned>(threads < most ? threads : most);
}
// Parts of a row, a CTA each, while the batch alone does not fill the GPU: a call of few tokens is as long as a thread's
// chain of loads and stores.  us with one CTA per token / with parts, at 7168 bf16 columns: gather of 1 token 3.9 / 2.3, of
// 333 tokens 14.8 / 8.1; combine 3.1 / 1.6 and 6.1 / 5.0.  (Twice as many parts: 333 tokens 7.6 and 5.8.)
constexpr unsigned TOKEN_FILL_CTAS = 4;   // per SM
static unsigned token_parts(unsigned ctas, int pieces, unsigned threads, int num_sms) {
  const unsigned most = (pieces + threads - 1) / threads;
  const unsigned want = (TOKEN_FILL_CTAS * num_sms + ctas - 1) / ctas;
  return want < most ? want : most;
}

int launch_token_gather(const void* x, long long x_pitch, int T, int K, int rows, int pieces, const int* row_pairs,
                        const int* scatter_map, void* out, int num_sms, cudaStream_t st) {
  const unsigned ctas = token_ctas(T, rows), threads = token_threads(pieces, 256);
  B200MOE_CUDA_TRY(launch_pdl(k_token_gather, dim3(ctas, token_parts(ctas, pieces, threads, num_sms)), dim3(threads), 0, st,
                              static_cast<const uint8_t*>(x), x_pitch, T, K, rows, rows_per_cta(rows, ctas), pieces, row_pairs,
                              scatter_map, static_cast<uint8_t*>(out)));
  return B200MOE_OK;
}

template <typename F>
static int with_row_type(int type, F&& f) {
  if (type == B200MOE_DTYPE_F32) return f(float());
  if (type == B200MOE_DTYPE_F16) return f(__half());
  return f(__nv_bfloat16());
}

int launch_token_combine(const void* in, long long in_pitch, int type, const float* weights, int T, int K, int rows,
                         int pieces, const int* scatter_map, void* out, int num_sms, cudaStream_t st) {
  return with_row_type(type, [&](auto xt) -> int {
    const unsigned threads = token_threads(pieces, 256);
    const unsigned parts = token_parts(T, pieces, threads, num_sms);
    B200MOE_CUDA_TRY(launch_pdl(k_token_combine<decltype(xt)>, dim3(T, parts), dim3(threads), 0, st,
                                static_cast<const uint8_t*>(in), in_pitch, weights, K, rows, pieces, scatter_map,
                                static_cast<uint8_t*>(out)));
    return B200MOE_OK;
  });
}

int launch_token_combine_backward(const void* grad, long long grad_pitch, const void* in, long long in_pitch, int type,
                                  const float* weights, int T, int K, int rows, int pieces, const int* row_pairs,
                                  const int* scatter_map, void* grad_in, float* grad_w, int num_sms,
                                  cudaStream_t st) {
  return with_row_type(type, [&](auto xt) -> int {
    using X = decltype(xt);
    const bool few = T <= num_sms;
    auto kern = few ? k_token_combine_backward<X, 512> : k_token_combine_backward<X, 256>;
    const unsigned ctas = grad_in ? token_ctas(T, rows) : static_cast<unsigned>(T);
    B200MOE_CUDA_TRY(launch_pdl(kern, dim3(ctas), dim3(token_threads(pieces, few ? 512 : 256)), 0, st,
                                static_cast<const uint8_t*>(grad), grad_pitch, static_cast<const uint8_t*>(in), in_pitch,
                                weights, T, K, rows, rows_per_cta(rows, ctas), pieces, row_pairs, scatter_map,
                                static_cast<uint8_t*>(grad_in), grad_w));
    return B200MOE_OK;
  });
}

int launch_route_weights(const float* logits, const int* topk_idx, int T, int K, float scale, float* weights,
                         cudaStream_t st) {
  B200MOE_CUDA_TRY(launch_pdl(k_route_weights, dim3((T + 31) / 32), dim3(256), 0, st, logits, topk_idx, T, K, scale,
                              weights));
  return B200MOE_OK;
}

int launch_route_weights_backward(const float* logits, const int* topk_idx, const float* grad, int T, int K, float scale,
                                  float* grad_logits, cudaStream_t st) {
  B200MOE_CUDA_TRY(launch_pdl(k_route_weights_backward,
                              dim3((T + ROUTE_GRAD_WARPS * ROUTE_GRAD_TOKENS - 1) / (ROUTE_GRAD_WARPS * ROUTE_GRAD_TOKENS)),
                              dim3(ROUTE_GRAD_WARPS * 32), 0, st, logits, topk_idx, grad, T, K,
                              scale, grad_logits));
  return B200MOE_OK;
}

}  // namespace b200moe
