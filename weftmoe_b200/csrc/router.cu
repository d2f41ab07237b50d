// Router operators: top-k choice with gates, per-expert counts, the balance loss, and their gradients.
//
// One warp holds one row of logits in registers (expert j * 32 + lane in slot j), so a row is read once
// and everything else is arithmetic on registers and shuffles.  With x the row, over its available experts
// (logit above -inf):
//   softmax   s_e = exp(x_e - m) / sum            sigmoid   s_e = 1 / (1 + exp(-x_e))
//   routes    the K largest of x (both scores rise with x), or of s + bias; ties to the lowest index
//   gates     scale * s_k, or scale * s_k / (sum of the chosen s)
//   p         s_e / (sum of the row's s)           the row's share of each expert
//   loss      mean over sequences b with a live row of  sum_e f_be P_be,
//             f_be = E c_be / sum_e c_be,  P_be = mean of p over the sequence's live rows
// Sums over rows are taken per block in a fixed order into records, and the records in a fixed order by a
// second kernel, so results do not depend on the order in which blocks run.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/weftmoe_b200.h"
#include "kernels.h"

using namespace wm;

namespace {

constexpr int kWarps = 8;
constexpr int kMaxExperts = 1024;
constexpr int kMaxBlocks = 1184;  // 148 SMs x 8
constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }  // the gradient's type
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }             // is the logits'

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, d));
  return v;
}
// Unsigned words in the order of the floats; 0 is below every one of them and means "not available".
__device__ __forceinline__ unsigned ordered(float v) {
  v += 0.0f;  // -0 and 0 tie
  const unsigned u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ unsigned long long ordered(double v) {
  v += 0.0;
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(v));
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

struct Rows {
  const void* logits;
  long long stride;
  int tokens, experts, top_k, sigmoid, renormalize;
  float scale;
  const float* bias;
  const uint8_t* padding;
  const int* sequences;
  int num_sequences;  // 1 without offsets
  int chunk;          // rows of one block
};

// Sequence of a row: the number of ends at or below it.  num_sequences = behind the last one.
__device__ __forceinline__ int sequence_of(const Rows& a, int row) {
  if (a.sequences == nullptr) return 0;
  int lo = 0, hi = a.num_sequences;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(a.sequences + mid + 1) <= row) lo = mid + 1; else hi = mid;
  }
  return lo;
}
__device__ __forceinline__ int sequence_end(const Rows& a, int b) {
  return a.sequences == nullptr || b >= a.num_sequences ? a.tokens : min(__ldg(a.sequences + b + 1), a.tokens);
}
// Rows that padding marks, or that no sequence holds, are dead: no route, no gradient, in no sum.
__device__ __forceinline__ bool row_live(const Rows& a, int row, int b) {
  if (a.padding != nullptr && a.padding[row]) return false;
  return a.sequences == nullptr || (b < a.num_sequences && row >= __ldg(a.sequences));
}

template <class T, int V>
__device__ __forceinline__ void load_row(const Rows& a, int row, int lane, float (&x)[V]) {
  const T* p = static_cast<const T*>(a.logits) + static_cast<long long>(row) * a.stride;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int e = j * 32 + lane;
    x[j] = e < a.experts ? as_float(p[e]) : -INFINITY;
  }
}

// What a row's arithmetic needs of the whole row.  top: the largest logit.  For softmax s_e = exp(x_e - top) / sum;
// for sigmoid, p_e = hat(x_e) / sum with hat(x) = s(x) * exp(-min(top, 0)): a row of very negative logits keeps
// its shares.
struct RowStats {
  float top, sum;
  bool bad, any;  // bad: NaN (or, for softmax, +inf) among the logits; any: an available expert
};
__device__ __forceinline__ float sigmoid_hat(float x, float top) {
  return expf(fminf(x, 0.0f) - fminf(top, 0.0f)) / (1.0f + expf(-fabsf(x)));
}
// 1 - s(x) without cancellation.
__device__ __forceinline__ float sigmoid_rest(float x) { return 1.0f / (1.0f + expf(x)); }

// h[j]: exp(x - top) or hat(x); the share of the row is h / sum.
template <int V>
__device__ __forceinline__ RowStats row_stats(const float (&x)[V], bool sigmoid, float (&h)[V]) {
  RowStats r;
  float top = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    top = fmaxf(top, x[j]);
    bad |= x[j] != x[j] || (!sigmoid && x[j] == INFINITY);
  }
  r.top = warp_max(top);
  r.bad = __any_sync(kAll, bad);
  r.any = r.top > -INFINITY;
  float sum = 0.0f;
  if (r.any) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      h[j] = sigmoid ? sigmoid_hat(x[j], r.top) : expf(x[j] - r.top);
      sum += h[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = 0.0f;
  }
  r.sum = warp_sum(sum);
  return r;
}

// K rounds of a warp-wide maximum.  Lane k gets choice k: its expert (-1 when none is left) and its logit.
template <int V>
__device__ __forceinline__ void choose_by_logit(const float (&x)[V], int top_k, int lane, int& expert, float& logit) {
  unsigned key[V];
#pragma unroll
  for (int j = 0; j < V; ++j) key[j] = x[j] > -INFINITY ? ordered(x[j]) : 0u;
  expert = -1;
  logit = 0.0f;
  for (int k = 0; k < top_k; ++k) {
    unsigned best = 0;
    int at = 0;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (key[j] > best) { best = key[j]; at = j; }
    const unsigned most = __reduce_max_sync(kAll, best);
    if (most == 0) break;
    const unsigned e = __reduce_min_sync(kAll, best == most ? at * 32 + lane : 0x7fffffffu);
    if (lane == k) { expert = static_cast<int>(e); logit = unordered(most); }
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j * 32 + lane == static_cast<int>(e)) key[j] = 0;
  }
}

// The same on s + bias.  Scores and their sums with the bias are taken in 64 bits: two experts whose 32-bit
// values are equal or swapped by a rounding would otherwise come out in another order than their scores have.
template <int V>
__device__ __forceinline__ void choose_by_score(const float (&x)[V], const Rows& a, float top, int lane, int& expert,
                                                float& logit) {
  double s[V];
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    s[j] = a.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(x[j]))) : exp(static_cast<double>(x[j]) - top);
    sum += s[j];
  }
  sum = warp_sum(sum);
  unsigned long long key[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int e = j * 32 + lane;
    key[j] = x[j] > -INFINITY
                 ? ordered((a.sigmoid ? s[j] : s[j] / sum) + static_cast<double>(__ldg(a.bias + e))) : 0ull;
  }
  expert = -1;
  logit = 0.0f;
  for (int k = 0; k < a.top_k; ++k) {
    unsigned long long best = 0;
    int at = 0;
    float its = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (key[j] > best) { best = key[j]; at = j; its = x[j]; }
    const unsigned high = static_cast<unsigned>(best >> 32), low = static_cast<unsigned>(best);
    const unsigned most_high = __reduce_max_sync(kAll, high);
    if (most_high == 0) break;
    const unsigned most_low = __reduce_max_sync(kAll, high == most_high ? low : 0u);
    const bool mine = high == most_high && low == most_low;
    const unsigned e = __reduce_min_sync(kAll, mine ? at * 32 + lane : 0x7fffffffu);
    const float v = __shfl_sync(kAll, its, e & 31);
    if (lane == k) { expert = static_cast<int>(e); logit = v; }
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j * 32 + lane == static_cast<int>(e)) key[j] = 0;
  }
}

// Lane k: choice k's weight (its gate without the scale).  stats belong to the whole row.
__device__ __forceinline__ float choice_weight(const Rows& a, const RowStats& stats, int expert, float logit) {
  const bool chosen = expert >= 0;
  if (a.renormalize) {
    const float top = warp_max(chosen ? logit : -INFINITY);
    float h = 0.0f;
    if (chosen) h = a.sigmoid ? sigmoid_hat(logit, top) : expf(logit - top);
    const float sum = warp_sum(h);
    return chosen ? h / sum : 0.0f;
  }
  if (!chosen) return 0.0f;
  return a.sigmoid ? sigmoid_hat(logit, 0.0f) : expf(logit - stats.top) / stats.sum;
}

// Records of the balance sums: record (chunk c, sequence b) is number c + b.  Chunks and sequences both walk the
// rows in order, so c + b names each pair that meets once.
struct Records {
  float* share;   // [records][experts] sum of p
  int* counts;    // [records][experts], null without a choice
  int* rows;      // [records][2] live rows, routes
  unsigned* ticket;
};

template <class T, int V>
__global__ void __launch_bounds__(kWarps * 32)
router_forward_kernel(const Rows a, int* __restrict__ routes, float* __restrict__ gates, const Records rec) {
  extern __shared__ float smem[];
  float* part = smem;                                              // [kWarps][experts]
  int* seen = reinterpret_cast<int*>(smem + kWarps * a.experts);   // [experts]
  __shared__ int live_rows[kWarps], live_routes[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool balance = rec.share != nullptr, choose = routes != nullptr;
  if (balance && blockIdx.x == 0 && threadIdx.x == 0) *rec.ticket = 0;   // for the kernel that sums the records
  const int first = blockIdx.x * a.chunk, last = min(first + a.chunk, a.tokens);
  if (balance)
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) seen[e] = 0;
  __syncthreads();

  int row0 = first;
  while (row0 < last) {
    const int b = sequence_of(a, row0);
    const int row1 = balance ? max(row0 + 1, min(last, sequence_end(a, b))) : last;
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.0f;
    int rows = 0, taken = 0;
    for (int row = row0 + warp; row < row1; row += kWarps) {
      float x[V], h[V];
      const bool live = row_live(a, row, balance ? b : sequence_of(a, row));
      int expert = -1;
      float weight = 0.0f;
      if (live) {
        load_row<T, V>(a, row, lane, x);
        const RowStats stats = row_stats<V>(x, a.sigmoid, h);
        if (choose) {
          float logit = 0.0f;
          if (stats.bad) {   // no distribution: valid routes and NaN gates, so that it shows in the output
            expert = lane < a.top_k ? lane : -1;
            weight = NAN;
          } else {
            if (a.bias != nullptr) choose_by_score<V>(x, a, stats.top, lane, expert, logit);
            else choose_by_logit<V>(x, a.top_k, lane, expert, logit);
            weight = choice_weight(a, stats, expert, logit);
          }
        }
        if (balance && (stats.any || stats.bad)) {
          ++rows;
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] += stats.bad ? NAN : h[j] / stats.sum;
          if (choose && expert >= 0) { atomicAdd(seen + expert, 1); ++taken; }
        }
      }
      if (choose && lane < a.top_k) {
        routes[static_cast<long long>(row) * a.top_k + lane] = expert;
        gates[static_cast<long long>(row) * a.top_k + lane] = expert >= 0 ? a.scale * weight : 0.0f;
      }
    }
    if (balance) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j * 32 + lane < a.experts) part[warp * a.experts + j * 32 + lane] = acc[j];
      taken = __reduce_add_sync(kAll, taken);
      if (lane == 0) { live_rows[warp] = rows; live_routes[warp] = taken; }
      __syncthreads();
      if (b < a.num_sequences) {
        const long long record = blockIdx.x + b;
        for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
          float sum = 0.0f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) sum += part[w * a.experts + e];
          rec.share[record * a.experts + e] = sum;
          if (choose) { rec.counts[record * a.experts + e] = seen[e]; seen[e] = 0; }
        }
        if (threadIdx.x == 0) {
          int n = 0, c = 0;
          for (int w = 0; w < kWarps; ++w) { n += live_rows[w]; c += live_routes[w]; }
          rec.rows[2 * record] = n;
          rec.rows[2 * record + 1] = c;
        }
      }
      __syncthreads();
    }
    row0 = row1;
  }
}

// Sums the records of one sequence for 32 experts per block (8 warps take every eighth record), then the last
// block to finish sums the blocks' parts of the loss in their order.
// table: [num_sequences][experts] of (f - 1) / n_b, the loss's slope by p up to a constant (p sums to one, so a
// constant drops out of the gradient; without it the differences near f = 1 keep their digits), then 1 / live sequences.
__global__ void __launch_bounds__(kWarps * 32)
balance_finish_kernel(const Rows a, const Records rec, const int* __restrict__ given, int* __restrict__ counts,
                      float* __restrict__ table, float* parts, float* __restrict__ loss) {
  __shared__ float share[kWarps][32];
  __shared__ int count[kWarps][32];
  __shared__ int rows[kWarps], taken[kWarps];
  __shared__ bool is_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.y, e = blockIdx.x * 32 + lane;
  const int row0 = a.sequences == nullptr ? 0 : max(0, __ldg(a.sequences + b));
  const int row1 = sequence_end(a, b);
  float sum = 0.0f;
  int c = 0, n = 0, total = 0;
  if (row0 < row1) {
    for (int chunk = row0 / a.chunk + warp; chunk <= (row1 - 1) / a.chunk; chunk += kWarps) {
      const long long record = chunk + b;
      if (e < a.experts) {
        sum += rec.share[record * a.experts + e];
        if (rec.counts != nullptr) c += rec.counts[record * a.experts + e];
      }
      n += rec.rows[2 * record];
      total += rec.rows[2 * record + 1];
    }
  }
  share[warp][lane] = sum;
  count[warp][lane] = c;
  if (lane == 0) { rows[warp] = n; taken[warp] = total; }
  __syncthreads();
  if (warp == 0) {
    sum = 0.0f;
    c = n = 0;
    long long all = 0;
    for (int w = 0; w < kWarps; ++w) { sum += share[w][lane]; c += count[w][lane]; n += rows[w]; all += taken[w]; }
    if (given != nullptr) {
      all = 0;
      for (int i = lane; i < a.experts; i += 32) all += given[static_cast<long long>(b) * a.experts + i];
#pragma unroll
      for (int d = 16; d; d >>= 1) all += __shfl_xor_sync(kAll, all, d);
      c = e < a.experts ? given[static_cast<long long>(b) * a.experts + e] : 0;
    }
    float f = 0.0f, part = 0.0f;
    if (e < a.experts) {
      f = all > 0 ? static_cast<float>(static_cast<double>(c) * a.experts / static_cast<double>(all)) : 0.0f;
      const float inv = n > 0 ? 1.0f / static_cast<float>(n) : 0.0f;
      part = n > 0 ? f * (sum / static_cast<float>(n)) : 0.0f;
      table[static_cast<long long>(b) * a.experts + e] = (f - 1.0f) * inv;
      if (counts != nullptr) counts[static_cast<long long>(b) * a.experts + e] = c;
    }
    part = warp_sum(part);
    if (lane == 0) {
      float* out = parts + 2 * (static_cast<long long>(b) * gridDim.x + blockIdx.x);
      out[0] = part;
      out[1] = blockIdx.x == 0 && n > 0 ? 1.0f : 0.0f;
      __threadfence();
      is_last = atomicAdd(rec.ticket, 1u) == gridDim.x * gridDim.y - 1;
    }
  }
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  __shared__ double sums[kWarps], lives[kWarps];
  double l = 0.0, live = 0.0;
  const long long blocks = static_cast<long long>(gridDim.x) * gridDim.y;
  for (long long i = threadIdx.x; i < blocks; i += blockDim.x) { l += __ldcg(parts + 2 * i); live += __ldcg(parts + 2 * i + 1); }
  l = warp_sum(l);
  live = warp_sum(live);
  if (lane == 0) { sums[warp] = l; lives[warp] = live; }
  __syncthreads();
  if (threadIdx.x == 0) {
    l = live = 0.0;
    for (int w = 0; w < kWarps; ++w) { l += sums[w]; live += lives[w]; }
    const double inv = live > 0.0 ? 1.0 / live : 0.0;
    *loss = static_cast<float>(live > 0.0 ? l * inv : 0.0);
    table[static_cast<long long>(a.num_sequences) * a.experts] = static_cast<float>(inv);
  }
}

// d logits of one row per warp:
//   gates, w = the choice's weight, g = scale * dgate:
//     softmax, renormalised  w_k (g_k - sum w g) at the chosen      softmax  s_e ([chosen] g_e - sum s g)
//     sigmoid, renormalised  (1 - s_k) w_k (g_k - sum w g)           sigmoid  (1 - s_k) s_k g_k
//   loss, q = the table's row times dloss / live sequences:  p_e (q_e - sum p q), times 1 - s_e for sigmoid.
template <class T, int V>
__global__ void __launch_bounds__(kWarps * 32)
router_backward_kernel(const Rows a, const int* __restrict__ routes, const float* __restrict__ dgates,
                       const float* __restrict__ table, const float* __restrict__ dloss, T* __restrict__ dlogits) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float push = table != nullptr
      ? __ldg(dloss) * __ldg(table + static_cast<long long>(a.num_sequences) * a.experts) : 0.0f;
  for (long long r = static_cast<long long>(blockIdx.x) * kWarps + warp; r < a.tokens;
       r += static_cast<long long>(gridDim.x) * kWarps) {
    const int row = static_cast<int>(r);
    const int b = sequence_of(a, row);
    float x[V], h[V], d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = 0.0f;
    if (row_live(a, row, b)) {
      load_row<T, V>(a, row, lane, x);
      const RowStats stats = row_stats<V>(x, a.sigmoid, h);
      if (stats.bad) {
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = NAN;
      } else if (stats.any) {
        const float inv = 1.0f / stats.sum;
        if (table != nullptr) {
          const float* q = table + static_cast<long long>(b) * a.experts;
          float mean = 0.0f, w[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int e = j * 32 + lane;
            w[j] = e < a.experts ? __ldg(q + e) : 0.0f;
            h[j] *= inv;
            mean = fmaf(h[j], w[j], mean);
          }
          mean = warp_sum(mean);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            d[j] = push * h[j] * (w[j] - mean);
            if (a.sigmoid) d[j] *= sigmoid_rest(x[j]);
          }
        }
        if (routes != nullptr) {
          int expert = -1;
          float logit = 0.0f, g = 0.0f;
          if (lane < a.top_k) {
            expert = routes[r * a.top_k + lane];
            if (static_cast<unsigned>(expert) >= static_cast<unsigned>(a.experts)) expert = -1;
            if (expert >= 0) {
              logit = as_float((static_cast<const T*>(a.logits) + r * a.stride)[expert]);
              g = a.scale * dgates[r * a.top_k + lane];
            }
          }
          const float w = choice_weight(a, stats, expert, logit);
          float mean = 0.0f;
          if (a.renormalize || !a.sigmoid) mean = warp_sum(w * g);
          float c = w * (a.renormalize ? g - mean : g);
          if (a.sigmoid) c *= sigmoid_rest(logit);
          if (!a.renormalize && !a.sigmoid) {
            const float factor = table != nullptr ? mean : mean * inv;   // h holds shares when the loss ran first
#pragma unroll
            for (int j = 0; j < V; ++j) d[j] -= h[j] * factor;
          }
          for (int k = 0; k < a.top_k; ++k) {
            const int e = __shfl_sync(kAll, expert, k);
            const float v = __shfl_sync(kAll, c, k);
            if (e >= 0 && (e & 31) == lane) {
#pragma unroll
              for (int j = 0; j < V; ++j)
                if (j == e >> 5) d[j] += v;
            }
          }
        }
      }
    }
    T* out = dlogits + r * a.experts;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = j * 32 + lane;
      if (e < a.experts) put(out + e, d[j]);
    }
  }
}

// Routes per expert: a block counts its rows in shared memory and adds the whole numbers to the result.
__global__ void __launch_bounds__(256)
expert_counts_kernel(const Rows a, const int* __restrict__ routes, int* __restrict__ counts) {
  extern __shared__ int seen_counts[];
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) seen_counts[e] = 0;
  __syncthreads();
  const int first = blockIdx.x * a.chunk, last = min(first + a.chunk, a.tokens);
  int row0 = first;
  while (row0 < last) {
    const int b = sequence_of(a, row0);
    const int row1 = max(row0 + 1, min(last, sequence_end(a, b)));
    if (b < a.num_sequences) {
      const int from = a.sequences == nullptr ? row0 : max(row0, __ldg(a.sequences));   // rows no sequence holds
      const long long end = static_cast<long long>(row1) * a.top_k;
      for (long long i = static_cast<long long>(from) * a.top_k + threadIdx.x; i < end; i += blockDim.x) {
        const int e = routes[i];
        if (static_cast<unsigned>(e) < static_cast<unsigned>(a.experts)) atomicAdd(seen_counts + e, 1);
      }
      __syncthreads();
      for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
        if (seen_counts[e]) atomicAdd(counts + static_cast<long long>(b) * a.experts + e, seen_counts[e]);
        seen_counts[e] = 0;
      }
      __syncthreads();
    }
    row0 = row1;
  }
}

// ------------------------------------------------------------------ host side
struct Plan {
  int chunk, blocks;
  long long records, parts;
  long long share, counts, rows, part, ticket, bytes;   // offsets into the workspace
};

Plan plan_of(const wm_router& r) {
  Plan p{};
  const int sequences = r.sequences ? r.num_sequences : 1;
  const int want = (r.tokens + kWarps - 1) / kWarps;
  const int blocks = want < kMaxBlocks ? (want > 0 ? want : 1) : kMaxBlocks;
  p.chunk = r.tokens > 0 ? (r.tokens + blocks - 1) / blocks : 1;
  p.blocks = r.tokens > 0 ? (r.tokens + p.chunk - 1) / p.chunk : 1;
  p.records = static_cast<long long>(p.blocks) + sequences;
  p.parts = static_cast<long long>((r.experts + 31) / 32) * sequences;
  p.share = 0;
  p.counts = p.share + p.records * r.experts * 4;
  p.rows = p.counts + p.records * r.experts * 4;
  p.part = p.rows + p.records * 8;
  p.ticket = p.part + p.parts * 8;
  p.bytes = p.ticket + 16;
  return p;
}

int check_rows(const char* what, const wm_router* r) {
  if (!r) { set_error("%s: null arguments", what); return WM_ERR_INVALID; }
  if (r->tokens < 0 || r->experts < 1 || r->experts > kMaxExperts || r->dtype < 0 || r->dtype > 2 ||
      r->row_stride < r->experts || (r->score != 0 && r->score != 1) || (r->tokens > 0 && !r->logits) ||
      (r->sequences ? r->num_sequences < 1 : r->num_sequences != 0) || r->num_sequences > 65535) {
    set_error("%s: logits must be [tokens][experts] BF16 / FP32 / FP16 rows of 1..%d experts, score 0 (softmax) or 1 "
              "(sigmoid), 1..65535 sequences with their offsets", what, kMaxExperts);
    return WM_ERR_INVALID;
  }
  return WM_OK;
}
int check_choice(const char* what, const wm_router* r) {
  if (r->top_k < 1 || r->top_k > 32 || r->top_k > r->experts || !(r->scale > 0.0f) || !(r->scale < INFINITY)) {
    set_error("%s: top_k must be in [1, min(32, experts)], scale finite and positive", what);
    return WM_ERR_INVALID;
  }
  return WM_OK;
}

Rows rows_of(const wm_router& r, const Plan& p) {
  return Rows{r.logits, r.row_stride, r.tokens, r.experts, r.top_k, r.score, r.renormalize, r.scale, r.bias, r.padding,
              r.sequences, r.sequences ? r.num_sequences : 1, p.chunk};
}
Records records_of(const Plan& p, void* workspace, bool counts) {
  char* w = static_cast<char*>(workspace);
  return Records{reinterpret_cast<float*>(w + p.share), counts ? reinterpret_cast<int*>(w + p.counts) : nullptr,
                 reinterpret_cast<int*>(w + p.rows), reinterpret_cast<unsigned*>(w + p.ticket)};
}

template <class T, int V>
int forward_of(const Rows& a, const Plan& p, int* routes, float* gates, const Records& rec, cudaStream_t stream) {
  const int smem = rec.share ? (kWarps + 1) * a.experts * 4 : 0;
  router_forward_kernel<T, V><<<p.blocks, kWarps * 32, smem, stream>>>(a, routes, gates, rec);
  return 0;
}
template <class T, int V>
int backward_of(const Rows& a, const int* routes, const float* dgates, const float* table, const float* dloss,
                void* dlogits, cudaStream_t stream) {
  const int want = (a.tokens + kWarps - 1) / kWarps;
  router_backward_kernel<T, V><<<want < 8 * kMaxBlocks ? want : 8 * kMaxBlocks, kWarps * 32, 0, stream>>>(
      a, routes, dgates, table, dloss, static_cast<T*>(dlogits));
  return 0;
}

// Calls f<T, V>: V slots of 32 experts hold a row.
#define WM_ROUTER_BY_SIZE(T, experts, f, ...)            \
  ((experts) <= 32    ? f<T, 1>(__VA_ARGS__)             \
   : (experts) <= 64  ? f<T, 2>(__VA_ARGS__)             \
   : (experts) <= 128 ? f<T, 4>(__VA_ARGS__)             \
   : (experts) <= 256 ? f<T, 8>(__VA_ARGS__)             \
   : (experts) <= 512 ? f<T, 16>(__VA_ARGS__)            \
                      : f<T, 32>(__VA_ARGS__))
#define WM_ROUTER_DISPATCH(dtype, experts, f, ...)                                  \
  ((dtype) == 0   ? WM_ROUTER_BY_SIZE(__nv_bfloat16, experts, f, __VA_ARGS__)       \
   : (dtype) == 1 ? WM_ROUTER_BY_SIZE(float, experts, f, __VA_ARGS__)               \
                  : WM_ROUTER_BY_SIZE(__half, experts, f, __VA_ARGS__))

int finish(const Rows& a, const Plan& p, const Records& rec, const int* given, int* counts, float* table,
           void* workspace, float* loss, cudaStream_t stream) {
  const dim3 grid((a.experts + 31) / 32, a.num_sequences);
  balance_finish_kernel<<<grid, kWarps * 32, 0, stream>>>(
      a, rec, given, counts, table, reinterpret_cast<float*>(static_cast<char*>(workspace) + p.part), loss);
  count_launch();
  WM_CUDA(cudaGetLastError());
  return WM_OK;
}

}  // namespace

extern "C" int wm_router_workspace(const wm_router* r, int64_t* bytes) {
  if (int rc = check_rows("wm_router_workspace", r)) return rc;
  if (!bytes) { set_error("wm_router_workspace: null result"); return WM_ERR_INVALID; }
  *bytes = plan_of(*r).bytes;
  return WM_OK;
}

extern "C" int wm_router_forward(const wm_router* r, int32_t* routes, float* gates, int32_t* counts, float* loss,
                                 float* table, void* workspace, int64_t workspace_bytes, void* stream_) {
  if (int rc = check_rows("wm_router_forward", r)) return rc;
  if (int rc = check_choice("wm_router_forward", r)) return rc;
  const Plan p = plan_of(*r);
  const bool balance = counts || loss || table || workspace;
  if ((r->tokens > 0 && (!routes || !gates)) ||
      (balance && (!counts || !loss || !table || !workspace || workspace_bytes < p.bytes ||
                   reinterpret_cast<uintptr_t>(workspace) % 16))) {
    set_error("wm_router_forward: null output, or a missing or small workspace (wm_router_workspace, 16-byte aligned)");
    return WM_ERR_INVALID;
  }
  if (r->tokens == 0 && !balance) return WM_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const Rows a = rows_of(*r, p);
  const Records rec = balance ? records_of(p, workspace, true) : Records{};
  // with no rows the kernel still clears the ticket of the kernel behind it
  WM_ROUTER_DISPATCH(r->dtype, r->experts, forward_of, a, p, routes, gates, rec, stream);
  count_launch();
  WM_CUDA(cudaGetLastError());
  return balance ? finish(a, p, rec, nullptr, counts, table, workspace, loss, stream) : WM_OK;
}

extern "C" int wm_balance_forward(const wm_router* r, const int32_t* counts, float* loss, float* table,
                                  void* workspace, int64_t workspace_bytes, void* stream_) {
  if (int rc = check_rows("wm_balance_forward", r)) return rc;
  const Plan p = plan_of(*r);
  if (!counts || !loss || !table || !workspace || workspace_bytes < p.bytes ||
      reinterpret_cast<uintptr_t>(workspace) % 16) {
    set_error("wm_balance_forward: null argument, or a small workspace (wm_router_workspace, 16-byte aligned)");
    return WM_ERR_INVALID;
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  Rows a = rows_of(*r, p);
  a.bias = nullptr;
  const Records rec = records_of(p, workspace, false);
  int* no_routes = nullptr;
  float* no_gates = nullptr;
  WM_ROUTER_DISPATCH(r->dtype, r->experts, forward_of, a, p, no_routes, no_gates, rec, stream);
  count_launch();
  WM_CUDA(cudaGetLastError());
  return finish(a, p, rec, counts, nullptr, table, workspace, loss, stream);
}

extern "C" int wm_router_backward(const wm_router* r, const int32_t* routes, const float* dgates, const float* table,
                                  const float* dloss, void* dlogits, void* stream_) {
  if (int rc = check_rows("wm_router_backward", r)) return rc;
  if (routes)
    if (int rc = check_choice("wm_router_backward", r)) return rc;
  if ((routes != nullptr) != (dgates != nullptr) || (table != nullptr) != (dloss != nullptr) || (!routes && !table) ||
      (r->tokens > 0 && !dlogits)) {
    set_error("wm_router_backward: routes go with dgates, table with dloss; one pair and dlogits are needed");
    return WM_ERR_INVALID;
  }
  if (r->tokens == 0) return WM_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const Rows a = rows_of(*r, plan_of(*r));
  WM_ROUTER_DISPATCH(r->dtype, r->experts, backward_of, a, routes, dgates, table, dloss, dlogits, stream);
  count_launch();
  WM_CUDA(cudaGetLastError());
  return WM_OK;
}

extern "C" int wm_expert_counts(const int32_t* routes, int32_t tokens, int32_t top_k, int32_t experts,
                                const int32_t* sequences, int32_t num_sequences, int32_t* counts, void* stream_) {
  if (tokens < 0 || top_k < 1 || top_k > 32 || experts < 1 || experts > kMaxExperts || !counts ||
      (tokens > 0 && !routes) || (sequences ? num_sequences < 1 : num_sequences != 0) || num_sequences > 65535) {
    set_error("wm_expert_counts: routes [tokens][1..32], 1..%d experts, 1..65535 sequences with their offsets",
              kMaxExperts);
    return WM_ERR_INVALID;
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int rows = sequences ? num_sequences : 1;
  WM_CUDA(cudaMemsetAsync(counts, 0, static_cast<size_t>(rows) * experts * 4, stream));
  if (tokens == 0) return WM_OK;
  const int want = (tokens + 127) / 128;
  const int blocks = want < 296 ? want : 296;
  Rows a{};
  a.tokens = tokens;
  a.experts = experts;
  a.top_k = top_k;
  a.sequences = sequences;
  a.num_sequences = rows;
  a.chunk = (tokens + blocks - 1) / blocks;
  expert_counts_kernel<<<(tokens + a.chunk - 1) / a.chunk, 256, experts * 4, stream>>>(a, routes, counts);
  count_launch();
  WM_CUDA(cudaGetLastError());
  return WM_OK;
}
