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
//
// What bounds it: instructions and their latency, not bytes.  A score costs an exponential, an addition and a reciprocal,
// the choice about as much again; 65536 rows of 512 BF16 logits (67 MB; 10 us at the copy rate) take 76 us for the choice by
// logits, 98 us by sigmoid + bias, 123 us with the loss on top.  Two thirds of the issue slots are taken; the other third is
// the wait for shuffles, shared memory and spilled registers, which 24 warps an SM do not cover.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include "../../include/weftmoe_b200.h"
#include "kernels.h"
#include "ptx.cuh"

using namespace wm;

namespace {

constexpr int kWarps = 8;
constexpr int kFinishWarps = 32;
constexpr int kMaxExperts = 1024;
constexpr int kMaxTokens = (1 << 26) - 1;   // x 32 routes: counts fit in 32 bits
// Records of the loss are one a block, so blocks are limited: 148 SMs x 8.  (512 experts have 444 places, so 2.6 rounds;
// other limits were not measured.)  A warp then adds the shares of up to tokens / 9472 rows one after another in FP32:
// 256 at 2.4 M tokens, 7086 at the most tokens there may be.
constexpr int kMaxBlocks = 1184;
constexpr int kFewChoices = 12;     // see choose
template <bool MANY>
constexpr int kCandidates = MANY ? 64 : 32;   // of one row, for its choice
constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void put(float& p, float v) { p = v; }
__device__ __forceinline__ void put(__nv_bfloat16& p, float v) { p = __float2bfloat16_rn(v); }  // the gradient's type
__device__ __forceinline__ void put(__half& p, float v) { p = __float2half_rn(v); }             // is the logits'

template <class F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
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
// The largest of the lanes' values, which holds no NaN.
__device__ __forceinline__ float warp_max(float v) { return unordered(__reduce_max_sync(kAll, ordered(v))); }
// The larger one; NaN if either is.
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 1 / y to one unit in the last place, for normal y below 2^126.
__device__ __forceinline__ float reciprocal(float y) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return r;
}
// 2^t by the exponent unit, two units in the last place; 0 at -inf and below 2^-126.
__device__ __forceinline__ float power_of_2(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
// Exponentials are powers of 2 of x log2 e.  exp(x - top) is 2^(x log2 e - c) with c the rounded top log2 e: the
// rounding of c, up to half a step of c in the exponent, is a factor that all terms of a row share and that their shares do
// not see as long as it stays in range.  Up to kFarTop it is at most 2^0.5; from 2^31 on it passes 2^127 and the row's sum
// would be infinite or 0.  Beyond kFarTop the difference is taken first: it is exact where it counts (logits within a
// factor of two of top; the others' terms vanish), and its product with log2 e rounds like the fused one.
constexpr float kLog2E = 1.44269504f;
constexpr float kFarTop = 8388608.0f;   // 2^23: top log2 e is below 2^24, a step of it is at most 1
__device__ __forceinline__ float exp_below(float x, float top) {
  return power_of_2(fabsf(top) < kFarTop ? fmaf(x, kLog2E, -top * kLog2E) : (x - top) * kLog2E);
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

// Which experts a lane holds: pieces of VEC neighbours, so that a row moves in accesses of VEC elements.
// Experts rise with the slot, which is what the order of ties relies on.
template <int VEC>
__device__ __forceinline__ int expert_of(int slot, int lane) {
  return slot / VEC * (32 * VEC) + lane * VEC + slot % VEC;
}
template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Piece {
  T v[VEC];
};
// A lane's part of a row as it is stored, so that the next row can be on its way while this one is worked on.
template <class T, int V, int VEC>
struct RowPieces {
  Piece<T, VEC> piece[V / VEC];
};
template <class T, int V, int VEC>
__device__ __forceinline__ void fetch_row(const Rows& a, long long row, int lane, RowPieces<T, V, VEC>& r) {
  const T* p = static_cast<const T*>(a.logits) + row * a.stride;
#pragma unroll
  for (int j = 0; j < V / VEC; ++j) {
    const int e = expert_of<VEC>(j * VEC, lane);   // experts % VEC == 0: a piece is whole or absent
    if (e < a.experts) r.piece[j] = *reinterpret_cast<const Piece<T, VEC>*>(p + e);
  }
}
template <class T, int V, int VEC>
__device__ __forceinline__ void unpack_row(const Rows& a, int lane, const RowPieces<T, V, VEC>& r, float (&x)[V]) {
#pragma unroll
  for (int j = 0; j < V / VEC; ++j) {
    const bool there = expert_of<VEC>(j * VEC, lane) < a.experts;
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[j * VEC + i] = there ? as_float(r.piece[j].v[i]) : -INFINITY;
  }
}
template <class T, int V, int VEC>
__device__ __forceinline__ void store_row(T* out, int experts, int lane, const float (&d)[V]) {
#pragma unroll
  for (int j = 0; j < V; j += VEC) {
    const int e = expert_of<VEC>(j, lane);
    if (e < experts) {
      Piece<T, VEC> w;
#pragma unroll
      for (int i = 0; i < VEC; ++i) put(w.v[i], d[j + i]);
      *reinterpret_cast<Piece<T, VEC>*>(out + e) = w;
    }
  }
}

// s = 1 / (1 + E) with E = exp(-x), and its complement E s, neither of which cancels.  Below x = -87, where s is no
// normal number, both are 0.
__device__ __forceinline__ float sigmoid_of(float x, float& rest) {
  const float e = power_of_2(fminf(-x * kLog2E, 127.5f));
  const float s = reciprocal(1.0f + e);
  rest = e * s;
  return s;
}
// s(x) * exp(-min(top, 0)), for shares of a row whose largest logit `top` is so low that its sigmoids vanish.
__device__ __forceinline__ float sigmoid_far(float x, float top) {
  return expf(fminf(x, 0.0f) - fminf(top, 0.0f)) / (1.0f + expf(-fabsf(x)));
}
constexpr float kFar = -60.0f;   // sigmoids of a row with a logit above this are normal numbers

// Of a row: its largest logit, whether an expert is available, and whether it has no distribution (NaN, or for
// softmax +inf, among its logits).
struct RowTop {
  float top, lane_top;   // of the row, of this lane's part of it
  bool bad, any;
};
template <int V>
__device__ __forceinline__ RowTop row_top(const float (&x)[V], bool sigmoid) {
  RowTop r;
  float top = x[0];
#pragma unroll
  for (int j = 1; j < V; ++j) top = max_or_nan(top, x[j]);
  r.lane_top = top;
  r.bad = __any_sync(kAll, top != top);
  r.top = r.bad ? 0.0f : warp_max(top);
  r.bad |= !sigmoid && r.top == INFINITY;
  r.any = r.top > -INFINITY;
  return r;
}
// h[j] such that h / sum is the row's share: exp(x - top), or the sigmoid (with its complement in rest).
// Returns the sum over the row; the row has an available expert.
template <int V>
__device__ __forceinline__ float row_shares(const float (&x)[V], bool sigmoid, float top, float (&h)[V],
                                            float (&rest)[V]) {
  float sum = 0.0f;
  if (!sigmoid) {
    const float c = top * kLog2E;
    if (fabsf(top) < kFarTop) {
#pragma unroll
      for (int j = 0; j < V; ++j) { h[j] = power_of_2(fmaf(x[j], kLog2E, -c)); sum += h[j]; }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) { h[j] = exp_below(x[j], top); sum += h[j]; }
    }
  } else if (top > kFar) {
#pragma unroll
    for (int j = 0; j < V; ++j) { h[j] = sigmoid_of(x[j], rest[j]); sum += h[j]; }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) { h[j] = sigmoid_far(x[j], top); rest[j] = 1.0f; sum += h[j]; }
  }
  return warp_sum(sum);
}

// The choice of one row from memory, in K rounds over all experts, by 64-bit scores: for rows with too many candidates
// (some 64 equal values).  Out of line and without arrays it costs the other rows no registers.
template <class T>
__device__ __noinline__ int choose_slowly(const T* logits, int experts, int top_k, const float* bias, bool sigmoid,
                                          float top, int lane) {
  double sum = 1.0;
  if (bias != nullptr && !sigmoid) {
    sum = 0.0;
    for (int e = lane; e < experts; e += 32) sum += exp(static_cast<double>(as_float(logits[e])) - top);
    sum = warp_sum(sum);
  }
  unsigned long long last = ~0ull;   // the order so far ends at (last, last_expert)
  int last_expert = -1, expert = -1;
  for (int k = 0; k < top_k; ++k) {
    unsigned long long best = 0;
    int at = 0x7fffffff;
    for (int e = lane; e < experts; e += 32) {
      const double x = as_float(logits[e]);
      if (!(x > -INFINITY)) continue;
      double v = x;
      if (bias != nullptr) v = (sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - top) / sum) + static_cast<double>(__ldg(bias + e));
      const unsigned long long key = ordered(v);
      if ((key < last || (key == last && e > last_expert)) && key > best) { best = key; at = e; }
    }
    const unsigned high = static_cast<unsigned>(best >> 32), low = static_cast<unsigned>(best);
    const unsigned most_high = __reduce_max_sync(kAll, high);
    if (most_high == 0) break;
    const unsigned most_low = __reduce_max_sync(kAll, high == most_high ? low : 0u);
    last_expert = __reduce_min_sync(kAll, high == most_high && low == most_low ? static_cast<unsigned>(at) : 0x7fffffffu);
    last = static_cast<unsigned long long>(most_high) << 32 | most_low;
    if (lane == k) expert = last_expert;
  }
  return expert;
}

// The n <= kCandidates candidates in `held` (any order), ranked by their 64-bit scores; lane k gets choice k.  A lane takes
// one candidate, or two for MANY, so this costs as many exponentials in 64 bits (and for softmax the row's sum).
template <bool MANY, class T>
__device__ __noinline__ int rank_in_64(const T* logits, int experts, int top_k, const float* bias, bool sigmoid,
                                       float top, int lane, float2* held, int n) {
  double sum = 1.0;
  if (!sigmoid) {
    sum = 0.0;
#pragma unroll 4
    for (int e = lane; e < experts; e += 32) sum += exp(static_cast<double>(as_float(logits[e])) - top);
    sum = warp_sum(sum);
  }
  constexpr int kEach = MANY ? 2 : 1;
  int expert[kEach], before[kEach];
  double v[kEach];
#pragma unroll
  for (int c = 0; c < kEach; ++c) {
    expert[c] = 0x7fffffff;
    before[c] = 0;
    v[c] = -INFINITY;
    if (lane + 32 * c >= n) continue;
    expert[c] = __float_as_int(held[lane + 32 * c].y);
    const double x = as_float(logits[expert[c]]);
    v[c] = (sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - top) / sum) + static_cast<double>(__ldg(bias + expert[c]));
  }
  for (int i = 0; i < n; ++i) {
    const double w = __shfl_sync(kAll, i < 32 ? v[0] : v[kEach - 1], i & 31);
    const int e = __shfl_sync(kAll, i < 32 ? expert[0] : expert[kEach - 1], i & 31);
#pragma unroll
    for (int c = 0; c < kEach; ++c) before[c] += w > v[c] || (w == v[c] && e < expert[c]);
  }
  __syncwarp();
#pragma unroll
  for (int c = 0; c < kEach; ++c)
    if (lane + 32 * c < n) held[before[c]].y = __int_as_float(expert[c]);
  __syncwarp();
  const int chosen = lane < min(n, top_k) ? __float_as_int(held[lane].y) : -1;
  __syncwarp();
  return chosen;
}

// How many of the first n candidates (n rounded up to four; those behind are last) come before this one.
__device__ __forceinline__ int before_of(const float2& me, const float2* held, int n) {
  int before = 0;
  for (int i = 0; i < n; i += 4) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float2 other = held[i + w];
      before += other.x > me.x || (other.x == me.x && __float_as_int(other.y) < __float_as_int(me.y));
    }
  }
  return before;
}
template <int V>
__device__ __forceinline__ int count_from(const float (&x)[V], float from) {
  int mine = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) mine += x[j] >= from;
  return __reduce_add_sync(kAll, mine);
}
// A higher border for a row with more than 64 values from `border` up: one with more than top_k of them, and
// few enough, by halving the words between it and `top`.  Unchanged where equal values leave none.
template <int V>
__device__ __forceinline__ float closer_border(const float (&x)[V], float border, float top, int top_k) {
  unsigned low = ordered(border), high = ordered(top) + 1;
  while (high - low > 1) {
    const unsigned middle = low + (high - low) / 2;
    const int n = count_from<V>(x, unordered(middle));
    if (n <= top_k) high = middle;
    else if (n > kCandidates<true> - 4) low = middle;   // a few places are left for the margin
    else return unordered(middle);
  }
  return border;
}

// The K largest (value, lowest expert first) of the warp's V x 32 values, `most` the lane's largest; -inf is no
// candidate.  The (K+1)th largest of the lanes' maxima is at most the (K+1)th largest value, so the values from it up
// hold the choice and the one behind it; they are few (for unequal values K + 1 and a few lanes' second ones).  They,
// and with a margin what is at most so much smaller, are gathered in `held` (kCandidates of this warp), and each counts
// the ones before it.  Lane k gets choice k and its value; `behind` the next value (-inf: none).  Returns the number of
// candidates, which stay in `held` in their order; above kCandidates (many equal values) nothing is chosen.
// MANY: for K above kFewChoices the border of 32 lanes leaves more candidates (24 on average at K = 16, all values at
// K = 32): room for 64, two a lane, and a border moved up by halving.  65536 x 512 BF16 by logits, with / without: K = 8
// 80 / 76 us, K = 16 116 / 329, K = 32 202 / 1959; up to 12 the 32 places overflow in less than one row of 10000.
template <bool MANY, int V, int VEC>
__device__ __forceinline__ int choose(const float (&x)[V], float most, float margin, int top_k, int lane, float2* held,
                                      int& expert, float& its, float& behind) {
  unsigned key = most > -INFINITY ? ordered(most) : 0u, top = 0, border = 0;
  for (int k = 0; k <= top_k; ++k) {   // equal maxima go at once: the border is then lower, which is as good
    const unsigned next = __reduce_max_sync(kAll, key);
    if (k == 0) top = next;
    if (next == 0) {   // fewer lanes: the least of their maxima may do, or else all values
      if (!MANY || (border != 0 && count_from<V>(x, unordered(border)) <= top_k)) border = 0;
      break;
    }
    border = next;
    if (key == next) key = 0;
  }
  float from = -FLT_MAX;
  if (border != 0) from = fmaxf(from, unordered(border) - margin * (1.0f + fabsf(unordered(border))));   // never -inf
  int mine = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) mine += x[j] >= from;
  int n = 0;
  if constexpr (MANY) n = __reduce_add_sync(kAll, mine);
  if (MANY && n > kCandidates<true>) {
    const float closer = closer_border<V>(x, from, unordered(top), top_k);
    from = fmaxf(from, closer - margin * (1.0f + fabsf(closer)));
    mine = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) mine += x[j] >= from;
    n = __reduce_add_sync(kAll, mine);
    if (n > kCandidates<true>) return n;
  }
  // places: lanes before this one with at least 1, 2, ... candidates
  int at = 0;
  const unsigned before_me = (1u << lane) - 1;
  for (int c = 1;; ++c) {
    const unsigned lanes = __ballot_sync(kAll, mine >= c);
    if (lanes == 0) break;
    at += __popc(lanes & before_me);
    if (!MANY) n += __popc(lanes);
  }
  if (!MANY && n > kCandidates<false>) return n;
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (x[j] >= from) held[at++] = make_float2(x[j], __int_as_float(expert_of<VEC>(j, lane)));
  __syncwarp();
  const float2 last = make_float2(-INFINITY, __int_as_float(0x7fffffff));   // ranks behind all candidates
  if (lane >= n) held[lane] = last;
  if (MANY && n > 32 && lane + 32 >= n) held[lane + 32] = last;
  __syncwarp();
  const float2 me = held[lane];
  const int before = before_of(me, held, n);
  if (MANY && n > 32) {
    const float2 other = held[lane + 32];
    const int before_other = before_of(other, held, n);
    __syncwarp();
    if (lane + 32 < n) held[before_other] = other;
  }
  __syncwarp();
  if (lane < n) held[before] = me;
  __syncwarp();
  expert = -1;
  its = -INFINITY;
  if (lane < min(n, top_k)) {
    const float2 w = held[lane];
    its = w.x;
    expert = __float_as_int(w.y);
  }
  behind = n > top_k ? held[top_k].x : -INFINITY;
  __syncwarp();
  return n;
}

// (A border guessed from the warp's last row instead of the reductions, with the candidates' values worked out again
// from memory, ran fewer instructions and took 7 % longer: more of them wait for one another.)
// The choice by s + bias.  In 32 bits v = s + bias is off by less than doubt * (1 + |v|): a sigmoid by 9 half units
// (exponential 4, addition 1, reciprocal 2, product 1, and the residual), a softmax by 46 (0.37 for the difference,
// exponential 4, 37 additions, reciprocal and product), and v by its own rounding.  Where two neighbours of the
// order, or the last choice and the one behind it, are nearer than twice that, 64 bits decide among the candidates
// (0.3 % of rows for sigmoids of 512 experts).  Experts of equal logit and equal bias have equal scores and need no more
// digits.  False: too many candidates, nothing is chosen.
template <bool MANY, class T, int V, int VEC>
__device__ __forceinline__ bool choose_by_score(const float (&x)[V], const float (&h)[V], float sum, const Rows& a,
                                                const T* logits, float top, int lane, float2* held, int& expert) {
  const float doubt = a.sigmoid ? 1e-6f : 4e-6f;
  float v[V];
  const float inv = a.sigmoid ? 1.0f : reciprocal(sum);
#pragma unroll
  for (int j = 0; j < V; j += VEC) {
    const int e = expert_of<VEC>(j, lane);
    const bool there = e < a.experts;
#pragma unroll
    for (int i = 0; i < VEC; i += VEC % 4 == 0 ? 4 : 1) {
      float bias[4] = {};
      if (there) {
        if constexpr (VEC % 4 == 0) *reinterpret_cast<float4*>(bias) = __ldg(reinterpret_cast<const float4*>(a.bias + e + i));
        else bias[0] = __ldg(a.bias + e + i);
      }
#pragma unroll
      for (int w = 0; w < (VEC % 4 == 0 ? 4 : 1); ++w) {
        const int at = j + i + w;
        const float s = a.sigmoid && top <= kFar ? 0.0f : h[at] * inv;   // sigmoids of such a row are below 1e-26
        v[at] = x[at] > -INFINITY ? s + bias[w] : -INFINITY;
      }
    }
  }
  float mine, behind;
  float most = v[0];
#pragma unroll
  for (int j = 1; j < V; ++j) most = fmaxf(most, v[j]);
  const int n = choose<MANY, V, VEC>(v, most, 2.0f * doubt, a.top_k, lane, held, expert, mine, behind);
  if (n > kCandidates<MANY>) return false;
  float next = __shfl_down_sync(kAll, mine, 1);
  int next_expert = __shfl_down_sync(kAll, expert, 1);
  if (lane >= a.top_k - 1) { next = behind; next_expert = -1; }
  bool doubtful = false;
  if (expert >= 0 && next > -INFINITY && !(mine - next > 2.0f * doubt * (1.0f + fabsf(mine)))) {
    doubtful = true;
    if (next_expert >= 0)
      doubtful = as_float(logits[expert]) != as_float(logits[next_expert]) ||
                 __ldg(a.bias + expert) != __ldg(a.bias + next_expert);
  }
  if (__any_sync(kAll, doubtful))
    expert = rank_in_64<MANY, T>(logits, a.experts, a.top_k, a.bias, a.sigmoid != 0, top, lane, held, n);
  return true;
}

// Lane k: choice k's weight (its gate without the scale).  top and sum belong to the whole row; sum is that of
// exp(x - top) and is used by softmax without renormalisation alone.
__device__ __forceinline__ float choice_weight(const Rows& a, float top, float sum, int expert, float logit) {
  const bool chosen = expert >= 0;
  float rest;
  if (a.renormalize) {
    const float most = warp_max(chosen ? logit : -INFINITY);
    float h = 0.0f;
    if (chosen) h = !a.sigmoid ? exp_below(logit, most) : most > kFar ? sigmoid_of(logit, rest) : sigmoid_far(logit, most);
    const float all = warp_sum(h);
    return chosen ? h / all : 0.0f;
  }
  if (!chosen) return 0.0f;
  return a.sigmoid ? sigmoid_of(logit, rest) : exp_below(logit, top) / sum;
}

// Records of the balance sums: record (chunk c, sequence b) is number c + b.  Chunks and sequences both walk the
// rows in order, so c + b names each pair that meets once.
struct Records {
  float* share;   // [records][experts] sum of p
  int* counts;    // [records][experts], null without a choice
  int* rows;      // [records][2] live rows, routes
  unsigned* ticket;
};

// Blocks of an SM that the registers are shared out for.  Forward and backward of 65536 rows of 512 BF16 experts took 211 us
// with 3 blocks, 213 us with 2 for the backward kernel, 18 us more with 4; the other sizes were not measured.  Limits
// of 64 and 80 registers spill.  Forward kernels, bytes of spill stores a thread with vector loads and up to 12 choices,
// BF16 / FP32: 32 experts 60 / 60, 64: 88 / 112, 128: 116 / 156, 256: 216 / 178, 512: 104 / 316, 1024: none.  Backward
// kernels: 256 experts 0 / 8, 512: 112 / 168, the others none.
template <int V>
constexpr int kResident = V <= 8 ? 4 : V <= 16 ? 3 : 1;

// A warp per row, its logits and then its scores in registers: one read of the logits, one exponential a score.  A block
// walks its chunk of rows with eight warps and the next row on its way; with the loss each warp adds its rows' p in its own
// part of shared memory (experts slots, no atomics), and counts go through shared whole-number atomics.
template <class T, int V, int VEC, bool MANY>
__global__ void __launch_bounds__(kWarps * 32, kResident<V>)
router_forward_kernel(const Rows a, int* __restrict__ routes, float* __restrict__ gates, const Records rec) {
  extern __shared__ float4 smem_sums[];                            // (16-byte aligned)
  float* part = reinterpret_cast<float*>(smem_sums);               // [kWarps][experts], each warp's sums of p
  float* mine = part + (threadIdx.x >> 5) * a.experts;
  int* seen = reinterpret_cast<int*>(part + kWarps * a.experts);   // [experts]
  __shared__ int live_rows[kWarps], live_routes[kWarps];
  __shared__ float2 held[kWarps][kCandidates<MANY>];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool balance = rec.share != nullptr, pick = routes != nullptr;
  const bool whole = balance || a.bias != nullptr || (!a.renormalize && !a.sigmoid);   // scores of all experts
  if (balance) {
    cudaTriggerProgrammaticLaunchCompletion();   // the kernel that sums the records may take its place; it waits for these
    if (blockIdx.x == 0 && threadIdx.x == 0) *rec.ticket = 0;
  }
  const int first = blockIdx.x * a.chunk, last = min(first + a.chunk, a.tokens);
  if (balance) {
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) seen[e] = 0;
    __syncthreads();
  }

  int row0 = first;
  while (row0 < last) {
    const int b = sequence_of(a, row0);
    const int row1 = balance ? max(row0 + 1, min(last, sequence_end(a, b))) : last;
    if (balance) {
#pragma unroll
      for (int j = 0; j < V; j += VEC) {
        const int e = expert_of<VEC>(j, lane);
        if (e < a.experts) *reinterpret_cast<Piece<float, VEC>*>(mine + e) = Piece<float, VEC>{};
      }
    }
    int rows = 0, taken = 0;
    RowPieces<T, V, VEC> next;
    if (row0 + warp < row1) fetch_row<T, V, VEC>(a, row0 + warp, lane, next);
    for (int row = row0 + warp; row < row1; row += kWarps) {
      const RowPieces<T, V, VEC> here = next;
      if (row + kWarps < row1) fetch_row<T, V, VEC>(a, row + kWarps, lane, next);
      int expert = -1;
      float weight = 0.0f;
      if (row_live(a, row, balance ? b : sequence_of(a, row))) {
        float x[V], h[V], rest[V];
        unpack_row<T, V, VEC>(a, lane, here, x);
        const RowTop r = row_top<V>(x, a.sigmoid);
        float sum = 1.0f;
        if (whole && r.any && !r.bad) sum = row_shares<V>(x, a.sigmoid, r.top, h, rest);
        if (balance && (r.any || r.bad)) {
          ++rows;
          const float inv = 1.0f / sum;
#pragma unroll
          for (int j = 0; j < V; j += VEC) {
            const int e = expert_of<VEC>(j, lane);
            if (e < a.experts) {
              Piece<float, VEC>& w = *reinterpret_cast<Piece<float, VEC>*>(mine + e);
              Piece<float, VEC> acc = w;
#pragma unroll
              for (int i = 0; i < VEC; ++i) acc.v[i] = r.bad ? NAN : fmaf(h[j + i], inv, acc.v[i]);
              w = acc;
            }
          }
        }
        if (pick && r.bad) {   // no distribution: valid routes and NaN gates, so that it shows in the output
          expert = lane < a.top_k ? lane : -1;
          weight = NAN;
        } else if (pick && r.any) {
          const T* logits = static_cast<const T*>(a.logits) + static_cast<long long>(row) * a.stride;
          float logit = 0.0f, behind;
          bool settled;
          if (a.bias != nullptr) {
            settled = choose_by_score<MANY, T, V, VEC>(x, h, sum, a, logits, r.top, lane, held[warp], expert);
            if (settled && expert >= 0) logit = as_float(logits[expert]);
          } else {
            settled = choose<MANY, V, VEC>(x, r.lane_top, 0.0f, a.top_k, lane, held[warp], expert, logit, behind) <=
                      kCandidates<MANY>;
          }
          if (!settled) {
            expert = choose_slowly<T>(logits, a.experts, a.top_k, a.bias, a.sigmoid != 0, r.top, lane);
            if (expert >= 0) logit = as_float(logits[expert]);
          }
          weight = choice_weight(a, r.top, sum, expert, logit);
        }
        if (balance && pick && expert >= 0) { atomicAdd(seen + expert, 1); ++taken; }
      }
      if (pick && lane < a.top_k) {
        routes[static_cast<long long>(row) * a.top_k + lane] = expert;
        gates[static_cast<long long>(row) * a.top_k + lane] = expert >= 0 ? a.scale * weight : 0.0f;
      }
    }
    if (balance) {
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
          if (pick) { rec.counts[record * a.experts + e] = seen[e]; seen[e] = 0; }
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

// Sums the records of one sequence for 32 experts per block (32 warps take every 32nd record), then the last
// block to finish sums the blocks' parts of the loss in their order.  Bound by latency: 13 us for 1171 + 16 records of
// 512 experts (4.9 MB), a chain of loads, sums and the last block's join.
// table: [num_sequences][experts] of (f - 1) / n_b, the loss's slope by p up to a constant (p sums to one, so a
// constant drops out of the gradient; without it, taken off before f is rounded, the differences near f = 1 keep their
// digits), then 1 / live sequences.
__global__ void __launch_bounds__(kFinishWarps * 32)
balance_finish_kernel(const Rows a, const Records rec, const int* __restrict__ given, int* __restrict__ counts,
                      float* __restrict__ table, float* parts, float* __restrict__ loss) {
  __shared__ float share[kFinishWarps][32];
  __shared__ int count[kFinishWarps][32];
  __shared__ int rows[kFinishWarps], taken[kFinishWarps];
  __shared__ long long given_sum[kFinishWarps];
  __shared__ bool is_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.y, e = blockIdx.x * 32 + lane;
  cudaGridDependencySynchronize();   // launched while the kernel that writes the records still runs
  const int row0 = a.sequences == nullptr ? 0 : max(0, __ldg(a.sequences + b));
  const int row1 = sequence_end(a, b);
  float sum = 0.0f;
  int c = 0, n = 0, total = 0;
  if (row0 < row1) {
    const int end = (row1 - 1) / a.chunk;
    if (e < a.experts) {
#pragma unroll 8
      for (int chunk = row0 / a.chunk + warp; chunk <= end; chunk += kFinishWarps) {
        const long long at = static_cast<long long>(chunk + b) * a.experts + e;
        sum += rec.share[at];
        if (rec.counts != nullptr) c += rec.counts[at];
      }
    }
    for (int chunk = row0 / a.chunk + threadIdx.x; chunk <= end; chunk += blockDim.x) {
      n += rec.rows[2 * static_cast<long long>(chunk + b)];
      total += rec.rows[2 * static_cast<long long>(chunk + b) + 1];
    }
  }
  long long all = 0;
  if (given != nullptr)
    for (int i = threadIdx.x; i < a.experts; i += blockDim.x) all += given[static_cast<long long>(b) * a.experts + i];
  share[warp][lane] = sum;
  count[warp][lane] = c;
  n = __reduce_add_sync(kAll, n);
  total = __reduce_add_sync(kAll, total);
  all = warp_sum(all);
  if (lane == 0) { rows[warp] = n; taken[warp] = total; given_sum[warp] = all; }
  __syncthreads();
  if (warp == 0) {
    sum = 0.0f;
    c = 0;
#pragma unroll
    for (int w = 0; w < kFinishWarps; ++w) { sum += share[w][lane]; c += count[w][lane]; }
    n = __reduce_add_sync(kAll, rows[lane]);
    all = warp_sum(given != nullptr ? given_sum[lane] : static_cast<long long>(taken[lane]));
    if (given != nullptr) c = e < a.experts ? given[static_cast<long long>(b) * a.experts + e] : 0;
    float part = 0.0f;
    if (e < a.experts) {
      const double f = all > 0 ? static_cast<double>(c) * a.experts / static_cast<double>(all) : 0.0;
      const float inv = n > 0 ? 1.0f / static_cast<float>(n) : 0.0f;
      part = n > 0 ? static_cast<float>(f) * (sum / static_cast<float>(n)) : 0.0f;
      table[static_cast<long long>(b) * a.experts + e] = static_cast<float>(f - 1.0) * inv;
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
  __shared__ double sums[kFinishWarps], lives[kFinishWarps];
  double l = 0.0, live = 0.0;
  const long long blocks = static_cast<long long>(gridDim.x) * gridDim.y;
  for (long long i = threadIdx.x; i < blocks; i += blockDim.x) { l += __ldcg(parts + 2 * i); live += __ldcg(parts + 2 * i + 1); }
  l = warp_sum(l);
  live = warp_sum(live);
  if (lane == 0) { sums[warp] = l; lives[warp] = live; }
  __syncthreads();
  if (warp == 0) {
    l = warp_sum(sums[lane]);
    live = warp_sum(lives[lane]);
    if (lane == 0) {
      const double inv = live > 0.0 ? 1.0 / live : 0.0;
      *loss = static_cast<float>(live > 0.0 ? l * inv : 0.0);
      table[static_cast<long long>(a.num_sequences) * a.experts] = static_cast<float>(inv);
    }
  }
}

// d logits of one row per warp:
//   gates, w = the choice's weight, g = scale * dgate:
//     softmax, renormalised  w_k (g_k - sum w g) at the chosen      softmax  s_e ([chosen] g_e - sum s g)
//     sigmoid, renormalised  (1 - s_k) w_k (g_k - sum w g)           sigmoid  (1 - s_k) s_k g_k
//   loss, q = the table's row times dloss / live sequences:  p_e (q_e - sum p q), times 1 - s_e for sigmoid.
// The choices' part goes through a row of shared memory that is zero between rows.  A warp takes a.chunk rows in a row, and
// fetches the next one's logits, routes and dgates ahead.  Bound by instructions and their latency (62 % of the issue slots
// taken): 85 us under ncu for 65536 rows of 512 BF16 logits, 134 MB in and out, which a copy moves in 20 us.
template <class T, int V, int VEC>
__global__ void __launch_bounds__(kWarps * 32, kResident<V>)
router_backward_kernel(const Rows a, const int* __restrict__ routes, const float* __restrict__ dgates,
                       const float* __restrict__ table, const float* __restrict__ dloss, T* __restrict__ dlogits) {
  extern __shared__ float4 smem_rows[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* chosen = reinterpret_cast<float*>(smem_rows) + warp * (V * 32);
  const float push = table != nullptr
      ? __ldg(dloss) * __ldg(table + static_cast<long long>(a.num_sequences) * a.experts) : 0.0f;
  const bool shares = table != nullptr || (!a.renormalize && !a.sigmoid);
  if (routes != nullptr) {
#pragma unroll
    for (int j = 0; j < V; ++j) chosen[j * 32 + lane] = 0.0f;
    __syncwarp();
  }
  const long long from = (static_cast<long long>(blockIdx.x) * kWarps + warp) * a.chunk;
  const int end = static_cast<int>(min(from + a.chunk, static_cast<long long>(a.tokens)));
  int b = 0, b_end = -1;
  RowPieces<T, V, VEC> next;
  int next_expert = -1;
  float next_g = 0.0f;
  const auto fetch_choice = [&](int row) {
    if (routes == nullptr || lane >= a.top_k) return;
    const long long at = static_cast<long long>(row) * a.top_k + lane;
    next_expert = routes[at];
    next_g = dgates[at];
  };
  if (from < end) {
    fetch_row<T, V, VEC>(a, from, lane, next);
    fetch_choice(static_cast<int>(from));
  }
  for (int row = static_cast<int>(min(from, static_cast<long long>(a.tokens))); row < end; ++row) {
    if (row >= b_end) {
      b = sequence_of(a, row);
      b_end = max(row + 1, sequence_end(a, b));
    }
    const RowPieces<T, V, VEC> here = next;
    int expert = next_expert;
    float g = a.scale * next_g;
    if (row + 1 < end) {
      fetch_row<T, V, VEC>(a, row + 1, lane, next);
      fetch_choice(row + 1);
    }
    float d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = 0.0f;
    if (row_live(a, row, b)) {
      float logit = 0.0f;
      if (static_cast<unsigned>(expert) >= static_cast<unsigned>(a.experts)) expert = -1;
      if (expert >= 0) logit = as_float((static_cast<const T*>(a.logits) + static_cast<long long>(row) * a.stride)[expert]);
      float x[V], h[V], rest[V];
      unpack_row<T, V, VEC>(a, lane, here, x);
      const RowTop r = row_top<V>(x, a.sigmoid);
      if (r.bad) {
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = NAN;
      } else if (r.any) {
        float sum = 1.0f;
        if (shares) sum = row_shares<V>(x, a.sigmoid, r.top, h, rest);
        const float inv = reciprocal(sum);
        if (table != nullptr) {
          const float* q = table + static_cast<long long>(b) * a.experts;
          float mean = 0.0f;
          constexpr int kWide = VEC % 4 == 0 ? 4 : 1;   // then experts % 4 == 0, and every row of the table is aligned
#pragma unroll
          for (int j = 0; j < V; j += kWide) {
            const int e = expert_of<VEC>(j, lane);
            Piece<float, kWide> w{};
            if (e < a.experts) w = *reinterpret_cast<const Piece<float, kWide>*>(q + e);
#pragma unroll
            for (int i = 0; i < kWide; ++i) {
              d[j + i] = w.v[i];
              mean = fmaf(h[j + i], w.v[i], mean);
            }
          }
          mean = warp_sum(mean) * inv;
          const float factor = push * inv;
#pragma unroll
          for (int j = 0; j < V; ++j) d[j] = (factor * (a.sigmoid ? h[j] * rest[j] : h[j])) * (d[j] - mean);
        }
        if (routes != nullptr) {
          const float w = choice_weight(a, r.top, sum, expert, logit);
          float mean = 0.0f;
          if (a.renormalize || !a.sigmoid) mean = warp_sum(w * g);
          float c = w * (a.renormalize ? g - mean : g);
          if (a.sigmoid) {
            float rest_k;
            sigmoid_of(logit, rest_k);
            c *= logit > kFar ? rest_k : 1.0f;
          }
          if (!a.renormalize && !a.sigmoid) {
#pragma unroll
            for (int j = 0; j < V; ++j) d[j] = fmaf(h[j], -mean * inv, d[j]);
          }
          if (expert >= 0) chosen[expert] = c;
          __syncwarp();
#pragma unroll
          for (int j = 0; j < V; j += VEC) {
            const Piece<float, VEC> piece = *reinterpret_cast<const Piece<float, VEC>*>(chosen + expert_of<VEC>(j, lane));
#pragma unroll
            for (int i = 0; i < VEC; ++i) d[j + i] += piece.v[i];
          }
          __syncwarp();
          if (expert >= 0) chosen[expert] = 0.0f;
          __syncwarp();
        }
      }
    }
    store_row<T, V, VEC>(dlogits + static_cast<long long>(row) * a.experts, a.experts, lane, d);
  }
}

// Routes per expert of one sequence by a cluster of eight CTAs: each counts an eighth of the rows in its shared memory,
// and the first sums each expert over all eight, a thread an expert.  Nothing has to be cleared before, so it is one
// launch: 3.5 us for 8192 x 8 routes to 256 experts, which is little more than a launch.
constexpr int kCountCtas = 8;
__global__ void __cluster_dims__(kCountCtas, 1, 1) __launch_bounds__(kMaxExperts)
expert_counts_cluster_kernel(const Rows a, const int* __restrict__ routes, int* __restrict__ counts) {
  extern __shared__ int cluster_counts[];
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) cluster_counts[e] = 0;
  __syncthreads();
  const int b = blockIdx.y, part = blockIdx.x;
  const int row0 = a.sequences == nullptr ? 0 : max(0, __ldg(a.sequences + b));
  const long long rows = max(0, sequence_end(a, b) - row0);
  const long long first = (row0 + rows * part / kCountCtas) * a.top_k;
  const long long last = (row0 + rows * (part + 1) / kCountCtas) * a.top_k;
  for (long long i = first + threadIdx.x; i < last; i += blockDim.x) {
    const int e = routes[i];
    if (static_cast<unsigned>(e) < static_cast<unsigned>(a.experts)) atomicAdd(cluster_counts + e, 1);
  }
  cluster_sync_all();
  const int e = threadIdx.x;
  if (part == 0 && e < a.experts) {
    const uint32_t at = smem_u32(cluster_counts + e);
    int c = 0;
#pragma unroll
    for (int s = 0; s < kCountCtas; ++s) {
      int v;
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(map_to_cta(at, s)) : "memory");
      c += v;
    }
    counts[static_cast<long long>(b) * a.experts + e] = c;
  }
  cluster_sync_all();   // the others' shared memory stays until it is read
}

// For many routes, or many sequences: a block counts its rows in shared memory and adds the whole numbers to the
// (cleared) result.
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
// Up to here one cluster a sequence is the quicker form of the counts (one launch instead of a clear and a launch).
constexpr int kClusterSequences = 32;
constexpr long long kClusterRoutes = 131072;

struct Plan {
  int chunk, blocks;
  long long records, parts;
  long long share, counts, rows, part, ticket, bytes;   // offsets into the workspace
};

Plan plan_of(const wm_router& r) {
  Plan p{};
  const int sequences = r.sequences ? r.num_sequences : 1;
  // Two rows a warp where that still gives every SM two blocks: fewer records for the kernel behind this one.
  const int want = r.tokens >= 2 * 296 * kWarps ? (r.tokens + 2 * kWarps - 1) / (2 * kWarps) : (r.tokens + kWarps - 1) / kWarps;
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

// Addresses that are multiples of `bytes` (null is one).
template <class... P>
bool aligned(uintptr_t bytes, P... p) {
  return ((reinterpret_cast<uintptr_t>(p) | ...) & (bytes - 1)) == 0;
}

int check_rows(const char* what, const wm_router* r) {
  if (!r) { set_error("%s: null arguments", what); return WM_ERR_INVALID; }
  if (r->tokens < 0 || r->tokens > kMaxTokens || r->experts < 1 || r->experts > kMaxExperts || r->dtype < 0 || r->dtype > 2 ||
      r->row_stride < r->experts || (r->score != 0 && r->score != 1) || (r->tokens > 0 && !r->logits) ||
      (r->sequences ? r->num_sequences < 1 : r->num_sequences != 0) || r->num_sequences > 65535) {
    set_error("%s: logits must be [fewer than 2^26 tokens][experts] BF16 / FP32 / FP16 rows of 1..%d experts, score 0 (softmax) "
              "or 1 (sigmoid), 1..65535 sequences with their offsets", what, kMaxExperts);
    return WM_ERR_INVALID;
  }
  if (!aligned(r->dtype == 1 ? 4 : 2, r->logits) || !aligned(4, r->bias, r->sequences)) {
    set_error("%s: logits, bias or sequences not aligned to their elements", what);
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

template <class T, int V, int VEC>
void forward_of(const Rows& a, const Plan& p, int* routes, float* gates, const Records& rec, cudaStream_t stream) {
  const int smem = rec.share ? (kWarps + 1) * a.experts * 4 : 0;
  // one lane's worth of experts: every value is a lane's maximum
  const bool many = V > 1 && routes != nullptr && a.top_k > kFewChoices;
  auto kernel = many ? router_forward_kernel<T, V, VEC, (V > 1)> : router_forward_kernel<T, V, VEC, false>;
  kernel<<<p.blocks, kWarps * 32, smem, stream>>>(a, routes, gates, rec);
}
template <class T, int V, int VEC>
void backward_of(const Rows& a, const int* routes, const float* dgates, const float* table, const float* dloss,
                 void* dlogits, cudaStream_t stream) {
  Rows rows = a;
  const int most = 2 * 148 * 3 * kWarps;   // warps: two rounds of what the SMs hold
  rows.chunk = (a.tokens + most - 1) / most;
  const int blocks = (a.tokens + rows.chunk * kWarps - 1) / (rows.chunk * kWarps);
  const int smem = routes ? kWarps * V * 32 * 4 : 0;
  router_backward_kernel<T, V, VEC><<<blocks, kWarps * 32, smem, stream>>>(rows, routes, dgates, table, dloss,
                                                                          static_cast<T*>(dlogits));
}

// Pieces of 16 bytes (of the lane's whole share, where that is less) when every row starts on one, else single elements.
template <class T, int V>
constexpr int kPiece = V < 16 / static_cast<int>(sizeof(T)) ? V : 16 / static_cast<int>(sizeof(T));
template <class T, int V>
bool in_pieces(const Rows& a, const void* other) {
  constexpr int n = kPiece<T, V>;
  constexpr uintptr_t bytes = n * sizeof(T);
  if (a.bias && reinterpret_cast<uintptr_t>(a.bias) % 16) return false;   // read with the row's layout
  return n > 1 && a.experts % n == 0 && a.stride % n == 0 && reinterpret_cast<uintptr_t>(a.logits) % bytes == 0 &&
         reinterpret_cast<uintptr_t>(other) % bytes == 0;
}
// Calls f<T, V, VEC>: V slots of 32 experts hold a row.
#define WM_ROUTER_WITH(T, V, f, a, other, ...)                                                       \
  (in_pieces<T, V>(a, other) ? f<T, V, kPiece<T, V>>(a, __VA_ARGS__) : f<T, V, 1>(a, __VA_ARGS__))
#define WM_ROUTER_BY_SIZE(T, f, a, other, ...)                                       \
  ((a).experts <= 32    ? WM_ROUTER_WITH(T, 1, f, a, other, __VA_ARGS__)             \
   : (a).experts <= 64  ? WM_ROUTER_WITH(T, 2, f, a, other, __VA_ARGS__)             \
   : (a).experts <= 128 ? WM_ROUTER_WITH(T, 4, f, a, other, __VA_ARGS__)             \
   : (a).experts <= 256 ? WM_ROUTER_WITH(T, 8, f, a, other, __VA_ARGS__)             \
   : (a).experts <= 512 ? WM_ROUTER_WITH(T, 16, f, a, other, __VA_ARGS__)            \
                        : WM_ROUTER_WITH(T, 32, f, a, other, __VA_ARGS__))
#define WM_ROUTER_DISPATCH(dtype, f, a, other, ...)                                  \
  ((dtype) == 0   ? WM_ROUTER_BY_SIZE(__nv_bfloat16, f, a, other, __VA_ARGS__)       \
   : (dtype) == 1 ? WM_ROUTER_BY_SIZE(float, f, a, other, __VA_ARGS__)               \
                  : WM_ROUTER_BY_SIZE(__half, f, a, other, __VA_ARGS__))

int finish(const Rows& a, const Plan& p, const Records& rec, const int* given, int* counts, float* table,
           void* workspace, float* loss, cudaStream_t stream) {
  const dim3 grid((a.experts + 31) / 32, a.num_sequences);
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(kFinishWarps * 32);
  config.stream = stream;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  WM_CUDA(cudaLaunchKernelEx(&config, balance_finish_kernel, a, rec, given, counts, table,
                             reinterpret_cast<float*>(static_cast<char*>(workspace) + p.part), loss));
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
  if ((r->tokens > 0 && (!routes || !gates)) || !aligned(4, routes, gates, counts, loss, table) ||
      (balance && (!counts || !loss || !table || !workspace || workspace_bytes < p.bytes ||
                   reinterpret_cast<uintptr_t>(workspace) % 16))) {
    set_error("wm_router_forward: null or misaligned output, or a missing or small workspace (wm_router_workspace, 16-byte aligned)");
    return WM_ERR_INVALID;
  }
  if (r->tokens == 0 && !balance) return WM_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const Rows a = rows_of(*r, p);
  const Records rec = balance ? records_of(p, workspace, true) : Records{};
  // with no rows the kernel still clears the ticket of the kernel behind it
  WM_ROUTER_DISPATCH(r->dtype, forward_of, a, nullptr, p, routes, gates, rec, stream);
  count_launch();
  WM_CUDA(cudaGetLastError());
  return balance ? finish(a, p, rec, nullptr, counts, table, workspace, loss, stream) : WM_OK;
}

extern "C" int wm_balance_forward(const wm_router* r, const int32_t* counts, float* loss, float* table,
                                  void* workspace, int64_t workspace_bytes, void* stream_) {
  if (int rc = check_rows("wm_balance_forward", r)) return rc;
  const Plan p = plan_of(*r);
  if (!counts || !loss || !table || !aligned(4, counts, loss, table) || !workspace || workspace_bytes < p.bytes ||
      reinterpret_cast<uintptr_t>(workspace) % 16) {
    set_error("wm_balance_forward: null or misaligned argument, or a small workspace (wm_router_workspace, 16-byte aligned)");
    return WM_ERR_INVALID;
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  Rows a = rows_of(*r, p);
  a.bias = nullptr;
  const Records rec = records_of(p, workspace, false);
  int* no_routes = nullptr;
  float* no_gates = nullptr;
  WM_ROUTER_DISPATCH(r->dtype, forward_of, a, nullptr, p, no_routes, no_gates, rec, stream);
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
  if (!aligned(4, routes, dgates, dloss) || !aligned(16, table) || !aligned(r->dtype == 1 ? 4 : 2, dlogits)) {
    set_error("wm_router_backward: misaligned argument (table: 16 bytes, the others to their elements)");
    return WM_ERR_INVALID;
  }
  if (r->tokens == 0) return WM_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const Rows a = rows_of(*r, plan_of(*r));
  WM_ROUTER_DISPATCH(r->dtype, backward_of, a, dlogits, routes, dgates, table, dloss, dlogits, stream);
  count_launch();
  WM_CUDA(cudaGetLastError());
  return WM_OK;
}

extern "C" int wm_expert_counts(const int32_t* routes, int32_t tokens, int32_t top_k, int32_t experts,
                                const int32_t* sequences, int32_t num_sequences, int32_t* counts, void* stream_) {
  if (tokens < 0 || tokens > kMaxTokens || top_k < 1 || top_k > 32 || experts < 1 || experts > kMaxExperts || !counts ||
      (tokens > 0 && !routes) || (sequences ? num_sequences < 1 : num_sequences != 0) || num_sequences > 65535 ||
      !aligned(4, routes, sequences, counts)) {
    set_error("wm_expert_counts: routes [fewer than 2^26 tokens][1..32], 1..%d experts, 1..65535 sequences with their offsets",
              kMaxExperts);
    return WM_ERR_INVALID;
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int rows = sequences ? num_sequences : 1;
  Rows a{};
  a.tokens = tokens;
  a.experts = experts;
  a.top_k = top_k;
  a.sequences = sequences;
  a.num_sequences = rows;
  if (rows <= kClusterSequences && static_cast<long long>(tokens) * top_k <= kClusterRoutes) {
    expert_counts_cluster_kernel<<<dim3(kCountCtas, rows), kMaxExperts, experts * 4, stream>>>(a, routes, counts);
    count_launch();
    WM_CUDA(cudaGetLastError());
    return WM_OK;
  }
  WM_CUDA(cudaMemsetAsync(counts, 0, static_cast<size_t>(rows) * experts * 4, stream));
  if (tokens == 0) return WM_OK;
  const int want = (tokens + 127) / 128;
  const int blocks = want < 296 ? want : 296;
  a.chunk = (tokens + blocks - 1) / blocks;
  expert_counts_kernel<<<(tokens + a.chunk - 1) / a.chunk, 256, experts * 4, stream>>>(a, routes, counts);
  count_launch();
  WM_CUDA(cudaGetLastError());
  return WM_OK;
}
