// ec_logprobs.hip — ec_token_logprobs and ec_token_logprobs_grad: log
// probabilities of given tokens over rows of logits, with the entropy and the
// likeliest tokens, and their gradient.
//
// Everything is in base 2: with c = scale * log2 e, logit x has exponent x * c and
// a row's reference is mc = (its largest logit) * c, rounded once.  Every term is
// 2^fma(x, c, -mc) and the results are taken relative to the same mc,
//   s = SUM 2^d,  d = x c - mc,    lse = (mc + log2 s) ln 2,
//   log p = (d - log2 s) ln 2,     H = (log2 s - (SUM 2^d d) / s) ln 2,
// so the rounding of mc cancels in log p and H.  lse is given relative to z = scale * m as fp32
// rounds it, m the largest logit: lse = z + (log2 s - fma(m, c, -mc)) ln 2, so that the
// gradient, which takes z - lse, gives a logit that dominates probability 1.  x c leaves fp32's range where x
// does not (a mask of the type's lowest value): rows that this touches, and rows
// with a NaN or infinity, are gone over once more with d = (x - m) c.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ec_types.h"
#include "fastdiv.h"
#include "routes.h"

namespace ec {
namespace {

constexpr int kLanes = 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;
constexpr float kInf = __builtin_inff();
constexpr float kMax = 3.402823466e38f;

__device__ __forceinline__ float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float log2_hw(float v) { return __builtin_amdgcn_logf(v); }

// scale * x and the sum with `more`, each rounded (not as one fma): the same product must be
// rounded alike in the log of the sum and in what is compared with it.
__device__ __forceinline__ float scaled_plus(float x, float scale, float more) {
#pragma clang fp contract(off)
  return x * scale + more;
}

// Group g of a row of `vocab` logits, -infinity past its end.
template <typename T, bool STREAM>
__device__ __forceinline__ typename Group<T>::vec load_logits(const T* row, uint32_t g,
                                                              uint32_t vocab) {
  typedef Group<T> G;
  const uint32_t j = g * G::kN;
  if (j + G::kN <= vocab) return load_group<T, STREAM>(row + j);
  typename G::vec v;
#pragma unroll
  for (int e = 0; e < G::kN; ++e) v[e] = j + e < vocab ? (T)gp(row)[j + e] : (T)-kInf;
  return v;
}

// Logits in an order: larger values first, equal ones by index, NaN last, as
// one 64-bit key (larger key first).  -0 counts as +0.
__device__ __forceinline__ uint32_t order_bits(float v) {
  if (v != v) return 0u;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float v, uint32_t index) {
  return (uint64_t)order_bits(v) << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float order_value(uint64_t key) {   // -0 comes back as +0
  const uint32_t b = (uint32_t)(key >> 32);
  return b == 0 ? __builtin_nanf("") : __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

struct LogprobArgs {
  const void* logits;
  const int64_t* targets;
  float* logprobs;
  float* lse;
  float* entropy;
  float* top_logprobs;
  int64_t* top_tokens;
  uint64_t stride;
  uint32_t vocab, groups;   // groups of a row, the last one short
  float scale, c;           // c = scale * log2 e
  int top;
};

// A lane's running state over the groups it has seen: the largest logit and the
// group where it first stood, the reference, the sum and the weighted sum.  The
// reference moves only when a group holds a larger logit, a few times per lane,
// so a term costs one fma, one exp2 and one add (and a max and an fma for the entropy).
template <bool ENTROPY>
struct Running {
  float m = -kInf, mc = 0.0f, s = 0.0f, t = 0.0f;
  uint32_t group;

  template <int N, typename W>
  __device__ __forceinline__ void add(const W& x, uint32_t g, float c) {
    float top = x[0];
#pragma unroll
    for (int e = 1; e < N; ++e) top = fmaxf(top, x[e]);
    if (top > m) {
      const float to = fmaxf(top * c, -kMax);   // finite: a term below it is 0
      if (s != 0.0f) {
        const float by = exp2_hw(mc - to);
        // (far behind, 0 times a distance that may be infinite with this lane's s: a mask's
        // terms are 2^(the rounding of its x c), up to 2^128)
        if (ENTROPY) t = by == 0.0f ? 0.0f : by * (t - (to - mc) * s);
        s *= by;
      }
      m = top;
      mc = to;
      group = g;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = __builtin_fmaf(x[e], c, -mc);
      const float p = exp2_hw(d);
      s += p;
      // -200: a masked logit's -infinity would make 0 * infinity
      if (ENTROPY) t = __builtin_fmaf(p, fmaxf(d, -200.0f), t);
    }
  }
};

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// The sums of the workgroup's s (and t), the same in every lane.
template <int WAVES, bool BOTH>
__device__ __forceinline__ void block_sums(float& s, float& t, float (&red)[3][WAVES]) {
  s = wave_sum(s);
  if (BOTH) t = wave_sum(t);
  if (threadIdx.x % kLanes == 0) {
    red[1][threadIdx.x / kLanes] = s;
    if (BOTH) red[2][threadIdx.x / kLanes] = t;
  }
  __syncthreads();
  s = red[1][0];
  if (BOTH) t = red[2][0];
  for (int w = 1; w < WAVES; ++w) {
    s += red[1][w];
    if (BOTH) t += red[2][w];
  }
}

constexpr uint32_t kCandidates = 512;
constexpr int kAhead = 4;   // groups of a lane in flight

// Lanes per row: 512 for long rows and for few rows, 128 for many short ones.
// Lanes 128 / 256 / 512 / 1024, bf16, us with the likeliest five (with the entropy
// instead): 1 x 50304 17.8 11.7 8.8 9.0 (14.4 8.5 6.2 6.5); 256 x 16384 11.6 9.0 7.5 7.9;
// 1024 x 1024 8.8 8.0 7.9 13.7; 4096 x 1024 16.1 17.0 24.0 45.5 (4.8 6.7 11.0 23.2);
// 4096 x 16384 35.7 35.6 39.0 61.0 (29.0 27.2 26.1 36.8); 4096 x 50304 89.6 82.1
// 79.5 99.1 (78.5 78.0 75.0 81.8).
constexpr int kWideLanes = 512, kShortLanes = 128;
constexpr uint64_t kFewRows = 1024;
constexpr uint32_t kWideGroups = 2048;

// Logits of more bytes than this are streamed: half the Infinity Cache, past which
// little of what a matrix product has just written is left there.  8192 x 50304 bf16:
// 143 us cached, 127 streamed (the gradient 253 and 247); 64 x 131072: 25 and 29, the
// gradient of 2048 x 32001: 43 and 48.
constexpr uint64_t kStreamBytes = 128u << 20;

// By one wave: the top-th largest of 64 keys, each the largest of the same lane of
// every wave; 0 where fewer than `top` lanes have a group (those without one have key 0),
// so that all logits pass.
template <int WAVES>
__device__ __forceinline__ void top_bound(const uint64_t* keys, int top, uint64_t& bound) {
  const uint32_t lane = threadIdx.x % kLanes;
  uint64_t best = keys[lane];
  for (int w = 1; w < WAVES; ++w) best = max(best, keys[w * kLanes + lane]);
  const uint32_t hi = (uint32_t)(best >> 32), lo = (uint32_t)best;
  int above = 0;
#pragma unroll 8
  for (int o = 0; o < kLanes; ++o) {
    const uint64_t other = (uint64_t)__builtin_amdgcn_readlane(hi, o) << 32 |
                           (uint32_t)__builtin_amdgcn_readlane(lo, o);
    above += other > best;
  }
  const uint64_t last = __ballot(above == top - 1 && best != 0);
  if (last ? lane == (uint32_t)__builtin_ctzll(last) : lane == 0) bound = last ? best : 0;
}

// One workgroup of B lanes per row; lane l takes groups l, l + B, ...  Bound by memory, with the
// entropy nearly by the vector ALUs (10 slots an element, 4 of them the exp2): 8192 x 50304
// bf16 in 121 us (6.8 TB/s; 118 to 123).
//
// The `top` largest: any lane's largest logit that is among the `top` largest of
// the lanes' own bounds the answer from below, so the logits that are not behind
// the top-th largest of 64 groups of lanes (lane l of every wave) hold it.  They
// lie in the lanes whose own largest is not behind it; those lanes' groups are
// read again (about `top` lanes: a few percent of the row, from the caches), and
// the few logits that pass are ranked by counting.  Where more pass than
// kCandidates (logits that repeat with the workgroup's period) the row is
// searched `top` times instead.
template <typename T, int B, bool ENTROPY, bool TOP, bool STREAM>
__global__ void __launch_bounds__(B) logprob_kernel(const LogprobArgs a) {
  typedef Group<T> G;
  constexpr int kWaves = B / kLanes;
  __shared__ float red[3][kWaves];
  const uint32_t tid = threadIdx.x, lane = tid % kLanes, wave = tid / kLanes;
  const uint64_t r = blockIdx.x;
  const T* row = (const T*)a.logits + r * a.stride;

  const int64_t target = gp(a.targets)[r];   // not waited for before the loop's end
  Running<ENTROPY> run;
  run.group = tid;
  // whole groups: loads without conditions (lanes behind the row's end load its last group
  // again), so that a batch is in flight together
  const uint32_t full = a.vocab / G::kN;
  for (uint32_t g = tid; g < full; g += B * kAhead) {
    typename G::vec v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      v[u] = load_group<T, STREAM>(row + (uint64_t)min(g + u * B, full - 1) * G::kN);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (g + u * B < full) run.template add<G::kN>(widen<T>(v[u]), g + u * B, a.c);
  }
  if (full < a.groups && tid == full % B)
    run.template add<G::kN>(widen<T>(load_logits<T, false>(row, full, a.vocab)), full, a.c);

  float given = 0.0f;
  if (tid == 0 && target >= 0 && target < (int64_t)a.vocab) given = (float)gp(row)[target];

  // the workgroup's reference, then the sums relative to it
  __shared__ uint64_t keys[TOP ? (kCandidates > B ? kCandidates : B) : 1];
  __shared__ uint64_t bound_shared;
  __shared__ uint32_t lanes_list[TOP ? B : 1];
  __shared__ uint32_t n_lanes, n_keys;
  uint64_t mine = 0;
  if constexpr (TOP) {
    mine = tid < a.groups ? order_key(run.m, run.group) : 0;
    keys[tid] = mine;
    if (tid == 0) n_lanes = n_keys = 0;
  }
  const float wm = wave_max(run.m);
  if (lane == 0) red[0][wave] = wm;
  __syncthreads();
  if constexpr (TOP) {
    if (wave == 0) top_bound<kWaves>(keys, a.top, bound_shared);
  }
  float m = red[0][0];
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, red[0][w]);
  const float mc = fmaxf(m * a.c, -kMax);
  float s = 0.0f, t = 0.0f;
  if (run.s != 0.0f) {
    const float by = exp2_hw(run.mc - mc);
    s = run.s * by;
    // a lane that is far behind adds nothing; its distance may be infinite
    if (ENTROPY) t = by == 0.0f ? 0.0f : by * (run.t - (mc - run.mc) * run.s);
  }
  block_sums<kWaves, ENTROPY>(s, t, red);
  // every logit -infinity, or one of the rows that need d = (x - m) c
  const bool empty = m == -kInf && s == 0.0f;
  const bool again = !empty && !(s > 0.0f && s < kInf && (!ENTROPY || __builtin_isfinite(t)));
  if (again) {
    s = t = 0.0f;
    for (uint32_t g = tid; g < a.groups; g += B) {
      const typename G::wide x = widen<T>(load_logits<T, false>(row, g, a.vocab));
#pragma unroll
      for (int e = 0; e < G::kN; ++e) {
        const float d = (x[e] - m) * a.c;
        const float p = exp2_hw(d);
        s += p;
        if (ENTROPY) t = __builtin_fmaf(p, fmaxf(d, -200.0f), t);
      }
    }
    __syncthreads();
    block_sums<kWaves, ENTROPY>(s, t, red);
  }
  const float log2s = log2_hw(s);
  const auto logprob = [&](float x) {
    if (empty) return -kInf;
    return ((again ? (x - m) * a.c : __builtin_fmaf(x, a.c, -mc)) - log2s) * kLn2;
  };
  if (tid == 0) {
    // (an exponent of m is 0 but for the rounding of mc)
    const float rest = again ? log2s : log2s - __builtin_fmaf(m, a.c, -mc);
    gp(a.lse)[r] = empty ? -kInf : scaled_plus(m, a.scale, rest * kLn2);
    gp(a.logprobs)[r] = target >= 0 && target < (int64_t)a.vocab ? logprob(given) : 0.0f;
    if (ENTROPY) gp(a.entropy)[r] = empty ? 0.0f : (log2s - t / s) * kLn2;
  }
  if constexpr (TOP) {
    const uint64_t bound = bound_shared;
    if (mine && mine >= bound) lanes_list[atomicAdd(&n_lanes, 1u)] = tid;
    __syncthreads();
    const uint32_t lanes = n_lanes;
    const uint32_t bound_value = (uint32_t)(bound >> 32), bound_group = ~(uint32_t)bound;
    for (uint32_t l = wave; l < lanes; l += kWaves) {
      const uint32_t first = lanes_list[l];
      for (uint32_t g = first + lane * B; g < a.groups; g += kLanes * B) {
        const typename G::vec v = load_logits<T, false>(row, g, a.vocab);
#pragma unroll
        for (int e = 0; e < G::kN; ++e) {
          const uint32_t j = g * G::kN + e, value = order_bits((float)v[e]);
          if (j < a.vocab && (value > bound_value || (value == bound_value && g <= bound_group))) {
            const uint32_t at = atomicAdd(&n_keys, 1u);
            if (at < kCandidates) keys[at] = (uint64_t)value << 32 | (uint32_t)~j;
          }
        }
      }
    }
    __syncthreads();
    const uint32_t n = n_keys;
    const auto put = [&](int rank, uint64_t key) {
      gp(a.top_tokens)[r * a.top + rank] = (uint32_t)~key;
      gp(a.top_logprobs)[r * a.top + rank] = logprob(order_value(key));
    };
    if (n <= kCandidates && n >= (uint32_t)a.top) {
      for (uint32_t i = tid; i < n; i += B) {
        const uint64_t key = keys[i];
        int above = 0;
        for (uint32_t o = 0; o < n; ++o) above += keys[o] > key;
        if (above < a.top) put(above, key);
      }
    } else {
      uint64_t before = ~0ull;
      for (int k = 0; k < a.top; ++k) {
        uint64_t best = 0;
        for (uint32_t g = tid; g < a.groups; g += B) {
          const typename G::vec v = load_logits<T, false>(row, g, a.vocab);
#pragma unroll
          for (int e = 0; e < G::kN; ++e) {
            const uint32_t j = g * G::kN + e;
            const uint64_t key = j < a.vocab ? order_key((float)v[e], j) : 0;
            if (key < before) best = max(best, key);
          }
        }
        __syncthreads();
        keys[tid] = best;
        __syncthreads();
        for (int o = B / 2; o; o >>= 1) {
          if (tid < (uint32_t)o) keys[tid] = max(keys[tid], keys[tid + o]);
          __syncthreads();
        }
        before = keys[0];
        if (tid == 0) put(k, before);
      }
    }
  }
}

// ---------------------------------------------------------------- gradient --
// dlogits = -p (A + B d) + scale g at the target, with d = z - lse, p = e^d, A = scale (g + h H),
// B = scale h.  z and the difference are rounded as in the forward pass, and only then taken to
// base 2: fma(x, c, -lse log2 e) is one instruction less, but off by the rounding of the two
// factors times log2 e, 2^-24 |lse|, and made probabilities above 1 of logits from 1e6 on.
// p is at most 1, also from an lse that was found elsewhere and rounded otherwise.
struct GradArgs {
  const void* logits;
  void* out;
  const int64_t* targets;
  const float* lse;
  const float* dlogprobs;
  const float* entropy;
  const float* dentropy;
  uint64_t stride, out_stride;
  FastDiv by_slabs;
  uint32_t vocab, groups, slabs;   // slabs: workgroups of a row
  float scale, masked;             // an lse below `masked`: a row of nothing but masked logits
};

// (fp32 has lost what tells such a row's logits apart; 2^127 / log2 e, a third of the range, and
// as much less as a scale below 1 brings the type's lowest value nearer)
constexpr float kMaskedLse = -0x1p127f / kLog2e;

// A lane takes one group, and the workgroups follow the memory's order: 8192 x 50304
// bf16 in 247 us (6.7 TB/s; a copy kernel of the same form takes 244, the library's
// copy 324), against 316 with four groups a lane and consecutive workgroups on
// different rows, 273 with four groups a lane in memory order.
constexpr int kGradLanes = 256;

template <typename T, bool ENTROPY, bool STREAM>
__global__ void __launch_bounds__(kGradLanes) logprob_grad_kernel(const GradArgs a) {
  typedef Group<T> G;
  constexpr int N = G::kN;
  const uint32_t r = fast_div(blockIdx.x, a.by_slabs);
  const uint32_t gi = (blockIdx.x - r * a.slabs) * kGradLanes + threadIdx.x;
  if (gi >= a.groups) return;
  const T* row = (const T*)a.logits + (uint64_t)r * a.stride;
  T* out = (T*)a.out + (uint64_t)r * a.out_stride;
  const typename G::vec v = load_logits<T, STREAM>(row, gi, a.vocab);
  const int64_t target = gp(a.targets)[r];
  const float lse = gp(a.lse)[r];
  const bool has = target >= 0 && target < (int64_t)a.vocab, empty = lse < a.masked;
  const float g = has ? (float)gp(a.dlogprobs)[r] : 0.0f;
  float A = a.scale * g, slope = 0.0f;
  if (ENTROPY) {
    const float h = gp(a.dentropy)[r];
    A += a.scale * h * gp(a.entropy)[r];
    slope = a.scale * h;
  }
  const typename G::wide x = widen<T>(v);
  typename G::wide w;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float d = __builtin_elementwise_minimum(scaled_plus(x[e], a.scale, -lse), 0.0f);   // NaN stays
    const float p = exp2_hw(d * kLog2e);
    const float by = ENTROPY ? __builtin_fmaf(fmaxf(d, -200.0f), slope, A) : A;
    w[e] = empty ? 0.0f : -p * by;
  }
  const uint32_t j = gi * N;
  if (has && !empty && (uint32_t)target - j < (uint32_t)N) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if ((uint32_t)target == j + e) w[e] += a.scale * g;
  }
  if (j + N <= a.vocab)
    store_wide<T, true>(out + j, w);
  else
    for (int e = 0; e < N; ++e)
      if (j + e < a.vocab) gp(out)[j + e] = (T)w[e];
}

int check_logits(const void* logits, int type, uint64_t rows, uint64_t vocab, uint64_t stride,
                 const int64_t* targets, float scale) {
  if (!known_type(type) || !(scale > 0.0f) || !std::isfinite(scale * kLog2e)) return EC_EINVAL;
  if (rows >= (1ull << 31) || vocab >= (1ull << 31)) return EC_ERANGE;
  if (rows && (!targets || (vocab && (!logits || stride < vocab)))) return EC_EINVAL;
  return EC_OK;
}

}  // namespace
}  // namespace ec

using namespace ec;

extern "C" {

int ec_token_logprobs(const void* d_logits, int type, uint64_t rows, uint64_t vocab,
                      uint64_t row_stride, const int64_t* d_targets, float scale,
                      float* d_logprobs, float* d_lse, float* d_entropy, int top,
                      float* d_top_logprobs, int64_t* d_top_tokens, ec_stream_t stream) {
  if (const int st = check_logits(d_logits, type, rows, vocab, row_stride, d_targets, scale))
    return st;
  if (top < 0 || (uint64_t)top > vocab) return EC_EINVAL;
  if (top > EC_MAX_TOP) return EC_ERANGE;
  if (!rows) return EC_OK;
  if (!d_logprobs || !d_lse || (top && (!d_top_logprobs || !d_top_tokens))) return EC_EINVAL;
  LogprobArgs a = {d_logits, d_targets, d_logprobs, d_lse, d_entropy, d_top_logprobs,
                   d_top_tokens, row_stride, (uint32_t)vocab, 0, scale, scale * kLog2e, top};
  const uint32_t per_group = 16 / type_bytes(type);
  a.groups = (uint32_t)((vocab + per_group - 1) / per_group);
  const bool streamed = rows * vocab * type_bytes(type) > kStreamBytes;
  const bool wide = rows <= kFewRows || a.groups >= kWideGroups;
  const uint64_t most = max_grid(wide ? kWideLanes : kShortLanes);   // rows of one launch
  const hipStream_t st = (hipStream_t)stream;
  return with_type(type, [&](auto t) {
    typedef decltype(t) T;
    const auto go = [&](auto entropy, auto tops, auto stream_) {
      constexpr bool E = decltype(entropy)::value, K = decltype(tops)::value;
      constexpr bool S = decltype(stream_)::value;
      for (uint64_t at = 0; at < rows; at += most) {
        const dim3 grid((uint32_t)std::min(most, rows - at));
        a.logits = (const T*)d_logits + at * row_stride;
        a.targets = d_targets + at;
        a.logprobs = d_logprobs + at;
        a.lse = d_lse + at;
        if (E) a.entropy = d_entropy + at;
        if (K) a.top_logprobs = d_top_logprobs + at * top;
        if (K) a.top_tokens = d_top_tokens + at * top;
        if (wide)
          logprob_kernel<T, kWideLanes, E, K, S><<<grid, kWideLanes, 0, st>>>(a);
        else
          logprob_kernel<T, kShortLanes, E, K, S><<<grid, kShortLanes, 0, st>>>(a);
      }
      return launched();
    };
    const std::true_type yes;
    const std::false_type no;
    const auto with = [&](auto entropy, auto tops) {
      return streamed ? go(entropy, tops, yes) : go(entropy, tops, no);
    };
    if (d_entropy) return top ? with(yes, yes) : with(yes, no);
    return top ? with(no, yes) : with(no, no);
  });
}

int ec_token_logprobs_grad(const void* d_logits, int type, uint64_t rows, uint64_t vocab,
                           uint64_t row_stride, const int64_t* d_targets, const float* d_lse,
                           const float* d_dlogprobs, const float* d_entropy,
                           const float* d_dentropy, float scale, void* d_dlogits,
                           uint64_t out_stride, ec_stream_t stream) {
  if (const int st = check_logits(d_logits, type, rows, vocab, row_stride, d_targets, scale))
    return st;
  if (!rows || !vocab) return EC_OK;
  if (!d_lse || !d_dlogprobs || !d_dlogits || out_stride < vocab) return EC_EINVAL;
  if (!d_entropy != !d_dentropy) return EC_EINVAL;
  GradArgs a = {d_logits, d_dlogits, d_targets, d_lse, d_dlogprobs, d_entropy, d_dentropy,
                row_stride, out_stride, {}, (uint32_t)vocab, 0, 0, scale, kMaskedLse * std::min(scale, 1.0f)};
  const uint32_t per_group = 16 / type_bytes(type);
  a.groups = (uint32_t)((vocab + per_group - 1) / per_group);
  const bool streamed = rows * vocab * type_bytes(type) > kStreamBytes;
  a.slabs = (a.groups + kGradLanes - 1) / kGradLanes;
  a.by_slabs = make_fastdiv(a.slabs);
  const uint64_t most = max_grid(kGradLanes) / a.slabs;   // rows of one launch; a row has at most 2^21
  const hipStream_t st = (hipStream_t)stream;
  return with_type(type, [&](auto t) {
    typedef decltype(t) T;
    const auto kernel = d_dentropy ? streamed ? logprob_grad_kernel<T, true, true>
                                              : logprob_grad_kernel<T, true, false>
                                   : streamed ? logprob_grad_kernel<T, false, true>
                                              : logprob_grad_kernel<T, false, false>;
    for (uint64_t at = 0; at < rows; at += most) {
      const uint32_t grid = (uint32_t)(std::min(most, rows - at) * a.slabs);
      a.logits = (const T*)d_logits + at * row_stride;
      a.out = (T*)d_dlogits + at * out_stride;
      a.targets = d_targets + at;
      a.lse = d_lse + at;
      a.dlogprobs = d_dlogprobs + at;
      if (d_dentropy) {
        a.entropy = d_entropy + at;
        a.dentropy = d_dentropy + at;
      }
      kernel<<<grid, kGradLanes, 0, st>>>(a);
    }
    return launched();
  });
}

}  // extern "C"
