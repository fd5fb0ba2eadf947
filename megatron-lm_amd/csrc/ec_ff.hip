// ec_ff.hip — ec_gated_ff and ec_gated_ff_grad: act(x Wg') * (x Wu') and its gradients.
//
// Forward: one product whose second operand is both weights' rows in turns, 32 of each, so that a
// wave holds the gate and the up projection of the same outputs in its accumulators and
// neither of them goes to memory.
//
// Backward: the same product again, whose epilogue turns g, u and dh into dg = dh u act'(g) and
// du = dh act(g) ([n][2 inner] in the workspace), then dx = dg Wg + du Wu and dW = d' x as two products
// more, 12 n width inner operations in all.  Computing the projections again costs 4 of
// them and keeps 2 n inner values from being stored between the passes.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "ec_gemm.h"
#include "ec_pack.h"

namespace ec {
namespace {

struct Act {
  float value, slope;
};

// The activation and its derivative at g, both from one exponential (or the error function).  The hardware's
// exp2 and reciprocal are 1 ulp off; the argument's rounding makes that |z| ulp of a sigmoid, where it is
// still felt at all. (With the library's exp and an exact division the epilogue took a fifth of 16384 x 2048 ->
// 8192: 960 us against 873.)
template <int ACT>
__device__ __forceinline__ Act activate(float g) {
  if constexpr (ACT == EC_ACT_GELU) {
    const float p = 0.5f * erfcf(-0.70710678f * g);
    return {g * p, p + g * 0.39894228f * __builtin_amdgcn_exp2f(-0.72134752f * g * g)};
  } else {
    // silu and the tanh form of gelu are g * sigmoid(z), z = g or 2 sqrt(2 / pi) (g + 0.044715 g^3)
    float z = g, dz = 1.0f;
    if constexpr (ACT == EC_ACT_GELU_TANH) {
      const float c = 1.59576912f, g2 = g * g;
      z = c * g * (1.0f + 0.044715f * g2);
      dz = c * (1.0f + 3.0f * 0.044715f * g2);
    }
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * z));
    // far out z' may overflow where s (1 - s) is 0
    const float bend = s * (1.0f - s);
    return {g * s, s + (bend > 0.0f ? g * bend * dz : 0.0f)};
  }
}

// f(activation) with the activation as a constant.
template <typename F>
__device__ __forceinline__ void with_activation(uint32_t act, F f) {
  if (act == EC_ACT_SILU)
    f(std::integral_constant<int, EC_ACT_SILU>());
  else if (act == EC_ACT_GELU)
    f(std::integral_constant<int, EC_ACT_GELU>());
  else
    f(std::integral_constant<int, EC_ACT_GELU_TANH>());
}

struct FfArgs {
  Operand x, w_gate, w_up;
  uint32_t n, width, inner, act;
  uint32_t tiles_m, tiles_n;
  char* h;
  uint64_t h_stride;
  const char* dh;        // backward
  uint64_t dh_stride;
  char* d;               // [n][2 padded] of T, and the second parts behind it
  uint32_t padded;
  uint64_t low;          // elements from a value of d to its second part; 0: none
  Splits splits;
};

template <class S, typename T>
__global__ void __launch_bounds__(S::kLanes, S::kPerSimd) ff_part_kernel(FfArgs p) {
  __shared__ __attribute__((aligned(1024))) char lds[S::kLds];
  const uint32_t tiles = p.tiles_m * p.tiles_n, t = xcd_order(blockIdx.x, gridDim.x), split = uniform(t / tiles);
  uint32_t tm, tn;
  tile_at(t % tiles, p.tiles_m, p.tiles_n, tm, tn);
  Acc<S> acc;
  acc.clear();
  const uint32_t s0 = split * p.splits.steps;
  product<S, T, false, false, true>(acc, (local<char>*)lds, from_step<T, false>(p.x, s0),
                                    from_step<T, false>(p.w_gate, s0), from_step<T, false>(p.w_up, s0),
                                    tm * S::BM, tn * S::BN, split_length<T>(p.splits, split, p.width));
  store_part(acc, p.splits.parts, t);
}

template <class S, typename T, bool GRAD, bool JOIN>
__global__ void __launch_bounds__(S::kLanes, S::kPerSimd) ff_kernel(FfArgs p) {
  __shared__ __attribute__((aligned(1024))) char lds[JOIN ? 16 : S::kLds];
  const uint32_t t = xcd_order(blockIdx.x, gridDim.x);
  uint32_t tm, tn;
  tile_at(t, p.tiles_m, p.tiles_n, tm, tn);
  // of each 64 columns of the tile the first 32 are gates, the others the ups
  static_assert(S::WN == 64, "a wave holds both projections of its 32 outputs");
  const uint32_t l = threadIdx.x % 64, w = threadIdx.x / 64;
  const uint32_t m0 = tm * S::BM + w / S::kWavesN * S::WM + l % 16 / 4 * 8 + l % 4;
  const uint32_t f = tn * (S::BN / 2) + w % S::kWavesN * 32 + l / 16 * 8;
  // dh is under way during the product; past its ends some other value, which is not used
  typedef T __attribute__((ext_vector_type(8), aligned(sizeof(T)))) any8;
  T __attribute__((ext_vector_type(8))) dhs[GRAD ? S::MI : 1];
  if constexpr (GRAD) {
    const bool whole = (tn + 1) * (S::BN / 2) <= p.inner;
#pragma unroll
    for (int i = 0; i < S::MI; ++i) {
      const T* row = (const T*)p.dh + min(m0 + i / 2 * 32 + i % 2 * 4, p.n - 1) * p.dh_stride;
      if (whole) {
        dhs[i] = *(const global<any8>*)(uintptr_t)(row + f);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) dhs[i][e] = gp(row)[min(f + e, p.inner - 1)];
      }
    }
  }
  Acc<S> acc;
  acc.clear();
  if constexpr (JOIN)
    add_parts(acc, p.splits.parts, t, gridDim.x, p.splits.n);
  else
    product<S, T, false, false, true>(acc, (local<char>*)lds, p.x, p.w_gate, p.w_up, tm * S::BM,
                                      tn * S::BN, p.width);
  with_activation(p.act, [&](auto which) {
    constexpr int ACT = decltype(which)::value;
#pragma unroll
    for (int i = 0; i < S::MI; ++i) {
      const uint32_t m = m0 + i / 2 * 32 + i % 2 * 4;
      if (m >= p.n) continue;
      const f8 g = acc.pair(i, 0), u = acc.pair(i, 2);
      if constexpr (!GRAD) {
        f8 h;
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = activate<ACT>(g[e]).value * u[e];
        store8<T>((T*)p.h + m * p.h_stride, f, p.inner, h);
      } else {
        const f8 dh = __builtin_convertvector(dhs[i], f8);
        f8 dg, du;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const Act a = activate<ACT>(g[e]);
          const bool in = f + e < p.inner;   // zeros in the padding, which is summed over
          dg[e] = in ? dh[e] * u[e] * a.slope : 0.0f;
          du[e] = in ? dh[e] * a.value : 0.0f;
        }
        T* row = (T*)p.d + (uint64_t)m * 2 * p.padded;
        store8<T>(row, f, p.padded, dg);
        store8<T>(row + p.padded, f, p.padded, du);
        if (p.low) {
          f8 lg, lu;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            lg[e] = dg[e] - (float)(T)dg[e];
            lu[e] = du[e] - (float)(T)du[e];
          }
          store8<T>(row + p.low, f, p.padded, lg);
          store8<T>(row + p.low + p.padded, f, p.padded, lu);
        }
      }
    }
  });
}

// Few rows: the weights are read once, straight to registers, and the reading bounds it.  A workgroup takes 16
// outputs, 16 rows of either weight; its waves split the width.  A wave's weights are the first
// operand of 16 x 16 products, 16 * TT rows of x the second, so a lane holds four outputs of one row of x.  The waves'
// sums are added in order through LDS.  Rows may have any address and length, so nothing is copied first.
constexpr int kFewWaves = 8, kFewAhead = 4;

template <typename T, int TT>
__global__ void __launch_bounds__(kFewWaves * 64) few_kernel(FfArgs p) {
  typedef Group<T> G;
  constexpr uint32_t kChunk = 4 * G::kN;   // of a row, that a fragment's four lanes read
  const uint32_t l = threadIdx.x % 64, wave = uniform(threadIdx.x / 64), i = l % 16, q = l / 16;
  const uint32_t f0 = blockIdx.x * 16;
  const uint64_t row = min(f0 + i, p.inner - 1);   // the last rows again past the end, not stored
  const T* gate = (const T*)(p.w_gate.p + row * p.w_gate.ld);
  const T* up = (const T*)(p.w_up.p + row * p.w_up.ld);
  const T* x[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t)   // and so with the rows of x
    x[t] = (const T*)(p.x.p + (uint64_t)min(t * 16 + i, p.n - 1) * p.x.ld);
  f4 g[TT], u[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) g[t] = u[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  // kFewAhead chunks from c on, `get` brings what is at element k of a row
  const auto chunks_of = [&](uint32_t c, auto get) {
    typename G::vec wg[kFewAhead], wu[kFewAhead], xv[kFewAhead][TT];
#pragma unroll
    for (int a = 0; a < kFewAhead; ++a) {
      const uint32_t k = (c + a) * kChunk + q * G::kN;
      wg[a] = get(gate, k);
      wu[a] = get(up, k);
#pragma unroll
      for (int t = 0; t < TT; ++t) xv[a][t] = get(x[t], k);
    }
#pragma unroll
    for (int a = 0; a < kFewAhead; ++a)
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const Frag<T> fx = {{__builtin_bit_cast(s8, xv[a][t])}};
        mma<T>(g[t], fx, Frag<T>{{__builtin_bit_cast(s8, wg[a])}});
        mma<T>(u[t], fx, Frag<T>{{__builtin_bit_cast(s8, wu[a])}});
      }
  };
  const uint32_t chunks = (p.width + kChunk - 1) / kChunk;
  const uint32_t each = ((chunks + kFewWaves - 1) / kFewWaves + kFewAhead - 1) / kFewAhead * kFewAhead;
  const uint32_t first = wave * each, last = min(first + each, chunks);
  uint32_t c = first;
  for (; c + kFewAhead <= last && (c + kFewAhead) * kChunk <= p.width; c += kFewAhead)
    chunks_of(c, [](const T* row, uint32_t k) { return load_group<T, false>(row + k); });
  if (c < last) {
    const uint32_t end = min(last * kChunk, p.width);   // zeros behind it
    chunks_of(c, [&](const T* row, uint32_t k) {
      typename G::vec v = {};
      if (k + G::kN <= end) return load_group<T, false>(row + k);
#pragma unroll
      for (int e = 0; e < G::kN; ++e)
        if (k + e < end) v[e] = gp(row)[k + e];
      return v;
    });
  }
  __shared__ f4 sums[kFewWaves][2][TT][64];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    sums[wave][0][t][l] = g[t];
    sums[wave][1][t][l] = u[t];
  }
  __syncthreads();
  if (wave >= TT) return;
  f4 gs = sums[0][0][wave][l], us = sums[0][1][wave][l];
#pragma unroll
  for (int w = 1; w < kFewWaves; ++w) {
    gs += sums[w][0][wave][l];
    us += sums[w][1][wave][l];
  }
  const uint32_t m = wave * 16 + i, f = f0 + q * 4;
  if (m >= p.n) return;
  T* out = (T*)p.h + m * p.h_stride;
  with_activation(p.act, [&](auto which) {
    constexpr int ACT = decltype(which)::value;
    f4 h;
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = activate<ACT>(gs[e]).value * us[e];
    typedef T __attribute__((ext_vector_type(4))) t4;
    typedef T __attribute__((ext_vector_type(4), aligned(sizeof(T)))) any4;
    if (f + 4 <= p.inner) {
      *(global<any4>*)(uintptr_t)(out + f) = __builtin_convertvector(h, t4);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (f + e < p.inner) gp(out)[f + e] = (T)h[e];
    }
  });
}

// C = the sum of up to four products, all across in their second operand.
struct SumArgs {
  Operand a[4], b[4];
  uint32_t parts, K, M, N;
  uint32_t tiles_m, tiles_n;
  char* out[2];   // blockIdx.y's
  uint64_t out_stride[2];
  uint64_t a_step;   // bytes from blockIdx.y = 0's first operand to 1's
  bool accumulate;   // added to what is there
  Splits splits;     // each takes its steps of every product
};

template <class S, typename T, bool ACROSS_A>
__device__ __forceinline__ void sum_products(Acc<S>& acc, local<char>* lds, const SumArgs& p, uint32_t tm,
                                             uint32_t tn, uint32_t which, uint32_t split, uint32_t K) {
  const uint32_t s0 = split * p.splits.steps;
  for (uint32_t i = 0; i < p.parts; ++i) {
    Operand a = from_step<T, ACROSS_A>(p.a[i], s0);
    a.p += which * p.a_step;
    const Operand b = from_step<T, true>(p.b[i], s0);
    product<S, T, ACROSS_A, true, false>(acc, lds, a, b, b, tm * S::BM, tn * S::BN, K);
  }
}

// Workgroup t of a split's, or a result's `which`-th sum.
template <class S, typename T, bool ACROSS_A>
__device__ __forceinline__ void sum_part(const SumArgs& p, local<char>* lds, uint32_t t, uint32_t which) {
  const uint32_t tiles = p.tiles_m * p.tiles_n, split = uniform(t / tiles);
  uint32_t tm, tn;
  tile_at(t % tiles, p.tiles_m, p.tiles_n, tm, tn);
  Acc<S> acc;
  acc.clear();
  sum_products<S, T, ACROSS_A>(acc, lds, p, tm, tn, which, split, split_length<T>(p.splits, split, p.K));
  store_part(acc, p.splits.parts, (uint64_t)which * tiles * p.splits.n + t);
}

template <class S, typename T, typename O, bool ACROSS_A, bool JOIN>
__device__ __forceinline__ void sum_tile(const SumArgs& p, local<char>* lds, uint32_t t, uint32_t which) {
  uint32_t tm, tn;
  tile_at(t, p.tiles_m, p.tiles_n, tm, tn);
  const uint32_t tiles = p.tiles_m * p.tiles_n;
  Acc<S> acc;
  acc.clear();
  if constexpr (JOIN)
    add_parts(acc, p.splits.parts, (uint64_t)which * tiles * p.splits.n + t, tiles, p.splits.n);
  else
    sum_products<S, T, ACROSS_A>(acc, lds, p, tm, tn, which, 0, p.K);
  O* out = (O*)p.out[which];
  const uint64_t stride = p.out_stride[which];
  const uint32_t m0 = tm * S::BM, n0 = tn * S::BN;
  const auto put = [&](uint32_t m, uint32_t n, const f8& v) {
    m += m0;
    n += n0;
    if (m < p.M && n < p.N) store8<O>(out + m * stride, n, p.N, v);
  };
  if (ACROSS_A && p.accumulate)
    acc.each_with([&](uint32_t m, uint32_t n) { return load8(out + min(m0 + m, p.M - 1) * stride, n0 + n, p.N); },
                  [&](uint32_t m, uint32_t n, const f8& v, const f8& x) { put(m, n, v + x); });
  else
    acc.each(put);
}

template <class S, typename T, bool ACROSS_A>
__global__ void __launch_bounds__(S::kLanes, S::kPerSimd) sum_part_kernel(SumArgs p) {
  __shared__ __attribute__((aligned(1024))) char lds[S::kLds];
  sum_part<S, T, ACROSS_A>(p, (local<char>*)lds, xcd_order(blockIdx.x, gridDim.x), blockIdx.y);
}

template <class S, typename T, typename O, bool ACROSS_A, bool JOIN>
__global__ void __launch_bounds__(S::kLanes, S::kPerSimd) sum_kernel(SumArgs p) {
  __shared__ __attribute__((aligned(1024))) char lds[JOIN ? 16 : S::kLds];
  sum_tile<S, T, O, ACROSS_A, JOIN>(p, (local<char>*)lds, xcd_order(blockIdx.x, gridDim.x), blockIdx.y);
}

// dx in small tiles (SPLIT: the splits of them) and both dW in tiles of S, in one launch: neither fills the CUs by itself
// (777 rows 1001 -> 1333 fp16 22.4 us, 17.3 and 14.5 one after the other).
template <class S, typename T, typename O, bool SPLIT>
__global__ void __launch_bounds__(S::kLanes, S::kPerSimd) sum_both_kernel(SumArgs x, SumArgs w) {
  static_assert(S::kLanes == Small::kLanes, "one workgroup size");
  __shared__ __attribute__((aligned(1024))) char lds[S::kLds > Small::kLds ? S::kLds : Small::kLds];
  const uint32_t first = x.tiles_m * x.tiles_n * x.splits.n;
  if (blockIdx.x < first) {
    const uint32_t t = xcd_order(blockIdx.x, first);
    if constexpr (SPLIT)
      sum_part<Small, T, false>(x, (local<char>*)lds, t, 0);
    else
      sum_tile<Small, T, T, false, false>(x, (local<char>*)lds, t, 0);
  } else {
    const uint32_t tiles = w.tiles_m * w.tiles_n, t = xcd_order(blockIdx.x - first, 2 * tiles);
    sum_tile<S, T, O, true, false>(w, (local<char>*)lds, t % tiles, uniform(t / tiles));
  }
}

// Rows up to which few_kernel takes the forward pass. 2048 -> 8192 bf16, eight sets of weights in turns, us: 1 row 14.9,
// 16 rows 17.1, 32 rows 20.5, 64 rows 28.8; tiles take 20.2 for 65 rows.
constexpr uint64_t kFewForward = 32;

struct FfWork {
  uint64_t x, w_gate, w_up, d, parts, total;   // offsets; kNone: read in place
  bool low;
};
constexpr uint64_t kNone = ~0ull;
constexpr uint32_t kMostWidth = 1u << 19;

// Up to this many rows the gradients of the projections keep a second part, the first one's
// rounding error, and the products take it along: the roundings of few rows do not
// average out, and the products cost little there.
constexpr uint64_t kFewRows = 256;

struct FfCall {
  const void *x, *w_gate, *w_up;
  uint64_t x_stride, gate_stride, up_stride, n;
  uint32_t width, inner;
  int type;
};

template <typename T>
Choice choose_ff(uint64_t n, uint64_t width, uint64_t inner) {
  return choose<T, Flat>([&](auto s) { return tiles_of(n, 2 * inner, s.BM, s.BN); }, steps_of<T>(width));
}

// An m x n sum of `parts` products over K, `outs` times.
template <typename T>
Choice choose_sum(uint64_t m, uint64_t n, uint64_t K, uint64_t parts, uint64_t outs) {
  const uint64_t steps = std::max<uint64_t>(1, steps_of<T>(K));
  Choice c = choose<T, Small>([&](auto s) { return outs * tiles_of(m, n, s.BM, s.BN); }, steps * parts);
  c.splits.steps = (uint32_t)((steps + c.splits.n - 1) / c.splits.n);   // of each product
  c.splits.n = (uint32_t)((steps + c.splits.steps - 1) / c.splits.steps);
  return c;
}

// Products of the gradients with the low parts: twice as many.
uint64_t low_parts(const FfWork& w) { return w.low ? 2 : 1; }

FfWork ff_work(const FfCall& c, bool grad) {
  const uint32_t b = type_bytes(c.type);
  const uint64_t row = up_to((uint64_t)c.width * b, 16);
  FfWork w = {kNone, kNone, kNone, kNone, kNone, 0, false};
  const auto take = [&](uint64_t bytes) {
    const uint64_t at = w.total;
    w.total += part(bytes);
    return at;
  };
  if (!c.n || (!grad && c.n <= kFewForward)) return w;   // none are read, or read as they are
  if (!readable(c.x, c.width, c.x_stride, b)) w.x = take(c.n * row);
  // the two weights are read in turns, so their rows have to be equally far apart
  if (c.gate_stride != c.up_stride || !readable(c.w_gate, c.width, c.gate_stride, b) ||
      !readable(c.w_up, c.width, c.up_stride, b)) {
    w.w_gate = take(c.inner * row);
    w.w_up = take(c.inner * row);
  }
  if (grad) {
    w.low = c.type != EC_F32 && c.n <= kFewRows;
    w.d = take(c.n * 2 * up_to(c.inner, 8) * b * low_parts(w));
  }
  uint64_t bytes = 0;
  with_type(c.type, [&](auto t) {
    typedef decltype(t) T;
    bytes = choose_ff<T>(c.n, c.width, c.inner).bytes;
    if (grad) {
      bytes = std::max(bytes, choose_sum<T>(c.n, c.width, c.inner, 2 * low_parts(w), 1).bytes);
      bytes = std::max(bytes, choose_sum<T>(c.inner, c.width, c.n, low_parts(w), 2).bytes);
    }
    return EC_OK;
  });
  if (bytes) w.parts = take(bytes);
  return w;
}

template <typename T>
Operand in_place(const void* p, uint64_t stride, uint64_t rows, uint32_t width, uint64_t at, char* work,
                 Packer<T>& packer) {
  if (at == kNone) return {(const char*)p, stride * sizeof(T), (uint32_t)rows};
  packer.add((const T*)p, stride, rows, (T*)(work + at));
  return {work + at, up_to(width, Group<T>::kN) * sizeof(T), (uint32_t)rows};
}

// The call's operands, packed where they have to be.
template <typename T>
void place(FfArgs& p, const FfCall& c, const FfWork& w, char* work, hipStream_t st) {
  Packer<T> packer(c.width);
  p.x = in_place<T>(c.x, c.x_stride, c.n, c.width, w.x, work, packer);
  p.w_gate = in_place<T>(c.w_gate, c.gate_stride, c.inner, c.width, w.w_gate, work, packer);
  p.w_up = in_place<T>(c.w_up, c.up_stride, c.inner, c.width, w.w_up, work, packer);
  packer.run(st);
}

template <typename T>
void run_few(const FfArgs& p, hipStream_t st) {
  const uint32_t blocks = (p.inner + 15) / 16;
  if (p.n <= 16)
    few_kernel<T, 1><<<blocks, kFewWaves * 64, 0, st>>>(p);
  else
    few_kernel<T, 2><<<blocks, kFewWaves * 64, 0, st>>>(p);
}

template <typename T, bool GRAD>
void run_ff(FfArgs& p, char* parts, hipStream_t st) {
  const Choice c = choose_ff<T>(p.n, p.width, p.inner);
  p.splits = c.splits;
  p.splits.parts = (float*)parts;
  with_shape<T, Flat>(c, [&](auto s) {
    typedef decltype(s) S;
    p.tiles_m = (p.n + S::BM - 1) / S::BM;
    p.tiles_n = (p.inner + S::BN / 2 - 1) / (S::BN / 2);
    const uint32_t tiles = p.tiles_m * p.tiles_n;
    if (c.splits.n > 1) {
      ff_part_kernel<S, T><<<tiles * c.splits.n, S::kLanes, 0, st>>>(p);
      ff_kernel<S, T, GRAD, true><<<tiles, S::kLanes, 0, st>>>(p);
    } else {
      ff_kernel<S, T, GRAD, false><<<tiles, S::kLanes, 0, st>>>(p);
    }
  });
}

template <class S>
uint32_t set_tiles(SumArgs& p) {
  p.tiles_m = (p.M + S::BM - 1) / S::BM;
  p.tiles_n = (p.N + S::BN - 1) / S::BN;
  return p.tiles_m * p.tiles_n;
}

template <typename T, typename O, bool ACROSS_A>
void run_sum(SumArgs& p, uint32_t outs, char* parts, hipStream_t st) {
  const Choice c = choose_sum<T>(p.M, p.N, p.K, std::max(1u, p.parts), outs);
  p.splits = c.splits;
  p.splits.parts = (float*)parts;
  with_shape<T, Small>(c, [&](auto s) {
    typedef decltype(s) S;
    const uint32_t tiles = set_tiles<S>(p);
    if (c.splits.n > 1) {
      sum_part_kernel<S, T, ACROSS_A><<<dim3(tiles * c.splits.n, outs), S::kLanes, 0, st>>>(p);
      sum_kernel<S, T, O, ACROSS_A, true><<<dim3(tiles, outs), S::kLanes, 0, st>>>(p);
    } else {
      sum_kernel<S, T, O, ACROSS_A, false><<<dim3(tiles, outs), S::kLanes, 0, st>>>(p);
    }
  });
}

// dx and both dW, in one launch (and dx's join) where dx takes small tiles, and dW such or middle ones and no splits; large
// ones of few steps are no better than middle ones (tile_ns).
template <typename T, typename O>
void run_sums(SumArgs& x, SumArgs& w, char* parts, hipStream_t st) {
  Choice cx = choose_sum<T>(x.M, x.N, x.K, x.parts, 1), cw = choose_sum<T>(w.M, w.N, w.K, w.parts, 2);
  if (cw.shape == 0 && steps_of<T>(w.K) * w.parts <= kFewSteps) cw.shape = 1;
  const uint64_t tiles = tiles_of(x.M, x.N, Small::BM, Small::BN);
  if (cx.shape != 2 || tiles * cx.splits.n > 2 * kCus || cw.shape == 0 || cw.splits.n > 1) {
    run_sum<T, T, false>(x, 1, parts, st);
    run_sum<T, O, true>(w, 2, parts, st);
    return;
  }
  x.splits = cx.splits, w.splits = cw.splits;
  x.splits.parts = (float*)parts;
  set_tiles<Small>(x);
  const auto run = [&](auto s, auto split) {
    typedef decltype(s) S;
    const uint32_t blocks = (uint32_t)tiles * x.splits.n + 2 * set_tiles<S>(w);
    sum_both_kernel<S, T, O, decltype(split)::value><<<blocks, S::kLanes, 0, st>>>(x, w);
  };
  const auto with_tiles = [&](auto split) { cw.shape == 1 ? run(Middle(), split) : run(Small(), split); };
  if (x.splits.n > 1) {
    with_tiles(std::true_type());
    sum_kernel<Small, T, T, false, true><<<(uint32_t)tiles, Small::kLanes, 0, st>>>(x);
  } else {
    with_tiles(std::false_type());
  }
}

int check_call(const FfCall& c, int act) {
  if (!known_type(c.type) || act < EC_ACT_SILU || act > EC_ACT_GELU_TANH) return EC_EINVAL;
  if (!c.width || !c.inner) return EC_EINVAL;
  if (c.x_stride < c.width || c.gate_stride < c.width || c.up_stride < c.width) return EC_EINVAL;
  if (!c.w_gate || !c.w_up || (c.n && !c.x)) return EC_EINVAL;
  if (c.n >= 1ull << 31 || c.width > kMostWidth || c.inner > kMostWidth) return EC_ERANGE;
  // a launch takes less than 2^32 lanes, whichever tiles are chosen
  constexpr uint64_t kMostTiles = 1u << 23;
  if (tiles_of(c.n, 2ull * c.inner, Middle::BM, Middle::BN) >= kMostTiles ||
      tiles_of(c.n, c.width, Middle::BM, Middle::BN) >= kMostTiles ||
      2 * tiles_of(c.inner, c.width, Middle::BM, Middle::BN) >= kMostTiles)
    return EC_ERANGE;
  return EC_OK;
}

int check_work(const void* work, uint64_t have, uint64_t need) {
  if (have < need || (need && !work)) return EC_EINVAL;
  return (uintptr_t)work & 15u ? EC_EALIGN : EC_OK;
}

}  // namespace
}  // namespace ec

using namespace ec;

extern "C" {

uint64_t ec_gated_ff_workspace(const void* d_x, uint64_t x_stride, const void* d_gate, uint64_t gate_stride,
                               const void* d_up, uint64_t up_stride, int type, uint64_t n, uint32_t width,
                               uint32_t inner, int grad) {
  const FfCall c = {d_x, d_gate, d_up, x_stride, gate_stride, up_stride, n, width, inner, type};
  return check_call(c, EC_ACT_SILU) == EC_OK ? ff_work(c, grad != 0).total : 0;
}

int ec_gated_ff(const void* d_x, uint64_t x_stride, const void* d_gate, uint64_t gate_stride,
                const void* d_up, uint64_t up_stride, int type, uint64_t n, uint32_t width,
                uint32_t inner, int activation, void* d_h, uint64_t h_stride, void* d_work,
                uint64_t work_bytes, ec_stream_t stream) {
  const FfCall c = {d_x, d_gate, d_up, x_stride, gate_stride, up_stride, n, width, inner, type};
  if (const int st = check_call(c, activation)) return st;
  if (h_stride < inner || (n && !d_h)) return EC_EINVAL;
  const FfWork w = ff_work(c, false);
  if (const int st = check_work(d_work, work_bytes, w.total)) return st;
  if (!n) return EC_OK;
  const auto st = (hipStream_t)stream;
  return with_type(type, [&](auto t) {
    typedef decltype(t) T;
    char* work = (char*)d_work;
    FfArgs p = {};
    place<T>(p, c, w, work, st);
    p.n = (uint32_t)n, p.width = width, p.inner = inner, p.act = (uint32_t)activation;
    p.h = (char*)d_h, p.h_stride = h_stride;
    if (n <= kFewForward)
      run_few<T>(p, st);
    else
      run_ff<T, false>(p, work + w.parts, st);
    return launched();
  });
}

int ec_gated_ff_grad(const void* d_dh, uint64_t dh_stride, const void* d_x, uint64_t x_stride,
                     const void* d_gate, uint64_t gate_stride, const void* d_up, uint64_t up_stride,
                     int type, uint64_t n, uint32_t width, uint32_t inner, int activation, void* d_dx,
                     uint64_t dx_stride, void* d_dgate, uint64_t dgate_stride, void* d_dup,
                     uint64_t dup_stride, int grad_type, int accumulate, void* d_work,
                     uint64_t work_bytes, ec_stream_t stream) {
  const FfCall c = {d_x, d_gate, d_up, x_stride, gate_stride, up_stride, n, width, inner, type};
  if (const int st = check_call(c, activation)) return st;
  if (dh_stride < inner || (n && !d_dh) || (d_dx && dx_stride < width)) return EC_EINVAL;
  if (!d_dgate != !d_dup || (n && !d_dx && !d_dgate)) return EC_EINVAL;   // (a dx of no rows may have no address)
  if (d_dgate && (dgate_stride < width || dup_stride < width)) return EC_EINVAL;
  if (grad_type != EC_F32 && grad_type != type) return EC_EINVAL;
  const FfWork w = ff_work(c, true);
  if (const int st = check_work(d_work, work_bytes, w.total)) return st;
  if (!n && (!d_dgate || accumulate)) return EC_OK;
  const auto st = (hipStream_t)stream;
  return with_type(type, [&](auto t) {
    typedef decltype(t) T;
    char* work = (char*)d_work;
    FfArgs p = {};
    p.n = (uint32_t)n, p.width = width, p.inner = inner, p.act = (uint32_t)activation;
    p.padded = (uint32_t)up_to(inner, 8);
    const uint64_t d_row = 2ull * p.padded;
    if (n) {
      place<T>(p, c, w, work, st);
      p.dh = (const char*)d_dh, p.dh_stride = dh_stride;
      p.d = work + w.d;
      p.low = w.low ? n * d_row : 0;
      run_ff<T, true>(p, work + w.parts, st);
    }
    const uint64_t ld = d_row * sizeof(T), half = p.padded * sizeof(T), low = p.low * sizeof(T);
    SumArgs x = {}, s = {};   // dx, dW
    if (d_dx && n) {
      x.parts = p.low ? 4 : 2;
      for (uint32_t i = 0; i < x.parts; ++i) {
        x.a[i] = {p.d + i % 2 * half + i / 2 * low, ld, p.n};
        x.b[i] = i % 2 ? p.w_up : p.w_gate;
        x.b[i].rows = width;
      }
      x.K = inner, x.M = p.n, x.N = width;
      x.out[0] = (char*)d_dx, x.out_stride[0] = dx_stride;
    }
    if (d_dgate) {
      s.parts = !n ? 0 : p.low ? 2 : 1;
      for (uint32_t i = 0; i < s.parts; ++i) {
        s.a[i] = {p.d + i * low, ld, inner};
        s.b[i] = p.x;
        s.b[i].rows = width;
      }
      s.a_step = half, s.accumulate = accumulate;
      s.K = p.n, s.M = inner, s.N = width;
      s.out[0] = (char*)d_dgate, s.out_stride[0] = dgate_stride;
      s.out[1] = (char*)d_dup, s.out_stride[1] = dup_stride;
    }
    char* parts = work + w.parts;
    const auto run = [&](auto o) {
      typedef decltype(o) O;
      x.parts ? run_sums<T, O>(x, s, parts, st) : run_sum<T, O, true>(s, 2, parts, st);
    };
    if (!d_dgate)
      run_sum<T, T, false>(x, 1, parts, st);
    else
      grad_type == EC_F32 ? run(float()) : run(T());
    return launched();
  });
}

}  // extern "C"
