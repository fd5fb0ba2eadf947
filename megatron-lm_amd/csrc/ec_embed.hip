// ec_embed.hip — ec_embed and ec_embed_grad: rows of an embedding table by
// token, and the table's gradient by sorted tokens.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "ec_types.h"

namespace ec {
namespace {

constexpr int kLanes = 64;
constexpr uint32_t kMaxHidden = 1u << 20;

// The row of the slice that token i asks for, or -1.
__device__ __forceinline__ int64_t row_of(const void* tokens, int token_bytes, uint32_t i,
                                          int64_t start, uint64_t vocab) {
  const int64_t t = token_bytes == 8 ? gp((const int64_t*)tokens)[i]
                                     : (int64_t)gp((const int32_t*)tokens)[i];
  // any 64-bit start and t: where t >= start, their difference modulo 2^64 is right
  const uint64_t row = (uint64_t)t - (uint64_t)start;
  return t >= start && row < vocab ? (int64_t)row : -1;
}

// ------------------------------------------------------------------ lookup --
// A wave copies kGroups groups (16 bytes each) per lane of one row, or, of rows
// that are shorter, 2^shift lanes take a row and the wave 64 >> shift of them.
// The last group of a row that is no multiple of a group long starts early,
// so that it ends with the row: two lanes then write some elements, the same
// values.  Rows of less than a group go element by element.
struct EmbedArgs {
  const void* tokens;
  const void* table;
  void* out;
  uint64_t vocab, table_stride;
  int64_t start;
  uint32_t n, hidden, groups;
  int token_bytes, shift;
  float scale;
};

constexpr int kEmbedGroups = 4;
constexpr int kEmbedWaves = 4;

template <typename T>
__global__ void __launch_bounds__(kEmbedWaves * kLanes) embed_kernel(const EmbedArgs a) {
  typedef Group<T> G;
  const uint32_t lane = threadIdx.x % kLanes, wave = threadIdx.x / kLanes;
  const uint32_t per_row = 1u << a.shift;
  const uint64_t i = ((uint64_t)blockIdx.x * kEmbedWaves + wave) * (kLanes >> a.shift) + (lane >> a.shift);
  if (i >= a.n) return;
  const uint32_t first = blockIdx.y * (per_row * kEmbedGroups) + (lane & (per_row - 1));
  const int64_t row = row_of(a.tokens, a.token_bytes, (uint32_t)i, a.start, a.vocab);
  T* out = (T*)a.out + i * a.hidden;
  const T* src = (const T*)a.table + (row < 0 ? 0 : (uint64_t)row * a.table_stride);
  if (a.hidden < (uint32_t)G::kN) {
    if (first == 0)
      for (uint32_t j = 0; j < a.hidden; ++j)
        gp(out)[j] = row < 0 ? (T)0.0f : (T)((float)gp(src)[j] * a.scale);
    return;
  }
  typename G::vec v[kEmbedGroups];
  uint32_t at[kEmbedGroups];
#pragma unroll
  for (int u = 0; u < kEmbedGroups; ++u) {
    const uint32_t g = first + u * per_row;
    at[u] = min(g * G::kN, a.hidden - G::kN);
    if (g < a.groups && row >= 0) v[u] = load_group<T, false>(src + at[u]);
  }
#pragma unroll
  for (int u = 0; u < kEmbedGroups; ++u) {
    if (first + u * per_row >= a.groups) continue;
    typename G::wide w = {};
    if (row >= 0) w = widen<T>(v[u]) * a.scale;
    store_wide<T, false>(out + at[u], w);
  }
}

// -------------------------------------------------------------------- sort --
// The tokens' rows in ascending order, equal ones by position, as (row,
// position) pairs: a least-significant-digit radix sort in digits of at most 10
// bits (two of 8 for a vocabulary of 50304).  Tokens outside the slice sort as row
// `vocab`, behind all others.  A pass is two launches: each workgroup counts
// the digits of its tile; then each sums the counts of the tiles before its own
// (and of the smaller digits) and scatters its tile.  The place of an item
// within its tile is its rank among the wave's items of the same digit (ballots
// find the equal lanes) plus the counts of the waves before it, so the order is
// the input's and no atomic decides it.
constexpr int kSortLanes = 256;
constexpr int kSortWaves = kSortLanes / kLanes;
constexpr int kSortSteps = 16;                       // items per lane
constexpr uint32_t kSortTile = kSortLanes * kSortSteps;
constexpr int kMaxDigit = 10;

struct SortArgs {
  const void* tokens;      // the first pass's input (null: the pairs)
  const uint32_t* keys;
  const uint32_t* pos;
  uint32_t* keys_out;
  uint32_t* pos_out;
  uint32_t* counts;        // [tiles][2^bits]
  int64_t start;
  uint64_t vocab;
  uint32_t n, tiles;
  int token_bytes, shift, bits;
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, uint32_t i) {
  if (!a.tokens) return gp(a.keys)[i];
  const int64_t row = row_of(a.tokens, a.token_bytes, i, a.start, a.vocab);
  return row < 0 ? (uint32_t)a.vocab : (uint32_t)row;
}

__global__ void __launch_bounds__(kSortLanes) sort_count_kernel(const SortArgs a) {
  __shared__ uint32_t count[1 << kMaxDigit];
  const uint32_t bins = 1u << a.bits;
  for (uint32_t b = threadIdx.x; b < bins; b += kSortLanes) count[b] = 0;
  __syncthreads();
  const uint32_t base = blockIdx.x * kSortTile;
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s) {
    const uint32_t i = base + s * kSortLanes + threadIdx.x;
    if (i < a.n) atomicAdd(&count[(sort_key(a, i) >> a.shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < bins; b += kSortLanes)
    gp(a.counts)[(uint64_t)blockIdx.x * bins + b] = count[b];
}

__global__ void __launch_bounds__(kSortLanes) sort_scatter_kernel(const SortArgs a) {
  __shared__ uint32_t count[kSortWaves][1 << kMaxDigit];
  __shared__ uint32_t total[kSortLanes];
  const uint32_t bins = 1u << a.bits, t = threadIdx.x, lane = t % kLanes, wave = t / kLanes;
  for (uint32_t b = t; b < kSortWaves * bins; b += kSortLanes) count[b >> a.bits][b & (bins - 1)] = 0;
  __syncthreads();

  // ranks within the wave; the wave's items are 64 consecutive ones per step
  const uint32_t base = blockIdx.x * kSortTile + wave * (kLanes * kSortSteps) + lane;
  uint32_t key[kSortSteps], rank[kSortSteps];
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s) {
    const uint32_t i = base + s * kLanes;
    key[s] = i < a.n ? sort_key(a, i) : 0xffffffffu;
  }
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s) {
    const bool in = base + s * kLanes < a.n;
    const uint32_t digit = (key[s] >> a.shift) & (bins - 1);
    uint64_t same = __ballot(in);
    for (int b = 0; b < a.bits; ++b) {
      const uint64_t ones = __ballot((digit >> b) & 1u);
      same &= (digit >> b) & 1u ? ones : ~ones;
    }
    const uint32_t before = __popcll(same & ((1ull << lane) - 1));
    uint32_t seen = 0;
    if (in) seen = count[wave][digit];
    rank[s] = seen + before;
    // the wave's lanes have read the count before the first of them writes it,
    // and it is written before the next step reads it: LDS operations of one wave
    // complete in order, and the fences keep the compiler to it
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (in && before == 0) count[wave][digit] = seen + (uint32_t)__popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();

  // where each digit of this tile begins: lane t owns the digits [t * per, ...)
  const uint32_t per = (bins + kSortLanes - 1) / kSortLanes, d0 = t * per;
  uint32_t mine = 0, here[(1 << kMaxDigit) / kSortLanes], all[(1 << kMaxDigit) / kSortLanes];
#pragma unroll
  for (uint32_t j = 0; j < (1 << kMaxDigit) / kSortLanes; ++j) {
    here[j] = all[j] = 0;
    if (j >= per || d0 + j >= bins) continue;
    uint32_t before = 0, sum = 0;
    for (uint32_t b = 0; b < a.tiles; ++b) {
      const uint32_t c = gp((const uint32_t*)a.counts)[(uint64_t)b * bins + d0 + j];
      before += b < blockIdx.x ? c : 0;
      sum += c;
    }
    here[j] = before;
    all[j] = sum;
    mine += sum;
  }
  total[t] = mine;
  __syncthreads();
  for (uint32_t o = 1; o < kSortLanes; o <<= 1) {   // inclusive scan
    const uint32_t v = t >= o ? total[t - o] : 0;
    __syncthreads();
    total[t] += v;
    __syncthreads();
  }
  uint32_t begin = total[t] - mine;
#pragma unroll
  for (uint32_t j = 0; j < (1 << kMaxDigit) / kSortLanes; ++j) {
    if (j >= per || d0 + j >= bins) continue;
    uint32_t at = begin + here[j];
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = count[w][d0 + j];
      count[w][d0 + j] = at;
      at += c;
    }
    begin += all[j];
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s) {
    const uint32_t i = base + s * kLanes;
    if (i >= a.n) continue;
    const uint32_t to = count[wave][(key[s] >> a.shift) & (bins - 1)] + rank[s];
    gp(a.keys_out)[to] = key[s];
    gp(a.pos_out)[to] = a.tokens ? i : gp(a.pos)[i];
  }
}

// ------------------------------------------------------------ segment sums --
// The sorted pairs in tiles of kTile, each summed by one wave for each 64
// groups of columns: the rows' loads in batches of kBatch, the running sum in
// fp32 registers, put out where the row changes.  A run of equal rows that lies
// within its tile goes to the gradient; one that begins before the tile, or
// goes on behind it, leaves its part in `parts` (slot 0: a run from before; slot
// 1: one that begins here), and join_kernel adds the parts of a run in order.
// The split does not look at the run's length, so a token on a tenth of all
// positions costs what others do.
constexpr uint32_t kTile = 32;
constexpr int kBatch = 8;
constexpr int kSumWaves = 4;

struct SumArgs {
  const uint32_t* keys;
  const uint32_t* pos;
  const void* dout;
  void* grad;
  float* parts;            // [tiles][2][hidden]
  uint64_t dout_stride, grad_stride, vocab;
  uint32_t n, tiles, hidden, slabs, sum_blocks;
  int accumulate;
  float scale;
};

// Elements [c, c + N) of a row of `hidden`, N of them or what is left.
template <typename T, int N>
__device__ __forceinline__ void put_row(T* row, uint32_t c, uint32_t hidden, const float* sum,
                                        float scale, bool add) {
  typedef Group<T> G;
#pragma unroll
  for (int h = 0; h < N; h += G::kN) {
    if (c + h + G::kN <= hidden) {
      typename G::wide w;
#pragma unroll
      for (int e = 0; e < G::kN; ++e) w[e] = sum[h + e] * scale;
      if (add) w += widen<T>(load_group<T, false>(row + c + h));
      store_wide<T, true>(row + c + h, w);
    } else {
#pragma unroll
      for (int e = 0; e < G::kN; ++e)
        if (c + h + e < hidden) {
          float v = sum[h + e] * scale;
          if (add) v += (float)gp(row)[c + h + e];
          gp(row)[c + h + e] = (T)v;
        }
    }
  }
}

// The rows of tokens that do not occur: a wave looks kZeroRows rows up among the
// sorted keys, one per lane, and writes the zeros of those that are missing.
constexpr uint32_t kZeroRows = 16;

template <typename O>
__device__ __forceinline__ void zero_rows(const SumArgs& a, uint64_t first) {
  typedef Group<O> G;
  const uint32_t lane = threadIdx.x % kLanes;
  const uint64_t row = first + lane;
  bool missing = false;
  if (lane < kZeroRows && row < a.vocab) {
    uint32_t lo = 0, hi = a.n;   // the first key >= row
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (gp(a.keys)[mid] < (uint32_t)row)
        lo = mid + 1;
      else
        hi = mid;
    }
    missing = lo == a.n || gp(a.keys)[lo] != (uint32_t)row;
  }
  const uint64_t todo = __ballot(missing);
  const typename G::wide zero = {};
  for (uint32_t r = 0; r < kZeroRows; ++r) {
    if (!((todo >> r) & 1u)) continue;
    O* out = (O*)a.grad + (first + r) * a.grad_stride;
    for (uint32_t c = lane * G::kN; c < a.hidden; c += kLanes * G::kN) {
      if (c + G::kN <= a.hidden)
        store_wide<O, true>(out + c, zero);
      else
        for (uint32_t e = c; e < a.hidden; ++e) gp(out)[e] = (O)0.0f;
    }
  }
}

template <typename T, typename O>
__global__ void __launch_bounds__(kSumWaves * kLanes) sum_kernel(const SumArgs a) {
  typedef Group<T> G;
  constexpr int N = G::kN;
  const uint32_t lane = threadIdx.x % kLanes;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
  if (blockIdx.x >= a.sum_blocks) {
    zero_rows<O>(a, ((uint64_t)(blockIdx.x - a.sum_blocks) * kSumWaves + wave) * kZeroRows);
    return;
  }
  const uint64_t job = (uint64_t)blockIdx.x * kSumWaves + wave;
  const uint32_t tile = (uint32_t)(job / a.slabs), slab = (uint32_t)(job % a.slabs);
  if (tile >= a.tiles) return;
  const uint32_t c = (slab * kLanes + lane) * N;   // this lane's columns
  const uint32_t first = tile * kTile, len = min(kTile, a.n - first);

  // lane l holds pair l of the tile, and its neighbours' keys the tile's ends
  uint32_t key = 0, pos = 0;
  if (lane < len) {
    key = gp(a.keys)[first + lane];
    pos = gp(a.pos)[first + lane];
  }
  const uint32_t none = 0xffffffffu;
  const uint32_t prev = first ? gp(a.keys)[first - 1] : none;
  const uint32_t next = first + len < a.n ? gp(a.keys)[first + len] : none;
  const uint32_t vocab = (uint32_t)a.vocab;

  float sum[N] = {};
  uint32_t run = __builtin_amdgcn_readlane(key, 0);
  bool from_before = run == prev;
  for (uint32_t b = 0; b < len; b += kBatch) {
    typename G::vec v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      v[u] = {};
      const uint32_t k = __builtin_amdgcn_readlane(key, (b + u) & 63);
      const uint32_t p = __builtin_amdgcn_readlane(pos, (b + u) & 63);
      if (b + u < len && k < vocab) {
        const T* src = (const T*)a.dout + (uint64_t)p * a.dout_stride + c;
        if (c + N <= a.hidden)
          v[u] = load_group<T, true>(src);
        else
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (c + e < a.hidden) v[u][e] = gp(src)[e];
      }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (b + u >= len) break;
      const uint32_t k = __builtin_amdgcn_readlane(key, (b + u) & 63);
      if (k != run) {   // the run ended within the tile
        if (run < vocab) {
          if (from_before) {
            float* part = a.parts + (uint64_t)tile * 2 * a.hidden;
            put_row<float, N>(part, c, a.hidden, sum, 1.0f, false);
          } else {
            put_row<O, N>((O*)a.grad + (uint64_t)run * a.grad_stride, c, a.hidden, sum, a.scale,
                          a.accumulate);
          }
        }
        run = k;
        from_before = false;
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = 0.0f;
      }
      const typename G::wide w = widen<T>(v[u]);
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] += w[e];
    }
  }
  if (run >= vocab) return;
  if (from_before || run == next) {
    float* part = a.parts + ((uint64_t)tile * 2 + (from_before ? 0 : 1)) * a.hidden;
    put_row<float, N>(part, c, a.hidden, sum, 1.0f, false);
  } else {
    put_row<O, N>((O*)a.grad + (uint64_t)run * a.grad_stride, c, a.hidden, sum, a.scale,
                  a.accumulate);
  }
}

// A workgroup for each tile's last run and 256 columns, if the run begins in the
// tile and goes on behind it: its waves share the tiles of the run, in order,
// and their sums are added in order.
constexpr int kJoinWaves = 8;
constexpr int kJoinBatch = 8;

template <typename O>
__global__ void __launch_bounds__(kJoinWaves * kLanes) join_kernel(const SumArgs a) {
  typedef Group<float> G;
  const uint32_t tile = blockIdx.x, last = tile * kTile + kTile - 1;
  if (last + 1 >= a.n) return;
  const uint32_t run = gp(a.keys)[last];
  if (run >= a.vocab || gp(a.keys)[last + 1] != run) return;
  const uint32_t first = tile * kTile;
  if (gp(a.keys)[first] == run && first && gp(a.keys)[first - 1] == run) return;
  uint32_t lo = last + 1, hi = a.n;   // the first key > run
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (gp(a.keys)[mid] <= run)
      lo = mid + 1;
    else
      hi = mid;
  }
  // the run's parts: slot 1 of `tile`, slot 0 of the tiles up to that of its end
  const uint32_t parts = (lo - 1) / kTile - tile + 1;
  const uint32_t lane = threadIdx.x % kLanes, wave = threadIdx.x / kLanes;
  const uint32_t c = (blockIdx.y * kLanes + lane) * G::kN;
  const uint32_t per = (parts + kJoinWaves - 1) / kJoinWaves;
  const uint32_t from = min(parts, wave * per), to = min(parts, from + per);
  float sum[G::kN] = {};
  for (uint32_t p = from; p < to; p += kJoinBatch) {
    G::vec v[kJoinBatch];
#pragma unroll
    for (int u = 0; u < kJoinBatch; ++u) {
      v[u] = {};
      if (p + u >= to) continue;
      const uint64_t slot = (uint64_t)(tile + p + u) * 2 + (p + u == 0 ? 1 : 0);
      const float* src = a.parts + slot * a.hidden + c;
      if (c + G::kN <= a.hidden)
        v[u] = load_group<float, true>(src);
      else
#pragma unroll
        for (int e = 0; e < G::kN; ++e)
          if (c + e < a.hidden) v[u][e] = gp(src)[e];
    }
#pragma unroll
    for (int u = 0; u < kJoinBatch; ++u)
#pragma unroll
      for (int e = 0; e < G::kN; ++e) sum[e] += v[u][e];
  }
  __shared__ float shared[kJoinWaves][kLanes][G::kN];
#pragma unroll
  for (int e = 0; e < G::kN; ++e) shared[wave][lane][e] = sum[e];
  __syncthreads();
  if (wave) return;
  for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
    for (int e = 0; e < G::kN; ++e) sum[e] += shared[w][lane][e];
  O* row = (O*)a.grad + (uint64_t)run * a.grad_stride;
#pragma unroll
  for (int e = 0; e < G::kN; ++e)
    if (c + e < a.hidden) {
      float v = sum[e] * a.scale;
      if (a.accumulate) v += (float)gp(row)[c + e];
      gp(row)[c + e] = (O)v;
    }
}

// ---------------------------------------------------------- host launchers --

int bits_of(uint64_t v) {   // of the largest key
  int b = 1;
  while (b < 32 && (v >> b)) ++b;
  return b;
}

constexpr uint64_t up16(uint64_t v) { return (v + 15) / 16 * 16; }

struct Work {
  uint64_t keys[2], pos[2], counts, parts, bytes;
  uint32_t sort_tiles, sum_tiles;
  int passes, bits;
};

Work work_of(uint64_t n, uint64_t vocab, uint32_t hidden) {
  Work w;
  const int all = bits_of(vocab);
  w.passes = (all + kMaxDigit - 1) / kMaxDigit;
  w.bits = (all + w.passes - 1) / w.passes;
  w.sort_tiles = (uint32_t)((n + kSortTile - 1) / kSortTile);
  w.sum_tiles = (uint32_t)((n + kTile - 1) / kTile);
  uint64_t at = 0;
  const auto take = [&at](uint64_t bytes) {
    const uint64_t here = at;
    at += up16(bytes);
    return here;
  };
  for (int i = 0; i < 2; ++i) w.keys[i] = take(4 * n);
  for (int i = 0; i < 2; ++i) w.pos[i] = take(4 * n);
  w.counts = take(4ull * w.sort_tiles << w.bits);
  w.parts = take(8ull * w.sum_tiles * hidden);
  w.bytes = at;
  return w;
}

int check_tokens(const void* tokens, int token_bytes, uint64_t n, uint32_t hidden) {
  if (token_bytes != 4 && token_bytes != 8) return EC_EINVAL;
  if (n >= (1ull << 31) || hidden > kMaxHidden) return EC_ERANGE;
  if (n && !tokens) return EC_EINVAL;
  return EC_OK;
}

}  // namespace
}  // namespace ec

using namespace ec;

extern "C" {

int ec_embed(const void* d_tokens, int token_bytes, uint64_t n, const void* d_table, int type,
             uint64_t vocab, uint32_t hidden, uint64_t table_stride, int64_t vocab_start,
             float scale, void* d_out, ec_stream_t stream) {
  if (!known_type(type) || !std::isfinite(scale)) return EC_EINVAL;
  if (const int st = check_tokens(d_tokens, token_bytes, n, hidden)) return st;
  if (!n || !hidden) return EC_OK;
  if (!d_out || (vocab && (!d_table || table_stride < hidden))) return EC_EINVAL;
  EmbedArgs a = {d_tokens, d_table, d_out, vocab, table_stride, vocab_start,
                 (uint32_t)n, hidden, 0, token_bytes, 0, scale};
  const uint32_t per_group = 16 / type_bytes(type);
  a.groups = (hidden + per_group - 1) / per_group;
  while (a.shift < 6 && (1u << a.shift) * kEmbedGroups < a.groups) ++a.shift;
  const uint32_t rows = kEmbedWaves * (kLanes >> a.shift), wide = kEmbedGroups << a.shift;
  const dim3 grid((a.n + rows - 1) / rows, (a.groups + wide - 1) / wide);
  return with_type(type, [&](auto t) {
    embed_kernel<decltype(t)><<<grid, kEmbedWaves * kLanes, 0, (hipStream_t)stream>>>(a);
    return launched();
  });
}

uint64_t ec_embed_grad_workspace(uint64_t n, uint64_t vocab, uint32_t hidden) {
  if (n >= (1ull << 31) || vocab >= (1ull << 31) || hidden > kMaxHidden) return 0;
  return work_of(n, vocab, hidden).bytes;
}

int ec_embed_grad(const void* d_tokens, int token_bytes, uint64_t n, const void* d_dout, int type,
                  uint64_t dout_stride, uint64_t vocab, uint32_t hidden, int64_t vocab_start,
                  float scale, void* d_grad, int grad_type, uint64_t grad_stride, int accumulate,
                  void* d_work, uint64_t work_bytes, ec_stream_t stream) {
  if (!known_type(type) || !std::isfinite(scale)) return EC_EINVAL;
  if (grad_type != type && grad_type != EC_F32) return EC_EINVAL;
  if (const int st = check_tokens(d_tokens, token_bytes, n, hidden)) return st;
  if (vocab >= (1ull << 31)) return EC_ERANGE;
  if (!vocab || !hidden || (!n && accumulate)) return EC_OK;
  if (!d_grad || grad_stride < hidden) return EC_EINVAL;
  if (n && (!d_dout || dout_stride < hidden)) return EC_EINVAL;
  const Work w = work_of(n, vocab, hidden);
  if (work_bytes < w.bytes || (w.bytes && !d_work)) return EC_EINVAL;
  if ((uintptr_t)d_work & 15u) return EC_EALIGN;
  uint8_t* work = (uint8_t*)d_work;
  const hipStream_t st = (hipStream_t)stream;

  SortArgs s = {};
  s.start = vocab_start;
  s.vocab = vocab;
  s.n = (uint32_t)n;
  s.tiles = w.sort_tiles;
  s.token_bytes = token_bytes;
  s.bits = w.bits;
  s.counts = (uint32_t*)(work + w.counts);
  for (int p = 0; n && p < w.passes; ++p) {
    s.tokens = p ? nullptr : d_tokens;
    s.keys = (const uint32_t*)(work + w.keys[(p + 1) & 1]);
    s.pos = (const uint32_t*)(work + w.pos[(p + 1) & 1]);
    s.keys_out = (uint32_t*)(work + w.keys[p & 1]);
    s.pos_out = (uint32_t*)(work + w.pos[p & 1]);
    s.shift = p * w.bits;
    sort_count_kernel<<<s.tiles, kSortLanes, 0, st>>>(s);
    sort_scatter_kernel<<<s.tiles, kSortLanes, 0, st>>>(s);
  }

  SumArgs a = {};
  a.keys = (const uint32_t*)(work + w.keys[(w.passes + 1) & 1]);
  a.pos = (const uint32_t*)(work + w.pos[(w.passes + 1) & 1]);
  a.dout = d_dout;
  a.grad = d_grad;
  a.parts = (float*)(work + w.parts);
  a.dout_stride = dout_stride;
  a.grad_stride = grad_stride;
  a.vocab = vocab;
  a.n = (uint32_t)n;
  a.tiles = w.sum_tiles;
  a.hidden = hidden;
  a.accumulate = accumulate != 0;
  a.scale = scale;
  const uint32_t per_group = 16 / type_bytes(type);
  a.slabs = (hidden + per_group * kLanes - 1) / (per_group * kLanes);
  const uint64_t sum_blocks = ((uint64_t)a.tiles * a.slabs + kSumWaves - 1) / kSumWaves;
  const uint64_t per_block = kZeroRows * kSumWaves;
  const uint64_t blocks = sum_blocks + (accumulate ? 0 : (vocab + per_block - 1) / per_block);
  if (blocks > 0x7fffffffull) return EC_ERANGE;
  a.sum_blocks = (uint32_t)sum_blocks;
  const dim3 join(a.tiles, (hidden + kLanes * 4 - 1) / (kLanes * 4));
  const auto go = [&](auto t, auto o) {
    typedef decltype(t) T;
    typedef decltype(o) O;
    if (blocks) sum_kernel<T, O><<<(uint32_t)blocks, kSumWaves * kLanes, 0, st>>>(a);
    if (a.tiles > 1) join_kernel<O><<<join, kJoinWaves * kLanes, 0, st>>>(a);
    return launched();
  };
  return with_type(type, [&](auto t) {
    return grad_type == EC_F32 ? go(t, float()) : go(t, t);
  });
}

}  // extern "C"
