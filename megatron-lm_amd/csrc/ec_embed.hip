// ec_embed.hip — ec_embed and ec_embed_grad: rows of an embedding table by
// token, and the table's gradient by sorted tokens.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "ec_types.h"
#include "fastdiv.h"
#include "routes.h"

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
// A wave copies kEmbedGroups groups (16 bytes each) per lane of one row, or, of
// rows that are shorter, 2^shift lanes take a row and the wave 64 >> shift of them.
// The last group of a row that is no multiple of a group long starts early,
// so that it ends with the row: two lanes then write some elements, the same
// values.  Rows of less than a group go element by element.
//
// Bound by memory: 32768 tokens of 2048 bf16 in 32 us, 134 MB written and 77 MB read (each
// XCD reads the rows of its own tokens: 6.6 TB/s).  One, two or eight groups a lane took
// 51, 49 and 44 us where four took 42 (cached stores, four tables in turn): the token's load is
// waited for once.
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
// Results of at least this many bytes, in rows of at least a KiB, are streamed past the
// caches (a call, four tables in turn): 32768 rows of 2048 bf16 40.5 -> 37.0 us, of 2047 48.2 ->
// 40.1, 65536 of 512 21.6 -> 17.2, 16384 of 4096 fp32 78.2 -> 70.7; but 131072 of 33 fp16, whose
// rows share lines, 6.7 -> 10.7.
constexpr uint64_t kEmbedStream = 64u << 20;
constexpr uint32_t kEmbedStreamGroups = 64;

template <typename T, bool STREAM>
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
  // (groups behind the row's end read and write its last one)
  typename G::vec v[kEmbedGroups];
  uint32_t at[kEmbedGroups];
#pragma unroll
  for (int u = 0; u < kEmbedGroups; ++u) {
    at[u] = min((first + u * per_row) * G::kN, a.hidden - G::kN);
    v[u] = {};
  }
  if (row >= 0) {
#pragma unroll
    for (int u = 0; u < kEmbedGroups; ++u) v[u] = load_group<T, false>(src + at[u]);
  }
#pragma unroll
  for (int u = 0; u < kEmbedGroups; ++u)
    if (first + u * per_row < a.groups)
      store_wide<T, STREAM>(out + at[u], widen<T>(v[u]) * a.scale);
}

// ------------------------------------------------------------------- zeros --
// The rows of tokens that do not occur, which the gradient has most of, need no
// sorted tokens: workgroups that write zeros ride along in the sort's launches, which
// leave the memory idle, and in the sums' launch.  Each takes the rows of 32 to 256 KiB and learns
// which of them occur from bits that the sort's first launch collected (one bit per row
// and span of the sort's tokens), or, for few tokens, from the tokens themselves.
enum ZeroMode : int { kZeroSeen, kZeroScan, kZeroAll };

struct Tokens {
  const void* tokens;
  int64_t start;
  uint64_t vocab;
  uint32_t n;
  int bytes;

  __device__ __forceinline__ int64_t row(uint32_t i) const {
    return row_of(tokens, bytes, i, start, vocab);
  }
};

struct ZeroArgs {
  uint8_t* grad;
  const uint32_t* seen;      // [spans][words]
  uint64_t stride;           // of the rows, in bytes
  FastDiv by_row;            // by row_bytes
  uint32_t row_bytes, words, spans;
  int shift;                 // a workgroup's rows: 32 << shift
  uint32_t first, blocks;    // workgroups before this launch's, and in it
  int mode;
};

// Bytes of a workgroup's rows, about: a 256th of the gradient's within these bounds, and at
// most 2048 rows.
constexpr uint64_t kLeastSpan = 32u << 10, kMostSpan = 256u << 10, kZeroSpans = 256;
constexpr int kZeroShift = 6;
// Rows of this many bytes and more are written one by a wave.  Narrower ones would leave most
// of a wave idle, and share lines: 67 tokens, 116317 x 64 fp32, 24 us by rows, 17 flat;
// 65536 tokens, 50304 x 2048, 134 and 162 (the flat form looks each 16 bytes' row up).
constexpr uint32_t kWideRow = 1024;

typedef uint32_t __attribute__((ext_vector_type(4))) zero16_t;
__device__ __forceinline__ void put_zeros(uint8_t* at) {
  const zero16_t zero = {};
  __builtin_nontemporal_store(zero, (global<zero16_t>*)(uintptr_t)at);
}
__device__ __forceinline__ void put_zero(uint8_t* at) { *gp((uint16_t*)at) = 0; }

// The rows of a span that lie back to back, as one range of memory: 16 bytes at a time at
// aligned addresses, where no row in them occurs, else (and at the range's ends) two.
__device__ __forceinline__ void zero_flat(const ZeroArgs& z, const uint32_t* bits, uint8_t* span,
                                          uint32_t rows) {
  const uint32_t bytes = rows * z.row_bytes;
  const auto occurs = [&](uint32_t r) { return (bits[r / 32] >> (r % 32)) & 1u; };
  const auto single = [&](uint32_t off) {
    if (!occurs(fast_div(off, z.by_row))) put_zero(span + off);
  };
  const uint32_t lead = min(bytes, (uint32_t)(-(uintptr_t)span % 16));
  const uint32_t chunks = (bytes - lead) / 16, behind = lead + chunks * 16;
  if (threadIdx.x < 8) {
    if (threadIdx.x * 2 < lead) single(threadIdx.x * 2);
    if (behind + threadIdx.x * 2 < bytes) single(behind + threadIdx.x * 2);
  }
  for (uint32_t i = threadIdx.x; i < chunks; i += blockDim.x) {
    const uint32_t off = lead + i * 16;
    const uint32_t r0 = fast_div(off, z.by_row), r1 = fast_div(off + 15, z.by_row);
    if (r1 - r0 <= 1 && !occurs(r0) && !occurs(r1))
      put_zeros(span + off);
    else if (r1 != r0 || !occurs(r0))
      for (uint32_t e = 0; e < 16; e += 2) single(off + e);
  }
}

// One row by a wave.
__device__ __forceinline__ void zero_row(uint8_t* row, uint32_t bytes) {
  const uint32_t lane = threadIdx.x % kLanes;
  const uint32_t lead = min(bytes, (uint32_t)(-(uintptr_t)row % 16));
  const uint32_t chunks = (bytes - lead) / 16, behind = lead + chunks * 16;
  if (lane * 2 < lead) put_zero(row + lane * 2);
  if (behind + lane * 2 < bytes) put_zero(row + behind + lane * 2);
  for (uint32_t g = lane; g < chunks; g += kLanes) put_zeros(row + lead + g * 16);
}

// By a whole workgroup of WAVES waves.
template <int WAVES>
__device__ __forceinline__ void zero_block(const ZeroArgs& z, const Tokens& tok, uint32_t block) {
  __shared__ uint32_t bits[1 << kZeroShift];   // the span's rows that occur
  constexpr uint32_t kAll = WAVES * kLanes;
  const uint32_t t = threadIdx.x, words = 1u << z.shift;
  const uint32_t w0 = (z.first + block) << z.shift;   // vocab < 2^31: fits
  const uint64_t first = (uint64_t)w0 * 32;
  if (t < words) bits[t] = 0;
  __syncthreads();
  if (z.mode == kZeroSeen) {
    const uint32_t w = t & (words - 1);
    uint32_t found = 0;
    if (w0 + w < z.words)
      for (uint32_t span = t >> z.shift; span < z.spans; span += kAll >> z.shift)
        found |= gp(z.seen)[(uint64_t)span * z.words + w0 + w];
    if (found) atomicOr(&bits[w], found);
  } else if (z.mode == kZeroScan) {
    for (uint32_t i = t; i < tok.n; i += kAll * 8) {
      int64_t row[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) row[u] = tok.row(min(i + u * kAll, tok.n - 1));
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const uint64_t r = (uint64_t)row[u] - first;   // far off for a token outside (-1)
        if (r < (uint64_t)words * 32) atomicOr(&bits[r / 32], 1u << (r % 32));
      }
    }
  }
  __syncthreads();
  if (first >= tok.vocab) return;
  const uint32_t rows = (uint32_t)min((uint64_t)words * 32, tok.vocab - first);
  uint8_t* span = z.grad + first * z.stride;
  if (z.stride == z.row_bytes && z.row_bytes < kWideRow) {
    zero_flat(z, bits, span, rows);
  } else {
    for (uint32_t r = __builtin_amdgcn_readfirstlane(t / kLanes); r < rows; r += WAVES)
      if (!((bits[r / 32] >> (r % 32)) & 1u)) zero_row(span + r * z.stride, z.row_bytes);
  }
}

// -------------------------------------------------------------------- sort --
// The tokens' rows in ascending order, equal ones by position, as (row,
// position) pairs: a least-significant-digit radix sort.  Tokens outside the
// slice sort as row `vocab`, behind all others.  The place of an item among those of its
// digit is its rank among the wave's items of the same digit (ballots find the
// equal lanes) plus the counts of the waves before it, so the order is the
// input's and no atomic decides it.
struct SortArgs {
  Tokens tok;
  const uint32_t* keys;    // the pairs (null: the first pass, over the tokens)
  const uint32_t* pos;
  uint32_t* keys_out;
  uint32_t* pos_out;
  uint32_t* counts;        // [spans][2^bits]
  uint32_t* seen;          // the first pass: [spans][words], a bit for each row that occurs
  ZeroArgs zero;
  uint32_t n, spans, walk, words;   // a span is `walk` tiles
  int shift, bits, passes;
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, uint32_t i) {
  if (a.keys) return gp(a.keys)[i];
  const int64_t row = a.tok.row(i);
  return row < 0 ? (uint32_t)a.tok.vocab : (uint32_t)row;
}

// The rank of this lane's item among those of its digit that the wave has seen;
// `count` holds the wave's counts and takes this step's.  !in: no item.
__device__ __forceinline__ uint32_t rank_in_wave(uint32_t* count, uint32_t digit, int bits, bool in) {
  uint64_t same = __ballot(in);
  for (int b = 0; b < bits; ++b) {
    const bool one = (digit >> b) & 1u;
    const uint64_t ones = __ballot(one);
    same &= one ? ones : ~ones;
  }
  const uint32_t before = __popcll(same & ((1ull << (threadIdx.x % kLanes)) - 1));
  uint32_t seen = 0;
  if (in) seen = count[digit];
  // the wave's lanes have read the count before the first of them writes it,
  // and it is written before the next step reads it: LDS operations of one wave
  // complete in order, and the fences keep the compiler to it
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (in && before == 0) count[digit] = seen + (uint32_t)__popcll(same);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  return seen + before;
}

// The exclusive sum of v over the workgroup's lanes (WAVES waves).
template <int WAVES>
__device__ __forceinline__ uint32_t scan_block(uint32_t v, uint32_t* shared) {
  const uint32_t lane = threadIdx.x % kLanes, wave = threadIdx.x / kLanes;
  uint32_t sum = v;
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) {
    const uint32_t from = __shfl_up(sum, o);
    sum += lane >= (uint32_t)o ? from : 0;
  }
  if (lane == kLanes - 1) shared[wave] = sum;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < WAVES; ++w) before += (uint32_t)w < wave ? shared[w] : 0;
  return before + sum - v;
}

// Up to kSmallSort tokens: one workgroup holds them in LDS and runs all passes, in
// digits of 8 bits: one launch of 6 us (16 tokens), 8 (2048), 20 (8192, where it takes
// as long as the four launches below).
constexpr int kSmallLanes = 1024;
constexpr int kSmallWaves = kSmallLanes / kLanes;
constexpr int kSmallSteps = 8;
constexpr uint32_t kSmallSort = kSmallLanes * kSmallSteps;
constexpr int kSmallBits = 8;

__global__ void __launch_bounds__(kSmallLanes) sort_small_kernel(const SortArgs a) {
  __shared__ uint32_t keys[kSmallSort], pos[kSmallSort];
  __shared__ uint32_t count[kSmallWaves][1 << kSmallBits];
  __shared__ uint32_t sums[kSmallWaves];
  if (blockIdx.x) return zero_block<kSmallWaves>(a.zero, a.tok, blockIdx.x - 1);
  const uint32_t t = threadIdx.x, lane = t % kLanes, wave = t / kLanes;
  // a wave's items are consecutive, and all waves have some
  const uint32_t steps = (a.n + kSmallLanes - 1) / kSmallLanes;
  const uint32_t base = wave * steps * kLanes + lane;
  uint32_t key[kSmallSteps], at[kSmallSteps], rank[kSmallSteps];
#pragma unroll
  for (int s = 0; s < kSmallSteps; ++s) {
    const uint32_t i = base + s * kLanes;
    at[s] = i;
    key[s] = (uint32_t)s < steps && i < a.n ? sort_key(a, i) : 0;
  }
  for (int p = 0; p < a.passes; ++p) {
    const int shift = p * kSmallBits;
    for (uint32_t b = t; b < kSmallWaves << kSmallBits; b += kSmallLanes) (&count[0][0])[b] = 0;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kSmallSteps; ++s)
      if ((uint32_t)s < steps)
        rank[s] = rank_in_wave(count[wave], (key[s] >> shift) & ((1u << kSmallBits) - 1), kSmallBits,
                               base + s * kLanes < a.n);
    __syncthreads();
    uint32_t all = 0;
    if (t < 1u << kSmallBits)
      for (int w = 0; w < kSmallWaves; ++w) all += count[w][t];
    uint32_t begin = scan_block<kSmallWaves>(all, sums);
    if (t < 1u << kSmallBits)
      for (int w = 0; w < kSmallWaves; ++w) {
        const uint32_t c = count[w][t];
        count[w][t] = begin;
        begin += c;
      }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kSmallSteps; ++s)
      if ((uint32_t)s < steps && base + s * kLanes < a.n) {
        const uint32_t to = count[wave][(key[s] >> shift) & ((1u << kSmallBits) - 1)] + rank[s];
        keys[to] = key[s];
        pos[to] = at[s];
      }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kSmallSteps; ++s)
      if ((uint32_t)s < steps && base + s * kLanes < a.n) {
        key[s] = keys[base + s * kLanes];
        at[s] = pos[base + s * kLanes];
      }
  }
#pragma unroll
  for (int s = 0; s < kSmallSteps; ++s)
    if ((uint32_t)s < steps && base + s * kLanes < a.n) {
      gp(a.keys_out)[base + s * kLanes] = key[s];
      gp(a.pos_out)[base + s * kLanes] = at[s];
    }
}

// More tokens: digits of at most 9 bits (two of 8 for a vocabulary of 50304, two of 9
// below 2^18), a pass of two launches.  Each workgroup counts the digits of its
// span; then each sums the counts of the spans before its own (and of the smaller
// digits) and scatters its span.  Bound by the latency of a few dependent loads: 5 and 7.5 us
// for 65536 tokens (7 and 20 with tiles of 4096 and each load waited for by itself).
// A span is one tile, or, of more than kMaxSpans tiles (2^20 tokens), as many as leave that many
// spans, one after the other: every workgroup reads the counts of all, which with a span
// for each tile grew with the tokens' square.
constexpr int kSortLanes = 512;
constexpr int kSortWaves = kSortLanes / kLanes;
constexpr int kSortSteps = 4;                        // items per lane
constexpr uint32_t kSortTile = kSortLanes * kSortSteps;
constexpr int kMaxDigit = 9;                         // a lane for each value
constexpr uint32_t kMaxSpans = 512;                  // two workgroups a CU
constexpr uint32_t kCountsAhead = 32;

__global__ void __launch_bounds__(kSortLanes) sort_count_kernel(const SortArgs a) {
  __shared__ uint32_t count[1 << kMaxDigit];
  extern __shared__ uint32_t seen[];   // the first pass: `words` of them
  if (blockIdx.x >= a.spans)
    return zero_block<kSortWaves>(a.zero, a.tok, blockIdx.x - a.spans);
  const uint32_t bins = 1u << a.bits, t = threadIdx.x;
  const uint32_t words = a.seen ? a.words : 0;
  count[t] = 0;
  for (uint32_t w = t; w < words; w += kSortLanes) seen[w] = 0;
  __syncthreads();
  for (uint32_t tile = 0; tile < a.walk; ++tile) {
    const uint32_t base = (blockIdx.x * a.walk + tile) * kSortTile;
    uint32_t key[kSortSteps];
#pragma unroll
    for (int s = 0; s < kSortSteps; ++s) {
      const uint32_t i = base + s * kSortLanes + t;
      key[s] = i < a.n ? sort_key(a, i) : 0;
    }
#pragma unroll
    for (int s = 0; s < kSortSteps; ++s)
      if (base + s * kSortLanes + t < a.n) {
        atomicAdd(&count[(key[s] >> a.shift) & (bins - 1)], 1u);
        if (words && key[s] < (uint32_t)a.tok.vocab) atomicOr(&seen[key[s] / 32], 1u << (key[s] % 32));
      }
  }
  __syncthreads();
  if (t < bins) gp(a.counts)[(uint64_t)blockIdx.x * bins + t] = count[t];
  for (uint32_t w = t; w < words; w += kSortLanes)
    gp(a.seen)[(uint64_t)blockIdx.x * words + w] = seen[w];
}

__global__ void __launch_bounds__(kSortLanes) sort_scatter_kernel(const SortArgs a) {
  __shared__ uint32_t count[kSortWaves][1 << kMaxDigit];
  __shared__ uint32_t sums[kSortWaves];
  if (blockIdx.x >= a.spans)
    return zero_block<kSortWaves>(a.zero, a.tok, blockIdx.x - a.spans);
  const uint32_t bins = 1u << a.bits, t = threadIdx.x, lane = t % kLanes, wave = t / kLanes;
  // the wave's items: 64 consecutive ones per step; all loads are issued up front
  uint32_t base = blockIdx.x * a.walk * kSortTile + wave * (kLanes * kSortSteps) + lane;
  uint32_t key[kSortSteps], at[kSortSteps], rank[kSortSteps];
  const auto load_tile = [&] {
#pragma unroll
    for (int s = 0; s < kSortSteps; ++s) {
      const uint32_t i = base + s * kLanes;
      key[s] = i < a.n ? sort_key(a, i) : 0;
      at[s] = !a.keys || i >= a.n ? i : gp(a.pos)[i];
    }
  };
  load_tile();
  // lane t owns digit t: how many of it lie in the spans before this one, and in all
  uint32_t here = 0, all = 0;
  if (t < bins) {
    const global<uint32_t>* c = gp((const uint32_t*)a.counts) + t;
    for (uint32_t b = 0; b < a.spans; b += kCountsAhead) {
      uint32_t v[kCountsAhead];
#pragma unroll
      for (uint32_t u = 0; u < kCountsAhead; ++u)
        v[u] = b + u < a.spans ? c[(uint64_t)(b + u) * bins] : 0;
#pragma unroll
      for (uint32_t u = 0; u < kCountsAhead; ++u) {
        here += b + u < blockIdx.x ? v[u] : 0;
        all += v[u];
      }
    }
  }
  uint32_t next = here;   // where the tile's first item of digit t goes
  for (uint32_t tile = 0;;) {
    for (int w = 0; w < kSortWaves; ++w) count[w][t] = 0;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kSortSteps; ++s)
      rank[s] = rank_in_wave(count[wave], (key[s] >> a.shift) & (bins - 1), a.bits,
                             base + s * kLanes < a.n);
    if (tile == 0)   // (a barrier in each branch: all counts are there)
      next += scan_block<kSortWaves>(all, sums);
    else
      __syncthreads();
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = count[w][t];
      count[w][t] = next;
      next += c;
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kSortSteps; ++s) {
      if (base + s * kLanes >= a.n) continue;
      const uint32_t to = count[wave][(key[s] >> a.shift) & (bins - 1)] + rank[s];
      gp(a.keys_out)[to] = key[s];
      gp(a.pos_out)[to] = at[s];
    }
    if (++tile == a.walk) break;
    base += kSortTile;
    load_tile();
    __syncthreads();   // the counts have been read
  }
}

// ------------------------------------------------------------ segment sums --
// The sorted pairs in tiles of 16 or 32, each summed by one wave for each 64
// groups of columns: the rows' loads in batches of kBatch, the running sum in
// fp32 registers, put out where the row changes.  A run of equal rows belongs to
// the tile it begins in, whose wave follows it into the next tile; only a run that
// covers the whole next tile is split: every tile it touches leaves its part
// in `parts`, and join_kernel adds them in order.  So a token on a tenth of all
// positions costs what others do, and the common short runs cost no second pass.
// (With every run that crosses a tile's end split, the join took 35 us, now 9.)
//
// Bound by memory, gathered rows of 4 KiB at that: 65536 tokens of 2048 bf16, with the zeros
// that ride along, in 95 us, 274 MB read and 294 MB written (6.0 TB/s).  The sums go through
// the caches, in whole lines (Columns): the whole call takes 134 us into one gradient buffer (143
// into another one each time); whole lines streamed 156, a lane's 8 fp32 as two stores of half
// lines 143.
//
// Tiles of 16 where there are few: more waves share the gathers' latency (tiles of 8 /
// 16 / 32, us for the whole call: 67 tokens of 64 bf16 15.7 16.7 19.4; 2048 of 1999 fp32
// 25.1 24.9 25.6; 16384 tokens, a gradient of 131072 x 1024, 120 120 121; 32768 tokens,
// 50304 x 2048, 128 116 114; 65536 of the same 163 139 134).
constexpr uint32_t kFewTokens = 16384;
constexpr uint32_t kMaxTile = 32;   // two tiles' pairs in the lanes of a wave
constexpr uint32_t tile_for(uint64_t n) { return n <= kFewTokens ? kMaxTile / 2 : kMaxTile; }
constexpr int kBatch = 16;
constexpr int kSumWaves = 2;

struct SumArgs {
  const uint32_t* keys;
  const uint32_t* pos;
  const void* dout;
  void* grad;
  float* parts;            // [tiles][2][hidden]: a run from before, a run that begins here
  Tokens tok;
  ZeroArgs zero;
  uint64_t dout_stride, grad_stride, vocab;
  uint32_t n, tile, tiles, hidden, slabs, sum_blocks, join_blocks, join_columns;
  int accumulate;
  float scale;
};

// Elements [c, c + N) of a row of `hidden`: N of them, 16 bytes or 8, or (TAIL) what is left.
template <typename T, int N, bool TAIL>
__device__ __forceinline__ void put_row(T* row, uint32_t c, uint32_t hidden, const float* sum,
                                        float scale, bool add) {
  if constexpr (!TAIL) {
    typedef T __attribute__((ext_vector_type(N), aligned(sizeof(T)))) some;
    typedef float __attribute__((ext_vector_type(N))) wide;
    auto* at = (global<some>*)(uintptr_t)(row + c);
    wide w;
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = sum[e] * scale;
    if (add) w += __builtin_convertvector(*at, wide);
    *at = __builtin_convertvector(w, some);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c + e < hidden) {
        float v = sum[e] * scale;
        if (add) v += (float)gp(row)[c + e];
        gp(row)[c + e] = (T)v;
      }
  }
}

// A lane's columns of a slab of 64 groups: a group, or, of 16-bit rows summed into fp32 ones,
// two halves of one that lie 64 halves apart, so that each store of the wave's is whole
// lines of the gradient.
template <typename T, typename O>
struct Columns {
  static constexpr int kPieces = sizeof(O) > sizeof(T) ? 2 : 1;
  static constexpr int kN = Group<T>::kN / kPieces;   // columns of a piece
  typedef T __attribute__((ext_vector_type(kN), aligned(sizeof(T)))) any;
  typedef T __attribute__((ext_vector_type(kN))) vec;
  typedef float __attribute__((ext_vector_type(kN))) wide;
};

// TAIL: the last group of a row is stored element by element.  Otherwise it starts
// early, so that it ends with the row; its lane then writes some elements that its
// neighbour writes too, the same values, which only a gradient that is written and not
// added to allows.
template <typename T, typename O, bool ADD, bool TAIL>
__global__ void __launch_bounds__(kSumWaves * kLanes) sum_kernel(const SumArgs a) {
  typedef Columns<T, O> C;
  constexpr int N = C::kN, P = C::kPieces;
  const uint32_t lane = threadIdx.x % kLanes;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
  // the workgroups that write zeros lie evenly between the others: the ones wait for
  // gathered reads, the others fill the time with stores
  const uint64_t blocks = (uint64_t)a.sum_blocks + a.zero.blocks;
  const uint32_t zeros = (uint32_t)(blockIdx.x * (uint64_t)a.zero.blocks / blocks);
  if ((uint32_t)((blockIdx.x + 1ull) * a.zero.blocks / blocks) != zeros)
    return zero_block<kSumWaves>(a.zero, a.tok, zeros);
  const uint64_t job = (uint64_t)(blockIdx.x - zeros) * kSumWaves + wave;
  const uint32_t tile = (uint32_t)(job / a.slabs), slab = (uint32_t)(job % a.slabs);
  if (tile >= a.tiles) return;
  // this lane's columns; lanes behind the row read what the last one reads
  uint32_t c[P];
  bool on[P];
#pragma unroll
  for (int q = 0; q < P; ++q) {
    c[q] = ((slab * P + q) * kLanes + lane) * N;
    on[q] = c[q] < a.hidden;
    if (!TAIL) c[q] = min(c[q], a.hidden - N);
  }
  const uint32_t first = tile * a.tile, len = min(a.tile, a.n - first);

  // lane l holds pair l of this tile and the next; `prev` and `before` are the
  // keys in front of this tile and of the one before it
  uint32_t key = 0xffffffffu, pos = 0;
  if (first + lane < a.n) {
    key = gp(a.keys)[first + lane];
    pos = gp(a.pos)[first + lane];
  }
  const uint32_t none = 0xffffffffu;
  const uint32_t prev = first ? gp(a.keys)[first - 1] : none;
  const uint32_t before = first > a.tile ? gp(a.keys)[first - a.tile - 1] : none;
  const uint32_t vocab = (uint32_t)a.vocab;
  const uint32_t head = __builtin_amdgcn_readlane(key, 0);
  const uint32_t tail = __builtin_amdgcn_readlane(key, len - 1);
  const uint32_t next_len = first + a.tile < a.n ? min(a.tile, a.n - first - a.tile) : 0;

  // the run from before: whose is it?  The tile it begins in takes it to its end,
  // unless it covers a whole tile behind that one (this one, or the one before)
  uint32_t b = 0;
  bool head_part = head == prev;
  if (head_part && tail != head && before != head) {
    b = __popcll(__ballot(lane < len && key == head));
    head_part = false;
  }
  // the run at the end: split if it covers the next tile, else followed into it
  bool tail_part = false;
  uint32_t end = len;
  if (next_len && tail < vocab) {
    const uint32_t first_next = __builtin_amdgcn_readlane(key, a.tile);
    const uint32_t last_next = __builtin_amdgcn_readlane(key, a.tile + next_len - 1);
    const bool mine = !(head_part && tail == head);
    if (mine && first_next == tail) {
      if (last_next == tail)
        tail_part = true;
      else
        end += __popcll(__ballot(lane >= a.tile && key == tail));
    }
  }
  // the tokens outside the slice are the last
  end = min(end, (uint32_t)__popcll(__ballot(key < vocab)));
  if (b >= end) return;

  float sum[P][N] = {};
  uint32_t run = __builtin_amdgcn_readlane(key, b);
  bool part = head_part;
  const auto put = [&](uint32_t slot) {
    float* const at = a.parts + ((uint64_t)tile * 2 + slot) * a.hidden;
    O* const row = (O*)a.grad + (uint64_t)run * a.grad_stride;
#pragma unroll
    for (int q = 0; q < P; ++q) {
      if (!on[q]) continue;
      if constexpr (sizeof(O) == 4 && !ADD)   // one place in the code for both
        put_row<float, N, TAIL>(part ? at : row, c[q], a.hidden, sum[q], part ? 1.0f : a.scale, false);
      else if (part)
        put_row<float, N, TAIL>(at, c[q], a.hidden, sum[q], 1.0f, false);
      else
        put_row<O, N, TAIL>(row, c[q], a.hidden, sum[q], a.scale, ADD);
    }
  };
  for (; b < end; b += kBatch) {
    typename C::vec v[kBatch][P];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {   // behind the end, the last row again
      const uint32_t p = __builtin_amdgcn_readlane(pos, min(b + u, end - 1));
      const T* src = (const T*)a.dout + (uint64_t)p * a.dout_stride;
#pragma unroll
      for (int q = 0; q < P; ++q) {
        if (!TAIL || c[q] + N <= a.hidden) {
          v[u][q] = __builtin_nontemporal_load((const global<typename C::any>*)(uintptr_t)(src + c[q]));
        } else {
          v[u][q] = {};
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (c[q] + e < a.hidden) v[u][q][e] = gp(src + c[q])[e];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (b + u >= end) break;
      const uint32_t k = __builtin_amdgcn_readlane(key, b + u);
      if (k != run) {   // the run ended
        put(0);
        run = k;
        part = false;
#pragma unroll
        for (int q = 0; q < P; ++q)
#pragma unroll
          for (int e = 0; e < N; ++e) sum[q][e] = 0.0f;
      }
#pragma unroll
      for (int q = 0; q < P; ++q) {
        const typename C::wide w = __builtin_convertvector(v[u][q], typename C::wide);
#pragma unroll
        for (int e = 0; e < N; ++e) sum[q][e] += w[e];
      }
    }
  }
  const uint32_t slot = part ? 0 : 1;
  part = part || tail_part;
  put(slot);
}

// A workgroup for 256 columns of the runs that begin in one of kJoinTiles tiles (as its
// last run) and cover the next one: its waves share the tiles of a run, in order,
// and their sums are added in order.
constexpr int kJoinTiles = 16;
constexpr int kJoinWaves = 8;
constexpr int kJoinBatch = 8;

template <typename O>
__global__ void __launch_bounds__(kJoinWaves * kLanes) join_kernel(const SumArgs a) {
  typedef Group<float> G;
  __shared__ float shared[kJoinWaves][kLanes][G::kN];
  if (blockIdx.x >= a.join_blocks)
    return zero_block<kJoinWaves>(a.zero, a.tok, blockIdx.x - a.join_blocks);
  const uint32_t lane = threadIdx.x % kLanes;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
  const uint32_t c = (blockIdx.x % a.join_columns * kLanes + lane) * G::kN;
  const uint32_t first = blockIdx.x / a.join_columns * kJoinTiles, mine = first + lane;
  uint32_t key = 0;
  bool head = false;
  if (lane < kJoinTiles && mine + 1 < a.tiles) {
    const uint32_t last = mine * a.tile + a.tile - 1;
    key = gp(a.keys)[last];
    const uint32_t next_last = gp(a.keys)[min(last + a.tile, a.n - 1)];
    // where the key in front of the tile is the run's, it began before
    const uint32_t prev = mine ? gp(a.keys)[mine * a.tile - 1] : 0xffffffffu;
    head = key < a.vocab && next_last == key && prev != key;
  }
  uint64_t heads = __ballot(head);
  while (heads) {
    const uint32_t h = __builtin_ctzll(heads), tile = first + h;
    heads &= heads - 1;
    const uint32_t run = __builtin_amdgcn_readlane(key, h);
    // the run's parts: slot 1 of `tile`, slot 0 of the tiles behind it that begin with it
    uint32_t parts = 2;
    for (;;) {
      const uint64_t at = (uint64_t)(tile + parts + lane) * a.tile;
      const uint64_t in = __ballot(at < a.n && gp(a.keys)[at < a.n ? at : 0] == run);
      if (in != ~0ull) {
        parts += __builtin_ctzll(~in);
        break;
      }
      parts += kLanes;
    }
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
#pragma unroll
    for (int e = 0; e < G::kN; ++e) shared[wave][lane][e] = sum[e];
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
        for (int e = 0; e < G::kN; ++e) sum[e] += shared[w][lane][e];
      O* const row = (O*)a.grad + (uint64_t)run * a.grad_stride;
      if (c + G::kN <= a.hidden)
        put_row<O, G::kN, false>(row, c, a.hidden, sum, a.scale, a.accumulate);
      else
        put_row<O, G::kN, true>(row, c, a.hidden, sum, a.scale, a.accumulate);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------- host launchers --

int bits_of(uint64_t v) {   // of the largest key
  int b = 1;
  while (b < 32 && (v >> b)) ++b;
  return b;
}

constexpr uint64_t up16(uint64_t v) { return (v + 15) / 16 * 16; }

// Rows up to which the sort's first launch collects which rows occur: a bit each
// in LDS.
constexpr uint64_t kMaxSeen = 1u << 18;

struct Work {
  uint64_t keys[2], pos[2], counts, seen, parts, bytes;
  uint32_t sort_spans, walk, sum_tiles, words;
  int passes, bits;
  bool small;
};

Work work_of(uint64_t n, uint64_t vocab, uint32_t hidden) {
  Work w = {};
  w.small = n <= kSmallSort;
  const int all = bits_of(vocab), digit = w.small ? kSmallBits : kMaxDigit;
  w.passes = (all + digit - 1) / digit;
  w.bits = (all + w.passes - 1) / w.passes;
  const uint64_t tiles = (n + kSortTile - 1) / kSortTile;
  w.walk = (uint32_t)((tiles + kMaxSpans - 1) / kMaxSpans);
  w.sort_spans = w.walk ? (uint32_t)((tiles + w.walk - 1) / w.walk) : 0;
  w.sum_tiles = (uint32_t)((n + tile_for(n) - 1) / tile_for(n));
  w.words = w.small || vocab > kMaxSeen ? 0 : (uint32_t)((vocab + 31) / 32);
  uint64_t at = 0;
  const auto take = [&at](uint64_t bytes) {
    const uint64_t here = at;
    at += up16(bytes);
    return here;
  };
  for (int i = 0; i < (w.small ? 1 : 2); ++i) {
    w.keys[i] = take(4 * n);
    w.pos[i] = take(4 * n);
  }
  if (!w.small) w.counts = take(4ull * w.sort_spans << w.bits);
  w.seen = take(4ull * w.sort_spans * w.words);
  w.parts = take(8ull * w.sum_tiles * hidden);
  w.bytes = at;
  return w;
}

// Bytes of zeros that a launch of the sort takes along at least: about what is written
// while it waits for its own loads.  It takes more where the sums' launch would be
// left with more zeros than it reads of dout, which is what hides behind its gathers.
// At least 0 / 20 / 40 / 60 / 100 / 200 MiB a launch, us for the whole call: 65536 tokens, 50304
// x 2048 bf16 to fp32 137 136 134 134 142 151; 32768 tokens of the same 115 115 114 112 115
// 125; 16384 tokens, 131072 x 1024 124 124 120 120 120 122.  (With all zeros in the sums'
// launch 65536 tokens took 165 us where 40 MiB a launch took 153.)
constexpr uint64_t kZeroBytes = 40u << 20;

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
  const bool streamed = a.groups >= kEmbedStreamGroups && n * hidden * type_bytes(type) >= kEmbedStream;
  while (a.shift < 6 && (1u << a.shift) * kEmbedGroups < a.groups) ++a.shift;
  const uint32_t rows = kEmbedWaves * (kLanes >> a.shift), wide = kEmbedGroups << a.shift;
  const uint64_t most = max_grid(kEmbedWaves * kLanes) * rows;   // tokens of one launch
  return with_type(type, [&](auto t) {
    const auto kernel = streamed ? embed_kernel<decltype(t), true> : embed_kernel<decltype(t), false>;
    for (uint64_t at = 0; at < n; at += most) {
      a.n = (uint32_t)std::min(most, n - at);
      a.tokens = (const uint8_t*)d_tokens + at * token_bytes;
      a.out = (uint8_t*)d_out + at * hidden * type_bytes(type);
      const dim3 grid((a.n + rows - 1) / rows, (a.groups + wide - 1) / wide);
      kernel<<<grid, kEmbedWaves * kLanes, 0, (hipStream_t)stream>>>(a);
    }
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

  const Tokens tok = {d_tokens, vocab_start, vocab, (uint32_t)n, token_bytes};
  ZeroArgs z = {};
  z.grad = (uint8_t*)d_grad;
  z.seen = (const uint32_t*)(work + w.seen);
  z.stride = grad_stride * type_bytes(grad_type);
  z.row_bytes = hidden * type_bytes(grad_type);
  z.words = w.words;
  z.spans = w.sort_spans;
  z.mode = w.small ? kZeroScan : w.words ? kZeroSeen : kZeroAll;
  z.by_row = make_fastdiv(z.row_bytes);
  const uint64_t span = std::min(kMostSpan, std::max(kLeastSpan, vocab * z.row_bytes / kZeroSpans));
  while (z.shift < kZeroShift && (64ull << z.shift) * z.row_bytes <= span) ++z.shift;
  const uint64_t zero_rows = 32ull << z.shift;
  const uint32_t all_zero = accumulate ? 0 : (uint32_t)((vocab + zero_rows - 1) / zero_rows);
  const uint64_t zero_bytes = vocab * z.row_bytes, read = n * hidden * type_bytes(type);
  const uint64_t launches = 2 * w.passes - (z.mode == kZeroSeen);
  const uint64_t bytes = std::max(kZeroBytes, zero_bytes > read ? (zero_bytes - read) / launches : 0);
  const uint64_t share = bytes / (z.row_bytes * zero_rows) + 1;
  const auto with_join = (uint32_t)std::min<uint64_t>(all_zero, kZeroBytes / (z.row_bytes * zero_rows));
  // the next launch's zero blocks: all that are left but `leave`
  const auto zeros = [&](uint64_t leave) {
    z.first += z.blocks;
    const uint64_t left = all_zero - z.first;
    z.blocks = (uint32_t)(left > leave ? left - leave : 0);
    return z.blocks;
  };
  // a sort launch's: its share
  const auto sort_zeros = [&] {
    const uint64_t left = all_zero - z.first - z.blocks;
    return zeros(left > share ? left - share : 0);
  };

  const int last = w.small ? 0 : (w.passes + 1) & 1;   // where the sorted pairs will be
  SumArgs a = {};
  a.keys = (const uint32_t*)(work + w.keys[last]);
  a.pos = (const uint32_t*)(work + w.pos[last]);
  a.dout = d_dout;
  a.grad = d_grad;
  a.parts = (float*)(work + w.parts);
  a.tok = tok;
  a.dout_stride = dout_stride;
  a.grad_stride = grad_stride;
  a.vocab = vocab;
  a.n = (uint32_t)n;
  a.tile = tile_for(n);
  a.tiles = w.sum_tiles;
  a.hidden = hidden;
  a.accumulate = accumulate != 0;
  a.scale = scale;
  const uint32_t per_group = 16 / type_bytes(type);
  a.slabs = (hidden + per_group * kLanes - 1) / (per_group * kLanes);
  const uint64_t sum_blocks = ((uint64_t)a.tiles * a.slabs + kSumWaves - 1) / kSumWaves;
  a.join_columns = (hidden + kLanes * 4 - 1) / (kLanes * 4);
  const uint64_t join_blocks =
      a.tiles > 1 ? (uint64_t)(a.tiles + kJoinTiles - 2) / kJoinTiles * a.join_columns : 0;
  // each launch as if it took all zeros along
  const auto past = [&](uint64_t blocks, uint64_t lanes) { return (blocks + all_zero) * lanes >= 1ull << 32; };
  if (past(sum_blocks, kSumWaves * kLanes) || past(join_blocks, kJoinWaves * kLanes) ||
      past(w.sort_spans, w.small ? kSmallLanes : kSortLanes))
    return EC_ERANGE;
  a.sum_blocks = (uint32_t)sum_blocks;
  a.join_blocks = (uint32_t)join_blocks;

  SortArgs s = {};
  s.tok = tok;
  s.n = (uint32_t)n;
  s.spans = w.sort_spans;
  s.walk = w.walk;
  s.words = w.words;
  s.bits = w.bits;
  s.passes = w.passes;
  s.counts = (uint32_t*)(work + w.counts);
  if (w.small && n) {
    s.keys_out = (uint32_t*)(work + w.keys[0]);
    s.pos_out = (uint32_t*)(work + w.pos[0]);
    const uint32_t extra = zeros(0);   // what the sums' launch would wait for longer
    s.zero = z;
    sort_small_kernel<<<1 + extra, kSmallLanes, 0, st>>>(s);
  }
  for (int p = 0; !w.small && p < w.passes; ++p) {
    s.keys = p ? (const uint32_t*)(work + w.keys[(p + 1) & 1]) : nullptr;
    s.pos = (const uint32_t*)(work + w.pos[(p + 1) & 1]);
    s.keys_out = (uint32_t*)(work + w.keys[p & 1]);
    s.pos_out = (uint32_t*)(work + w.pos[p & 1]);
    s.seen = p == 0 && w.words ? (uint32_t*)(work + w.seen) : nullptr;
    s.shift = p * w.bits;
    // the first launch collects the rows that occur, so it has none to write yet; where
    // none are collected all rows are zeroed, and before the sums write theirs
    uint32_t extra = p || z.mode == kZeroAll ? sort_zeros() : 0;
    s.zero = z;
    sort_count_kernel<<<s.spans + extra, kSortLanes, s.seen ? 4 * w.words : 0, st>>>(s);
    extra = z.mode == kZeroAll && p + 1 == w.passes ? zeros(0) : sort_zeros();
    s.zero = z;
    sort_scatter_kernel<<<s.spans + extra, kSortLanes, 0, st>>>(s);
  }

  const uint32_t behind = join_blocks ? with_join : 0;   // zeros that the join takes along
  const auto go = [&](auto t, auto o) {
    typedef decltype(t) T;
    typedef decltype(o) O;
    // a last piece that starts early needs a whole one, and rows that are written
    constexpr uint32_t kPiece = Columns<T, O>::kN;
    const bool tail = hidden < kPiece || (accumulate && hidden % kPiece);
    const auto sum = accumulate ? tail ? sum_kernel<T, O, true, true> : sum_kernel<T, O, true, false>
                                : tail ? sum_kernel<T, O, false, true> : sum_kernel<T, O, false, false>;
    uint32_t extra = zeros(behind);
    a.zero = z;
    if (a.sum_blocks + extra)
      sum<<<a.sum_blocks + extra, kSumWaves * kLanes, 0, st>>>(a);
    extra = zeros(0);
    a.zero = z;
    if (a.join_blocks) join_kernel<O><<<a.join_blocks + extra, kJoinWaves * kLanes, 0, st>>>(a);
    return launched();
  };
  return with_type(type, [&](auto t) {
    return grad_type == EC_F32 ? go(t, float()) : go(t, t);
  });
}

}  // extern "C"
