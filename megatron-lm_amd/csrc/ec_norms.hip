// ec_norms.hip — ec_residual_norm and ec_residual_norm_grad: what stands between two blocks of
// a residual stream, in one pass over each row.
//
//   u = branch, or branch_weight * branch / rms(branch)
//   sum = residual + scale * gate * u
//   normed = weight * sum / rms(sum)
//
// A row is held in the registers of a team of 64 to 1024 lanes, 16 bytes a lane and group,
// so that it is read once whatever is done with it.  The norms' sums go over
// the wave by shuffles and over the team's waves through LDS.
//
// Backward, a team goes over a run of rows and keeps the sums over them, of the weights' and the
// gate's gradients, in registers (those of the longest rows partly in LDS); each team leaves one row of partials, which a second launch
// adds in order.  No atomics.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "ec_types.h"
#include "routes.h"

namespace ec {
namespace {

constexpr uint32_t kMostWidth = 16384;
constexpr int kTeamLanes = 256;   // of a workgroup of teams of 64 lanes

template <int R>
constexpr int block_lanes() {
  return R > 64 ? R : kTeamLanes;
}

// The sum over a team's R lanes, in each of them.  `turn` alternates from call to call, so that a slot is
// not written again before every wave has read it: the barrier of the call in between is behind that.
template <int R>
__device__ __forceinline__ float team_sum(float v, int& turn) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (R > 64) {
    __shared__ float slots[2][R / 64];
    if (threadIdx.x % 64 == 0) slots[turn][threadIdx.x / 64] = v;
    __syncthreads();
    v = slots[turn][0];
#pragma unroll
    for (int w = 1; w < R / 64; ++w) v += slots[turn][w];
    turn ^= 1;
  }
  return v;
}

// A lane's groups of a row as they lie in memory: half the registers of 16-bit values, for rows that are under way.
template <typename T, int V>
struct Raw {
  typename Group<T>::vec x[V];
};

// V groups of a row, one after another R lanes apart: group v of lane l is at (v R + l) kN.
template <typename T, int R, int V>
struct Row {
  static constexpr int kN = Group<T>::kN;
  float x[V][kN];

  __device__ __forceinline__ static uint32_t at(int v) {
    return ((uint32_t)v * R + threadIdx.x % R) * kN;
  }

  template <bool STREAM>
  __device__ __forceinline__ static Raw<T, V> fetch(const T* p, uint32_t width) {
    Raw<T, V> raw;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const uint32_t i = at(v);
      raw.x[v] = {};
      if (i + kN <= width) {
        raw.x[v] = load_group<T, STREAM>(p + i);
      } else {
#pragma unroll
        for (int e = 0; e < kN; ++e)
          if (i + e < width) raw.x[v][e] = gp(p)[i + e];
      }
    }
    return raw;
  }

  __device__ __forceinline__ void take(const Raw<T, V>& raw) {
    each([&](int v, int e) { x[v][e] = (float)raw.x[v][e]; });
  }

  template <bool STREAM>
  __device__ __forceinline__ void load(const T* p, uint32_t width) {
    take(fetch<STREAM>(p, width));
  }

  template <typename O, bool STREAM>
  __device__ __forceinline__ void store(O* p, uint32_t width) const {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const uint32_t i = at(v);
      if (i + kN <= width) {
        typedef O __attribute__((ext_vector_type(kN), aligned(sizeof(O)))) some;
        some s;
#pragma unroll
        for (int e = 0; e < kN; ++e) s[e] = (O)x[v][e];
        auto* q = (global<some>*)(uintptr_t)(p + i);
        if constexpr (STREAM)
          __builtin_nontemporal_store(s, q);
        else
          *q = s;
      } else {
#pragma unroll
        for (int e = 0; e < kN; ++e)
          if (i + e < width) gp(p)[i + e] = (O)x[v][e];
      }
    }
  }

  __device__ __forceinline__ void fill(float value) {
    each([&](int v, int e) { x[v][e] = value; });
  }

  template <typename F>
  __device__ __forceinline__ static void each(F f) {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < kN; ++e) f(v, e);
  }
};

struct NormArgs {
  const void *residual, *branch, *gate, *branch_weight, *weight;
  uint64_t residual_stride, branch_stride, n, gate_share;   // rows that share a row of the gate
  uint64_t first;   // row of this launch
  uint32_t width;
  float scale, eps;
  void *sum, *normed;
  uint64_t sum_stride;
  float *rstd, *branch_rstd;
};

// Values past the row's end are zeros in every term of the sums.
template <typename T, int R, int V>
__global__ void __launch_bounds__(block_lanes<R>()) norm_kernel(NormArgs p) {
  typedef Row<T, R, V> row_t;
  constexpr uint32_t kTeams = block_lanes<R>() / R;
  const uint64_t row = p.first + (uint64_t)blockIdx.x * kTeams + (kTeams > 1 ? threadIdx.x / R : 0);
  if (row >= p.n) return;   // whole teams, of one wave where a workgroup has several
  // everything the row needs is under way before the first value is looked at (16384 x 2048 bf16 47 us, 52 otherwise); the
  // longest rows' factors are not, for want of registers (2048 x 16384 51 us, 62 with them)
  constexpr bool kEarly = R < 1024;
  const auto fetch = [&](const void* from, uint64_t at, bool now) {
    return from && now ? row_t::template fetch<false>((const T*)from + at, p.width) : Raw<T, V>{};
  };
  const uint64_t gate_at = row / p.gate_share * p.width;
  const Raw<T, V> r_raw = row_t::template fetch<true>((const T*)p.residual + row * p.residual_stride, p.width);
  Raw<T, V> y_raw = {};
  if (p.branch) y_raw = row_t::template fetch<true>((const T*)p.branch + row * p.branch_stride, p.width);
  const Raw<T, V> post = fetch(p.branch_weight, 0, kEarly), gate = fetch(p.gate, gate_at, kEarly);
  const Raw<T, V> pre = fetch(p.weight, 0, kEarly);
  int turn = 0;
  row_t r, f;
  r.take(r_raw);
  if (p.branch) {
    row_t y;
    y.take(y_raw);
    if (p.branch_weight) {
      float s = 0.0f;
      row_t::each([&](int v, int e) { s = __builtin_fmaf(y.x[v][e], y.x[v][e], s); });
      const float root = rsqrtf(team_sum<R>(s, turn) / (float)p.width + p.eps);
      if (threadIdx.x % R == 0 && p.branch_rstd) gp(p.branch_rstd)[row] = root;
      f.take(kEarly ? post : fetch(p.branch_weight, 0, true));
      row_t::each([&](int v, int e) { y.x[v][e] *= root * f.x[v][e]; });
    }
    if (p.gate) {
      f.take(kEarly ? gate : fetch(p.gate, gate_at, true));
      row_t::each([&](int v, int e) { y.x[v][e] *= f.x[v][e]; });
    }
    row_t::each([&](int v, int e) { r.x[v][e] = __builtin_fmaf(p.scale, y.x[v][e], r.x[v][e]); });
    r.template store<T, false>((T*)p.sum + row * p.sum_stride, p.width);
  }
  if (p.weight) {
    float s = 0.0f;
    row_t::each([&](int v, int e) { s = __builtin_fmaf(r.x[v][e], r.x[v][e], s); });
    const float root = rsqrtf(team_sum<R>(s, turn) / (float)p.width + p.eps);
    if (threadIdx.x % R == 0 && p.rstd) gp(p.rstd)[row] = root;
    f.take(kEarly ? pre : fetch(p.weight, 0, true));
    row_t::each([&](int v, int e) { r.x[v][e] *= root * f.x[v][e]; });
    r.template store<T, false>((T*)p.normed + row * p.width, p.width);
  }
}

struct GradArgs {
  const void *dsum, *dnormed, *sum, *branch, *gate, *branch_weight, *weight;
  uint64_t dsum_stride, dnormed_stride, sum_stride, branch_stride, n, gate_share;
  uint32_t width;
  float scale;
  const float *rstd, *branch_rstd;
  void *dresidual, *dbranch;
  float* dgate;        // written here where a team covers whole rows of the gate
  float *gate_parts, *branch_parts, *weight_parts;   // [teams][width]; null: not computed
  uint64_t teams, per_gate, rows;   // teams for a row of the gate; rows of a team
};

// A lane's sums over rows, of V groups: in registers, or for the longest rows in LDS, four neighbours at a time so that
// lanes meet no bank conflicts.
template <typename T, int R, int V, bool LDS>
struct Sums {
  typedef Row<T, R, V> row_t;
  row_t r;
  float* at;

  __device__ __forceinline__ void clear(float* lds) {
    at = lds + threadIdx.x * 4;
    fill();
  }
  __device__ __forceinline__ void fill() {
    if constexpr (LDS) {
#pragma unroll
      for (int i = 0; i < V * row_t::kN / 4; ++i) *(v4*)(at + i * R * 4) = v4{0.0f, 0.0f, 0.0f, 0.0f};
    } else {
      r.fill(0.0f);
    }
  }
  // += f(v, e)
  template <typename F>
  __device__ __forceinline__ void add(F f) {
    if constexpr (LDS) {
#pragma unroll
      for (int i = 0; i < V * row_t::kN / 4; ++i) {
        v4 s = *(v4*)(at + i * R * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += f(i * 4 / row_t::kN, i * 4 % row_t::kN + e);
        *(v4*)(at + i * R * 4) = s;
      }
    } else {
      row_t::each([&](int v, int e) { r.x[v][e] += f(v, e); });
    }
  }
  __device__ __forceinline__ void store(float* to, uint32_t width) {
    if constexpr (LDS) {
#pragma unroll
      for (int i = 0; i < V * row_t::kN / 4; ++i) {
        const v4 s = *(v4*)(at + i * R * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t c = row_t::at(i * 4 / row_t::kN) + i * 4 % row_t::kN + e;
          if (c < width) gp(to)[c] = s[e];
        }
      }
    } else {
      r.template store<float, false>(to, width);
    }
  }

 private:
  typedef float v4 __attribute__((ext_vector_type(4)));
};

// The rows of a team: a part of those of one row of the gate, or those of some.
template <typename T, int R, int V>
__global__ void __launch_bounds__(block_lanes<R>()) norm_grad_kernel(GradArgs p) {
  typedef Row<T, R, V> row_t;
  constexpr uint32_t kTeams = block_lanes<R>() / R;
  const uint64_t team = (uint64_t)blockIdx.x * kTeams + (kTeams > 1 ? threadIdx.x / R : 0);
  if (team >= p.teams) return;
  const uint64_t first = p.per_gate ? team / p.per_gate * p.gate_share + team % p.per_gate * p.rows
                                    : team * p.rows;
  const uint64_t past = p.per_gate ? (team / p.per_gate + 1) * p.gate_share : p.n;
  const uint64_t last = min(min(first + p.rows, past), p.n);
  row_t w, bw, gate;
  w.fill(0.0f), bw.fill(1.0f), gate.fill(1.0f);
  // the longest rows' factors are read again for each row, and two of their sums are in LDS, for want of registers (2048 x
  // 16384 bf16 186 us, 333 with all in registers, which spills)
  constexpr bool kKeep = R < 1024 || V == 1, kLong = R == 1024 && V * row_t::kN > 8;
  __shared__ float long_sums[kLong ? 2 * R * V * row_t::kN : 1];
  Sums<T, R, V, kLong> dbranch_weight, dgate;
  Sums<T, R, V, false> dweight;
  dbranch_weight.clear(long_sums), dgate.clear(long_sums + (kLong ? R * V * row_t::kN : 0)), dweight.clear(nullptr);
  const auto factors = [&](row_t& to, const void* from) {
    if (from) to.template load<false>((const T*)from, p.width);
  };
  if (kKeep) {
    factors(w, p.weight);
    factors(bw, p.branch_weight);
  }
  const float mean = 1.0f / (float)p.width;
  int turn = 0;
  // the next row's values are under way while a row is summed
  Raw<T, V> d_raw = {}, y_raw = {}, z_raw = {}, x_raw = {};
  const auto branch_of = [&](uint64_t row) {
    return row_t::template fetch<true>((const T*)p.branch + row * p.branch_stride, p.width);
  };
  const auto fetch = [&](uint64_t row) {
    if (p.dsum) d_raw = row_t::template fetch<true>((const T*)p.dsum + row * p.dsum_stride, p.width);
    if (p.branch && !kLong) y_raw = branch_of(row);
    if (p.weight) {
      z_raw = row_t::template fetch<true>((const T*)p.dnormed + row * p.dnormed_stride, p.width);
      x_raw = row_t::template fetch<true>((const T*)p.sum + row * p.sum_stride, p.width);
    }
  };
  constexpr bool kAhead = R < 1024;
  if (kAhead && first < last) fetch(first);
  for (uint64_t row = first; row < last; ++row) {
    if (!kAhead) fetch(row);
    if (p.gate && kKeep && (row == first || row % p.gate_share == 0))
      factors(gate, (const T*)p.gate + row / p.gate_share * p.width);
    row_t d, y, dz, x;
    d.take(d_raw), dz.take(z_raw), x.take(x_raw);
    if (!kLong) y.take(y_raw);
    if (kAhead && row + 1 < last) fetch(row + 1);
    if (p.weight) {
      const float root = gp(p.rstd)[row];
      float s = 0.0f;
      if (!kKeep) factors(w, p.weight);
      row_t::each([&](int v, int e) {
        x.x[v][e] *= root;
        dweight.r.x[v][e] = __builtin_fmaf(dz.x[v][e], x.x[v][e], dweight.r.x[v][e]);
        dz.x[v][e] *= w.x[v][e];
        s = __builtin_fmaf(dz.x[v][e], x.x[v][e], s);
      });
      s = team_sum<R>(s, turn) * mean;
      row_t::each([&](int v, int e) { d.x[v][e] += root * (dz.x[v][e] - x.x[v][e] * s); });
    }
    d.template store<T, false>((T*)p.dresidual + row * p.width, p.width);
    if (p.branch) {
      if (kLong) y.take(branch_of(row));
      const float root = p.branch_weight ? gp(p.branch_rstd)[row] : 1.0f;
      float s = 0.0f;
      if (!kKeep) {
        factors(bw, p.branch_weight);
        if (p.gate) factors(gate, (const T*)p.gate + row / p.gate_share * p.width);
      }
      row_t::each([&](int v, int e) {
        y.x[v][e] *= root;
        d.x[v][e] *= p.scale;
      });
      if (p.gate_parts || p.dgate) dgate.add([&](int v, int e) { return d.x[v][e] * (y.x[v][e] * bw.x[v][e]); });
      row_t::each([&](int v, int e) { d.x[v][e] *= gate.x[v][e]; });
      if (p.branch_parts) dbranch_weight.add([&](int v, int e) { return d.x[v][e] * y.x[v][e]; });
      row_t::each([&](int v, int e) {
        d.x[v][e] *= bw.x[v][e];
        s = __builtin_fmaf(d.x[v][e], y.x[v][e], s);
      });
      if (p.branch_weight) {
        s = team_sum<R>(s, turn) * mean;
        row_t::each([&](int v, int e) { d.x[v][e] = root * (d.x[v][e] - y.x[v][e] * s); });
      }
      d.template store<T, false>((T*)p.dbranch + row * p.width, p.width);
      if (p.dgate && (row + 1) % p.gate_share == 0) {
        dgate.store(p.dgate + row / p.gate_share * p.width, p.width);
        dgate.fill();
      }
    }
  }
  if (p.gate_parts) dgate.store(p.gate_parts + team * p.width, p.width);
  if (p.branch_parts) dbranch_weight.store(p.branch_parts + team * p.width, p.width);
  if (p.weight_parts) dweight.store(p.weight_parts + team * p.width, p.width);
}

// out[i] = the sum of `each` rows of parts from row i * each on, 64 columns a workgroup, 16 rows at a time.
struct JoinArgs {
  const float* parts[3];
  float* out[3];
  uint64_t each[3];
  uint32_t blocks[3];   // of rows of out times columns
  uint32_t width, columns;
};
constexpr int kJoinLanes = 1024;

__global__ void __launch_bounds__(kJoinLanes) join_parts_kernel(JoinArgs p) {
  uint32_t b = blockIdx.x;
  int which = 0;
  while (which < 2 && b >= p.blocks[which]) b -= p.blocks[which++];
  const uint64_t out_row = b / p.columns;
  const uint32_t c = b % p.columns * 64 + threadIdx.x % 64;
  constexpr int kRows = kJoinLanes / 64;
  float sum = 0.0f;
  if (c < p.width) {
    const float* from = p.parts[which] + out_row * p.each[which] * p.width + c;
#pragma unroll 8
    for (uint64_t i = threadIdx.x / 64; i < p.each[which]; i += kRows) sum += gp(from)[i * p.width];
  }
  __shared__ float shared[kRows][64];
  shared[threadIdx.x / 64][threadIdx.x % 64] = sum;
  __syncthreads();
  if (threadIdx.x < 64 && c < p.width) {
    for (int r = 1; r < kRows; ++r) sum += shared[r][threadIdx.x];
    gp(p.out[which])[out_row * p.width + c] = sum;
  }
}

// The teams' lanes and groups a lane for a row; f(lanes, groups), as constants.  Forward two groups a lane pay (16384 x
// 1000 bf16 28.8 us against 33.6 with one, 8192 x 4096 47.3 against 48.6), backward one (fewer registers: 1024 x 4096
// 21.0 us against 21.9).
template <typename T, bool PAIRS, typename F>
void with_team(uint32_t width, F f) {
  const uint32_t groups = (width + Group<T>::kN - 1) / Group<T>::kN;
  const auto run = [&](auto lanes, auto per_lane) { f(lanes, per_lane); };
  constexpr auto one = std::integral_constant<int, 1>();
  if (groups <= 64)
    run(std::integral_constant<int, 64>(), one);
  else if (groups <= 128)
    run(std::integral_constant<int, PAIRS ? 64 : 128>(), std::integral_constant<int, PAIRS ? 2 : 1>());
  else if (groups <= 256)
    run(std::integral_constant<int, 256>(), one);
  else if (groups <= 512)
    run(std::integral_constant<int, PAIRS ? 256 : 512>(), std::integral_constant<int, PAIRS ? 2 : 1>());
  else if (groups <= 1024)
    run(std::integral_constant<int, 1024>(), one);
  else if (groups <= 2048)
    run(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
  else if constexpr (sizeof(T) == 4)
    run(std::integral_constant<int, 1024>(), std::integral_constant<int, 4>());
}

// Teams for n rows: each row its own up to 256 (one for each CU), then four rows a team and more, as the partials are
// as large as the rows; and as many as the CUs hold (16384 x 2048 bf16: 1024 teams 83 us, 512 101; 16384 x 1000: 2048 teams
// 63 us, 1024 82).
constexpr uint64_t kLeastTeams = 256, kTeamRows = 4;

constexpr uint64_t most_teams(uint32_t width) { return width <= 512 ? 4096 : width <= 1024 ? 2048 : 1024; }

struct Split {
  uint64_t teams, per_gate, rows, gates;
  bool direct;   // each team covers whole rows of the gate
};

// Teams for n rows, of which gate_share each share a row of the gate.
Split split_rows(uint64_t n, uint64_t gate_share, uint32_t width) {
  Split s = {};
  const uint64_t most = std::min(most_teams(width), std::max(kLeastTeams, n / kTeamRows));
  s.gates = n / gate_share;
  s.direct = s.gates > most / 2;
  if (s.direct) {   // a run of whole gate rows each
    const uint64_t gates = (s.gates + most - 1) / most;
    s.rows = gates * gate_share;
    s.teams = (s.gates + gates - 1) / gates;
  } else {
    s.per_gate = std::max<uint64_t>(1, std::min(gate_share, most / s.gates));
    s.rows = (gate_share + s.per_gate - 1) / s.per_gate;
    s.per_gate = (gate_share + s.rows - 1) / s.rows;
    s.teams = s.gates * s.per_gate;
  }
  return s;
}

int check_rows(int type, uint64_t n, uint32_t width, uint64_t gate_rows) {
  if (!known_type(type) || !width) return EC_EINVAL;
  if (n && gate_rows && n % gate_rows) return EC_EINVAL;
  if (width > kMostWidth || n >= 1ull << 31) return EC_ERANGE;
  return EC_OK;
}

// Launches of at most 2^32 lanes: rows of one workgroup at the largest.
template <int R>
constexpr uint64_t most_blocks() {
  return max_grid(block_lanes<R>());
}

}  // namespace
}  // namespace ec

using namespace ec;

extern "C" {

int ec_residual_norm(const void* d_residual, uint64_t residual_stride, const void* d_branch,
                     uint64_t branch_stride, int type, uint64_t n, uint32_t width, const void* d_gate,
                     uint64_t gate_rows, float scale, const void* d_branch_weight,
                     const void* d_weight, float eps, void* d_sum, uint64_t sum_stride, void* d_normed,
                     float* d_rstd, float* d_branch_rstd, ec_stream_t stream) {
  if (!d_gate) gate_rows = 1;
  if (const int st = check_rows(type, n, width, gate_rows)) return st;
  if (!gate_rows || !std::isfinite(scale) || !(eps >= 0.0f) || !std::isfinite(eps)) return EC_EINVAL;
  if (!d_branch && (d_gate || d_branch_weight || !d_weight)) return EC_EINVAL;
  if (residual_stride < width || (d_branch && (branch_stride < width || sum_stride < width))) return EC_EINVAL;
  if (!n) return EC_OK;
  if (!d_residual || (d_branch && !d_sum) || (d_weight && !d_normed)) return EC_EINVAL;
  const auto st = (hipStream_t)stream;
  return with_type(type, [&](auto t) {
    typedef decltype(t) T;
    with_team<T, true>(width, [&](auto lanes, auto groups) {
      constexpr int R = decltype(lanes)::value, V = decltype(groups)::value;
      constexpr uint64_t kTeams = block_lanes<R>() / R;
      for (uint64_t row = 0; row < n;) {   // as many launches as the grid's limit asks for
        const uint64_t blocks = std::min((n - row + kTeams - 1) / kTeams, most_blocks<R>());
        NormArgs p = {};
        p.residual = d_residual, p.branch = d_branch, p.first = row;
        p.gate = d_gate, p.branch_weight = d_branch_weight, p.weight = d_weight;
        p.residual_stride = residual_stride, p.branch_stride = branch_stride;
        p.n = n, p.gate_share = n / gate_rows, p.width = width;
        p.scale = scale, p.eps = eps;
        p.sum = d_sum, p.sum_stride = sum_stride, p.normed = d_normed;
        p.rstd = d_rstd, p.branch_rstd = d_branch_rstd;
        norm_kernel<T, R, V><<<(uint32_t)blocks, block_lanes<R>(), 0, st>>>(p);
        row += blocks * kTeams;
      }
    });
    return launched();
  });
}

uint64_t ec_residual_norm_grad_workspace(uint64_t n, uint32_t width, uint64_t gate_rows) {
  if (check_rows(EC_F32, n, width, gate_rows) != EC_OK || !n) return 0;
  return 3 * split_rows(n, n / std::max<uint64_t>(1, gate_rows), width).teams * width * sizeof(float);
}

int ec_residual_norm_grad(const void* d_dsum, uint64_t dsum_stride, const void* d_dnormed,
                          uint64_t dnormed_stride, const void* d_sum, uint64_t sum_stride,
                          const void* d_branch, uint64_t branch_stride, int type, uint64_t n,
                          uint32_t width, const float* d_rstd, const float* d_branch_rstd,
                          const void* d_gate, uint64_t gate_rows, float scale,
                          const void* d_branch_weight, const void* d_weight, void* d_dresidual,
                          void* d_dbranch, float* d_dgate, float* d_dbranch_weight, float* d_dweight,
                          void* d_work, uint64_t work_bytes, ec_stream_t stream) {
  if (!d_gate) gate_rows = 1;
  if (const int st = check_rows(type, n, width, gate_rows)) return st;
  if (!gate_rows || !std::isfinite(scale)) return EC_EINVAL;
  if (!d_branch && (d_gate || d_branch_weight)) return EC_EINVAL;
  if (!d_weight != !d_dweight || !d_branch_weight != !d_dbranch_weight || !d_gate != !d_dgate) return EC_EINVAL;
  if (!d_weight && !d_dsum) return EC_EINVAL;
  if ((d_dsum && dsum_stride < width) || (d_weight && (dnormed_stride < width || sum_stride < width)) ||
      (d_branch && branch_stride < width))
    return EC_EINVAL;
  // without rows there may be any number of the gate's, whose gradients are zeros, as far as one launch goes
  if (!n && gate_rows > max_grid(kJoinLanes) / ((width + 63) / 64) - 2) return EC_ERANGE;
  const auto st = (hipStream_t)stream;
  if (n) {
    if (!d_dresidual || (d_branch && !d_dbranch)) return EC_EINVAL;
    if (d_weight && (!d_dnormed || !d_sum || !d_rstd)) return EC_EINVAL;
    if (d_branch_weight && !d_branch_rstd) return EC_EINVAL;
    if (!d_work || work_bytes < ec_residual_norm_grad_workspace(n, width, gate_rows)) return EC_EINVAL;
    if ((uintptr_t)d_work & 15u) return EC_EALIGN;
  }
  const Split s = n ? split_rows(n, n / gate_rows, width) : Split{0, 1, 0, gate_rows, false};
  float* parts = (float*)d_work;
  const uint64_t area = s.teams * width;
  GradArgs p = {};
  p.dsum = d_dsum, p.dnormed = d_dnormed, p.sum = d_sum, p.branch = d_branch;
  p.gate = d_gate, p.branch_weight = d_branch_weight, p.weight = d_weight;
  p.dsum_stride = dsum_stride, p.dnormed_stride = dnormed_stride;
  p.sum_stride = sum_stride, p.branch_stride = branch_stride;
  p.n = n, p.gate_share = n ? n / gate_rows : 1, p.width = width, p.scale = scale;
  p.rstd = d_rstd, p.branch_rstd = d_branch_rstd;
  p.dresidual = d_dresidual, p.dbranch = d_dbranch;
  p.dgate = d_gate && s.direct ? d_dgate : nullptr;
  p.gate_parts = d_gate && !s.direct ? parts : nullptr;
  p.branch_parts = d_branch_weight ? parts + area : nullptr;
  p.weight_parts = d_weight ? parts + 2 * area : nullptr;
  p.teams = s.teams, p.per_gate = s.per_gate, p.rows = s.rows;
  if (n)
    with_type(type, [&](auto t) {
      typedef decltype(t) T;
      with_team<T, false>(width, [&](auto lanes, auto groups) {
        constexpr int R = decltype(lanes)::value, V = decltype(groups)::value;
        constexpr uint64_t kTeams = block_lanes<R>() / R;
        norm_grad_kernel<T, R, V><<<(uint32_t)((s.teams + kTeams - 1) / kTeams), block_lanes<R>(), 0, st>>>(p);
      });
      return EC_OK;
    });
  JoinArgs j = {};
  j.width = width, j.columns = (width + 63) / 64;
  uint32_t blocks = 0;
  const auto join = [&](int i, const float* from, float* to, uint64_t out_rows, uint64_t each) {
    j.parts[i] = from, j.out[i] = to, j.each[i] = each;
    j.blocks[i] = (uint32_t)out_rows * j.columns;
    blocks += j.blocks[i];
  };
  if (d_gate && !s.direct) join(0, parts, d_dgate, s.gates, s.teams ? s.per_gate : 0);
  if (d_branch_weight) join(1, parts + area, d_dbranch_weight, 1, s.teams);
  if (d_weight) join(2, parts + 2 * area, d_dweight, 1, s.teams);
  if (blocks) join_parts_kernel<<<blocks, kJoinLanes, 0, st>>>(j);
  return launched();
}

}  // extern "C"
