// Log probabilities of given tokens with the rows' entropy and their most likely alternatives, the gradient of the
// first two, and the same on vocabulary shards.
//
// With m = max x, S = sum exp(x - m) and W = sum exp(x - m) (x - m) of a row:
//   log-sum-exp l = m + log S,   log p_t = (x_t - m) - log S,   entropy H = -sum p log p = log S - W / S.
// (m, S, W) of two parts of a row merge like the running maximum and sum of a softmax, W' = f (W + (m - m') S) with
// f = exp(m - m'), so one pass over the logits gives all three, and parts of a row (column segments, the shards of
// several devices) are merged by the same formula afterwards.
#include "hk_common.h"

#include <algorithm>
#include <type_traits>

namespace hk {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_huge_valf();
// differences of logits are cut here where they enter a product: exp() of it is 0, and 0 * -inf would be NaN
constexpr float kFarBelow = -1e4f;
constexpr int kMaxTop = 32;          // alternatives of a row
constexpr int kMaxShards = 64;       // lists that one wavefront merges
constexpr int kMaxSplits = 8;        // parts of a row
constexpr int kMaxCandidates = 512;

// (m, S, W) of some elements, S and W taken in the log2 domain against M = fl(m log2(e)): S = sum 2^t, W = sum 2^t t with
// t = x log2(e) - M, one multiply-add per element.  The rounding of M is common to all of them and drops out of what is
// made of S and W; towards other (m, S, W), t moves by a difference of two Ms.
struct LogprobTuple {
  static constexpr int K = 3;
  float v[3];
  static __device__ __forceinline__ LogprobTuple identity() { return LogprobTuple{{kNegInf, 0.f, 0.f}}; }
  // (finite below: an empty maximum; a maximum whose M is past the range of fp32 on either side goes to row_max_count)
  static __device__ __forceinline__ float base(float m) { return fmaxf(m * kLog2e, -kLog2Bound); }
  __device__ __forceinline__ void rebase(float from, float to) {
    const float d = fmaxf(from - to, kFarBelow), f = __builtin_amdgcn_exp2f(d);
    v[2] = f * fmaf(d, v[1], v[2]);
    v[1] *= f;
  }
  static __device__ __forceinline__ LogprobTuple merge(LogprobTuple a, LogprobTuple b) {
    const float m = fmaxf(a.v[0], b.v[0]), to = base(m);
    a.rebase(base(a.v[0]), to);
    b.rebase(base(b.v[0]), to);
    return LogprobTuple{{m, a.v[1] + b.v[1], a.v[2] + b.v[2]}};
  }
  // N more elements, whose maximum is m
  template <int N>
  __device__ __forceinline__ void add(const float* f, float m) {
    m = fmaxf(v[0], m);
    const float to = base(m);
    rebase(base(v[0]), to);
    v[0] = m;
    float s[2] = {v[1], 0.f}, w[2] = {v[2], 0.f};
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float t = fmaf(f[e], kLog2e, -to), x = __builtin_amdgcn_exp2f(t);
      s[e & 1] += x;
      w[e & 1] = fmaf(x, fmaxf(t, kFarBelow), w[e & 1]);
    }
    v[1] = s[0] + s[1];
    v[2] = w[0] + w[1];
  }
};
template <int N>
__device__ __forceinline__ float max_of(const float* f) {
  static_assert(N % 2 == 0, "pairs of elements per max3");
  float m = fmaxf(f[0], f[1]);
#pragma unroll
  for (int e = 2; e < N; e += 2) m = max3(m, f[e], f[e + 1]);
  return m;
}

// (m, S, W) as they go from device to device: S and W against m itself
struct LogprobStats {
  static constexpr int K = 3;
  float v[3];
  static __device__ __forceinline__ LogprobStats identity() { return LogprobStats{{kNegInf, 0.f, 0.f}}; }
  __device__ __forceinline__ void rebase(float to) {   // to: finite, or +inf, which ends in NaN
    const float d = fmaxf(v[0] - to, kFarBelow), f = __builtin_amdgcn_exp2f(d * kLog2e);
    v[2] = f * fmaf(d, v[1], v[2]);
    v[1] *= f;
  }
  static __device__ __forceinline__ LogprobStats merge(LogprobStats a, LogprobStats b) {
    const float m = fmaxf(a.v[0], b.v[0]), to = m == kNegInf ? 0.f : m;
    a.rebase(to);
    b.rebase(to);
    return LogprobStats{{m, a.v[1] + b.v[1], a.v[2] + b.v[2]}};
  }
};

// unsigned numbers in the order of the floats, the two zeros alike
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = f2u(f + 0.f);
  return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}
constexpr uint32_t kKeyNegInf = 0x007fffffu;

struct LogprobArgs {
  const void* logits;
  const int64_t* tokens;
  float *logprob, *entropy, *lse;   // MODE 0; MODE 1: logprob = stats, [splits, 4, rows]
  float* top_value;                 // [rows, top]; MODE 1: [splits, rows, top]
  int64_t* top_token;
  int64_t x_pitch, ignored_index, vocab_start;
  int rows, cols, seg;              // seg: columns of a workgroup's part of the row
  uint16_t threads;
  uint16_t top;
};
static_assert(sizeof(LogprobArgs) <= kCheapArgs, "");

// The columns [0, cols) of one part of a row as the 16-byte vectors that lie on 16-byte boundaries and, RAGGED, up to
// N - 1 elements before and after them, one of which each of the first 2 N threads takes.
template <typename T, bool RAGGED>
struct PartSpan {
  static constexpr int N = VecIO<T>::N;
  const T* row;
  int head, nvec, edge;
  __device__ __forceinline__ PartSpan(const T* row_, int cols, int t) : row(row_), head(0), nvec(cols / N), edge(-1) {
    if constexpr (RAGGED) {
      const int past = int(reinterpret_cast<uintptr_t>(row) & 15u) / int(sizeof(T));
      head = min((N - past) & (N - 1), cols);
      nvec = (cols - head) / N;
      const int rest = head + nvec * N, k = t - N;
      if (t < head) edge = t;
      else if (k >= 0 && k < cols - rest) edge = rest + k;
    }
  }
  __device__ __forceinline__ int column(int v) const { return head + v * N; }
  __device__ __forceinline__ u32x4 load(int v) const { return ld16(row + column(v)); }
  __device__ __forceinline__ u32x4 load_again(int v) const { return ld16_keep(row + column(v)); }
};

// Alternatives.  While the row streams by, a thread writes down the maximum of every few of its vectors.  Then the k-th
// largest of 64 groups' maxima (group l: lane l of every wavefront) is a lower bound of the row's k-th largest value; its
// leading bits are found by bisection.  The runs of vectors whose maximum reaches it, some k + k^2 / 128 of them, are shared
// out over the workgroup and read again, a vector a lane, all at once; elements that reach the bound become candidates, in
// any order, and a candidate's place is the number of candidates before it.
constexpr int kMaxSlots = 8;          // runs of vectors of a thread
constexpr int kMaxRuns = 256;
struct TopShared {
  __align__(16) uint32_t key[kMaxCandidates];
  __align__(16) int col[kMaxCandidates];
  float lane_max[8][kWave];           // of at most 512 threads
  uint16_t run[kMaxRuns];             // slot * 1024 + thread
  uint32_t runs, count;
};

// Bound by memory: 16384 x 32000 bf16 with 8 alternatives 180 us, without 164, of 150 that reading takes at 7 TB/s; the
// difference of the two is the bisection and the second look at the runs, which other workgroups' reading hides in part.
// MODE 0: one workgroup per row, final values.  MODE 1: workgroup (part, row) leaves the statistics and the alternatives
// of a part of the row.  TOP: with alternatives.
template <typename T, bool RAGGED, int MODE, bool TOP>
__global__ __launch_bounds__(512, 8)
void token_logprob_kernel(LogprobArgs a) {
  constexpr int VEC = VecIO<T>::N, U = sizeof(T) == 2 ? 4 : 8;
  __shared__ float red[kMaxWaves * 3];
  extern __shared__ __align__(16) float run_max[];   // TOP: [slots][threads]
  const int t = int(threadIdx.x), threads = a.threads, nwaves = threads >> 6;
  const int row = MODE ? int(blockIdx.y) : int(blockIdx.x);
  float* const top_value = TOP ? a.top_value + ((MODE ? int64_t(blockIdx.x) * a.rows : 0) + row) * a.top : nullptr;
  int64_t* const top_token = TOP ? a.top_token + ((MODE ? int64_t(blockIdx.x) * a.rows : 0) + row) * a.top : nullptr;
  float* const stats = MODE ? a.logprob + int64_t(blockIdx.x) * 4 * a.rows + row : nullptr;

  const int64_t token = a.tokens[row];
  if (token == a.ignored_index) {   // uniform
    if (TOP && t < a.top) {
      top_value[t] = kNegInf;
      top_token[t] = -1;
    }
    if (t == 0) {
      if constexpr (MODE) {
        stats[0] = kNegInf;
        stats[a.rows] = stats[2 * int64_t(a.rows)] = stats[3 * int64_t(a.rows)] = 0.f;
      } else {
        if (a.logprob) a.logprob[row] = 0.f;
        if (a.entropy) a.entropy[row] = 0.f;
        if (a.lse) a.lse[row] = 0.f;
      }
    }
    return;
  }
  const int first = MODE ? int(blockIdx.x) * a.seg : 0;
  const int cols = MODE ? min(a.seg, a.cols - first) : a.cols;
  const T* xr = static_cast<const T*>(a.logits) + int64_t(row) * a.x_pitch + first;
  const PartSpan<T, RAGGED> span(xr, cols, t);

  LogprobTuple p = LogprobTuple::identity();
  float edge = kNegInf;
  if constexpr (RAGGED) {
    if (span.edge >= 0) edge = Cvt<T>::load(xr + span.edge);
  }
  // rounds of U vectors a thread, `per_slot` of which share a maximum
  const int round = U * threads;
  [[maybe_unused]] const int per_slot = TOP ? (span.nvec + round * kMaxSlots - 1) / (round * kMaxSlots) : 0;
  [[maybe_unused]] int slot = 0, in_slot = 0;
  [[maybe_unused]] float cur = kNegInf;
  auto note = [&](float m) {
    if constexpr (TOP) {
      cur = fmaxf(cur, m);
      if (++in_slot == per_slot) {   // uniform
        run_max[slot++ * threads + t] = cur;
        in_slot = 0;
        cur = kNegInf;
      }
    }
  };
  int v = 0;
#pragma nounroll
  for (; v + round <= span.nvec; v += round) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = span.load(v + u * threads + t);
    float f[U * VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) VecIO<T>::unpack(raw[u], &f[u * VEC]);
    const float m = max_of<U * VEC>(f);
    p.template add<U * VEC>(f, m);
    note(m);
  }
  if (v < span.nvec) {   // what is left, a vector a thread at a time
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw[u] = neg_inf_vec<T>();
      if (v + u * threads + t < span.nvec) raw[u] = span.load(v + u * threads + t);
    }
    float most = kNegInf;
    if (v + (U - 1) * threads < span.nvec) {   // uniform: all of them in some thread
      float f[U * VEC];
#pragma unroll
      for (int u = 0; u < U; ++u) VecIO<T>::unpack(raw[u], &f[u * VEC]);
      most = max_of<U * VEC>(f);
      p.template add<U * VEC>(f, most);
    } else {
#pragma unroll
      for (int u = 0; u < U - 1; ++u) {
        if (v + u * threads < span.nvec) {   // uniform
          float f[VEC];
          VecIO<T>::unpack(raw[u], f);
          const float m = max_of<VEC>(f);
          p.template add<VEC>(f, m);
          most = fmaxf(most, m);
        }
      }
    }
    note(most);
  }
  if constexpr (TOP) {
    if (in_slot) run_max[slot++ * threads + t] = cur;   // uniform
  }
  if constexpr (RAGGED) p.template add<1>(&edge, edge);

  [[maybe_unused]] const float mine = p.v[0];   // the maximum of this thread's elements
  p = group_allreduce_tuple(p, red, 0, nwaves);
  float m = p.v[0], s = p.v[1], w = p.v[2], off = 0.f;   // off: the rounding of M
  if (__builtin_expect(m != kNegInf && !(fabsf(m * kLog2e) < kLog2Bound), 0)) {   // uniform; a NaN is none
    s = row_max_count<T>(xr, cols, t, threads, [&](auto x) { __syncthreads(); return group_allreduce_tuple(x, red, 0, nwaves); }, m);
    w = 0.f;
  } else if (m != kNegInf) {
    off = fmaf(m, kLog2e, -LogprobTuple::base(m));
  }
  const float log_s = logf(s) - off * kLn2, lse = m + log_s;
  if (t == 0) {
    const int64_t local = token - a.vocab_start - first;
    const bool inside = local >= 0 && local < cols;
    const float picked = inside ? Cvt<T>::load(xr + local) : 0.f;
    if constexpr (MODE) {
      const float f = __builtin_amdgcn_exp2f(-off);
      stats[0] = m;
      stats[a.rows] = s * f;
      stats[2 * int64_t(a.rows)] = kLn2 * f * fmaf(-off, s, w);
      stats[3 * int64_t(a.rows)] = picked;
    } else {
      // m - picked first: the difference of two logits is (nearly) exact however large their common offset is
      if (a.logprob) a.logprob[row] = inside ? (picked - m) - log_s : __builtin_nanf("");
      if (a.entropy) a.entropy[row] = logf(s) - kLn2 * (w / s);
      if (a.lse) a.lse[row] = lse;
    }
  }

  if constexpr (TOP) {
    constexpr int kBits = sizeof(T) == 4 ? 24 : std::is_same<T, bf16>::value ? 16 : 20;
    __shared__ TopShared sh;
    const int lane = t & 63;
    sh.lane_max[t >> 6][lane] = mine;
    if (t == 0) sh.runs = sh.count = 0;
    __syncthreads();
    float g = kNegInf;
    for (int i = 0; i < nwaves; ++i) g = fmaxf(g, sh.lane_max[i][lane]);
    const uint32_t gk = order_key(g);
    uint32_t bound = 0;
#pragma unroll
    for (int b = 31; b >= 32 - kBits; --b) {
      const uint32_t at = bound | (1u << b);
      if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(gk >= at)) >= int(a.top)) bound = at;
    }
    bound = max(bound, kKeyNegInf + 1);          // an element of -inf is no alternative
    // (places in the lists: one atomic a thread, whatever it has to put there; their order does not matter)
    auto offer = [&](auto elements, const float* f, int col) {
      constexpr int N = decltype(elements)::value;
      uint32_t k[N];
      int n = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        k[j] = f[j] == f[j] ? order_key(f[j]) : 0u;
        n += k[j] >= bound ? 1 : 0;
      }
      if (n == 0) return;
      uint32_t i = atomicAdd(&sh.count, uint32_t(n));
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (k[j] >= bound) {
          if (i < kMaxCandidates) { sh.key[i] = k[j]; sh.col[i] = col + j; }
          ++i;
        }
    };
    if (order_key(mine) >= bound) {
      uint32_t reach = 0;
#pragma unroll
      for (int i = 0; i < kMaxSlots; ++i)
        if (i < slot && order_key(run_max[i * threads + t]) >= bound) reach |= 1u << i;
      if (reach) {
        uint32_t r = atomicAdd(&sh.runs, uint32_t(__builtin_popcount(reach)));
        for (; reach; reach &= reach - 1, ++r)
          if (r < kMaxRuns) sh.run[r] = uint16_t(__builtin_ctz(reach) * 1024 + t);
      }
      if (RAGGED && span.edge >= 0) offer(std::integral_constant<int, 1>{}, &edge, span.edge);
    }
    __syncthreads();
    const int runs = int(sh.runs);
    if (runs <= kMaxRuns) {
      const int each = per_slot * U;   // vectors of a run
      for (int i = t; i < runs * each; i += threads) {
        const int r = i / each, k = i - r * each, at = sh.run[r];
        const int vec = ((at >> 10) * each + k) * threads + (at & 1023);
        if (vec < span.nvec) {
          float f[VEC];
          VecIO<T>::unpack(span.load_again(vec), f);
          offer(std::integral_constant<int, VEC>{}, f, span.column(vec));
        }
      }
    }
    __syncthreads();
    const int n = int(sh.count);
    const bool none = MODE == 0 && !(fabsf(lse) < __builtin_huge_valf());   // no probabilities: no alternatives
    const float base = MODE ? 0.f : lse;
    const int64_t number0 = a.vocab_start + first;
    if (t < a.top && (none || (t >= n && runs <= kMaxRuns))) {
      top_value[t] = none ? __builtin_nanf("") : kNegInf;
      top_token[t] = -1;
    }
    if (none) return;
    auto put = [&](int place, uint32_t key, int col) {
      const float f = u2f(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
      top_value[place] = f - base;
      top_token[place] = number0 + col;
    };
    if (n <= kMaxCandidates && runs <= kMaxRuns) {
      for (int i = t; i < n; i += threads) {
        const uint32_t k = sh.key[i];
        const int c = sh.col[i];
        int place = 0;
        for (int j = 0; j < n; j += 4) {   // four at a time; what stands behind the n-th is not counted
          const u32x4 ks = *reinterpret_cast<const u32x4*>(&sh.key[j]), cs = *reinterpret_cast<const u32x4*>(&sh.col[j]);
#pragma unroll
          for (int q = 0; q < 4; ++q) place += (j + q < n && (ks[q] > k || (ks[q] == k && int(cs[q]) < c))) ? 1 : 0;
        }
        if (place < a.top) put(place, k, c);
      }
      return;
    }
    // More elements than that share the largest values (a row of equal logits): one after the other, each time the
    // best behind the last one over all elements.
    uint32_t last_key = 0xffffffffu;
    int last_col = -1;
    for (int place = 0; place < a.top; ++place) {
      uint32_t best = 0;
      int best_col = 0x7fffffff;
      auto look = [&](float f, int col) {
        const uint32_t k = order_key(f);
        const bool behind = k < last_key || (k == last_key && col > last_col);
        if (f == f && behind && (k > best || (k == best && col < best_col))) { best = k; best_col = col; }
      };
      for (int i = t; i < span.nvec; i += threads) {
        float f[VEC];
        VecIO<T>::unpack(span.load_again(i), f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) look(f[j], span.column(i) + j);
      }
      if (RAGGED && span.edge >= 0) look(edge, span.edge);
      __syncthreads();   // the count, the candidates and the last round's result have been read
      if (t == 0) { sh.count = 0; sh.col[0] = 0x7fffffff; }
      __syncthreads();
      atomicMax(&sh.count, best);
      __syncthreads();
      if (best == sh.count) atomicMin(&sh.col[0], best_col);
      __syncthreads();
      last_key = sh.count;
      last_col = sh.col[0];
      if (t == 0) put(place, last_key, last_col);
    }
  }
}

// ---------------------------------------------------------------------------
// Parts of rows merged: stats [n, 4, rows], alternatives [n, rows, top], sorted lists.  A wavefront per row with
// alternatives or for few rows, a thread per row otherwise.  Final values (logprob, entropy, lse), or,
// with out_stats, the statistics of the merged part.
// ---------------------------------------------------------------------------
struct LogprobCombineArgs {
  const float* stats;
  const float* in_value;
  const int64_t* in_token;
  const int64_t* tokens;
  float *logprob, *entropy, *lse, *out_stats;
  float* top_value;
  int64_t* top_token;
  int64_t ignored_index;
  int64_t vocab_size;    // tokens outside [0, vocab_size) have no logit; < 0: unknown
  int rows;
  uint16_t n, top;
};
static_assert(sizeof(LogprobCombineArgs) <= kCheapArgs, "");

template <bool WAVE>
__global__ __launch_bounds__(WAVE ? 64 : 256)
void token_logprob_combine_kernel(LogprobCombineArgs a) {
  extern __shared__ __align__(16) unsigned char lists[];   // tokens int64_t [n * top], then keys uint32_t [n * top]
  const int row = WAVE ? int(blockIdx.x) : int(blockIdx.x) * 256 + int(threadIdx.x);
  if (row >= a.rows) return;
  const int lane = WAVE ? int(threadIdx.x) : 0;
  const int64_t R = a.rows;
  const int64_t token = a.tokens[row];
  const bool ignored = token == a.ignored_index;
  LogprobStats p = LogprobStats::identity();
  float picked = 0.f;
  if constexpr (WAVE) {
    if (lane < a.n) {
      const float* s = a.stats + lane * 4 * R + row;
      p = LogprobStats{{s[0], s[R], s[2 * R]}};
      picked = s[3 * R];
    }
    p = wave_allreduce_tuple(p);
    SumTuple<1> one{{picked}};
    picked = wave_allreduce_tuple(one).v[0];
  } else {
    for (int k = 0; k < a.n; ++k) {
      const float* s = a.stats + k * 4 * R + row;
      p = LogprobStats::merge(p, LogprobStats{{s[0], s[R], s[2 * R]}});
      picked += s[3 * R];
    }
  }
  const float log_s = logf(p.v[1]), lse = p.v[0] + log_s;
  if (lane == 0) {
    if (a.out_stats) {
      a.out_stats[row] = p.v[0];
      a.out_stats[R + row] = p.v[1];
      a.out_stats[2 * R + row] = p.v[2];
      a.out_stats[3 * R + row] = picked;
    } else {
      const bool outside = token < 0 || (a.vocab_size >= 0 && token >= a.vocab_size);
      if (a.logprob) a.logprob[row] = ignored ? 0.f : outside ? __builtin_nanf("") : (picked - p.v[0]) - log_s;
      if (a.entropy) a.entropy[row] = ignored ? 0.f : log_s - p.v[2] / p.v[1];
      if (a.lse) a.lse[row] = ignored ? 0.f : lse;
    }
  }
  if constexpr (WAVE) {
    if (a.top == 0) return;   // uniform
    const int total = a.n * a.top, each = (total + kWave - 1) / kWave;
    int64_t* const lt = reinterpret_cast<int64_t*>(lists);
    uint32_t* const lk = reinterpret_cast<uint32_t*>(lt + total);
    const bool none = !ignored && !a.out_stats && !(fabsf(lse) < __builtin_huge_valf());
    const float base = a.out_stats ? 0.f : lse;
    float* const value = a.top_value + int64_t(row) * a.top;
    int64_t* const number = a.top_token + int64_t(row) * a.top;
    auto put = [&](int place, uint32_t k, int64_t tok) {
      value[place] = u2f(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)) - base;
      number[place] = tok;
    };
    auto fill = [&](int found) {
      if (lane < a.top && lane >= found) {
        value[lane] = none ? __builtin_nanf("") : kNegInf;
        number[lane] = -1;
      }
    };
    // a key of 0: no alternative
    if (total <= kWave) {   // uniform: one a lane, each one's place among them
      uint32_t k = 0;
      int64_t tok = -1;
      if (lane < total) {
        const int64_t at = (int64_t(lane / a.top) * R + row) * a.top + lane % a.top;
        tok = a.in_token[at];
        k = none || ignored || tok < 0 ? 0 : order_key(a.in_value[at]);
      }
      int place = 0;
#pragma unroll 4
      for (int j = 0; j < total; ++j) {
        const uint32_t kj = __builtin_amdgcn_readlane(int(k), j);
        const int64_t tj = int64_t(uint64_t(uint32_t(__builtin_amdgcn_readlane(int(tok >> 32), j))) << 32 |
                                   uint32_t(__builtin_amdgcn_readlane(int(tok), j)));
        place += (kj > k || (kj == k && tj < tok)) ? 1 : 0;
      }
      if (k != 0 && place < a.top) put(place, k, tok);
      fill(__builtin_popcountll(__builtin_amdgcn_ballot_w64(k != 0)));
      return;
    }
    constexpr int KEEP = 4;                 // keys that a lane keeps; the rest stay in LDS
    uint32_t key[KEEP] = {};
    for (int j = 0; j < each; ++j) {
      const int i = j * kWave + lane;
      if (i < total) {
        const int64_t at = (int64_t(i / a.top) * R + row) * a.top + i % a.top;
        const int64_t tok = a.in_token[at];
        const uint32_t k = none || ignored || tok < 0 ? 0 : order_key(a.in_value[at]);
        lt[i] = tok;
        lk[i] = k;
        static_for<KEEP>([&](auto q) { if (j == q) key[q] = k; });
      }
    }
    __syncthreads();
    // the k-th largest key by bisection, and how many reach it
    uint32_t bound = 0;
    for (int b = 31; b >= 0; --b) {
      const uint32_t at = bound | (1u << b);
      int n = 0;
#pragma unroll
      for (int q = 0; q < KEEP; ++q) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[q] >= at));
      for (int j = KEEP; j < each; ++j)
        n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(j * kWave + lane < total && lk[j * kWave + lane] >= at));
      if (n >= int(a.top)) bound = at;
      if (n == int(a.top)) break;   // uniform
    }
    bound = max(bound, 1u);
    // those, moved to the front of the list, and each one's place among them
    int left = 0;
    for (int j = 0; j < each; ++j) {
      const int i = j * kWave + lane;
      const uint32_t k = i < total ? lk[i] : 0;
      const int64_t tok = i < total ? lt[i] : 0;
      const uint64_t mask = __builtin_amdgcn_ballot_w64(k >= bound);
      __syncthreads();   // (a place that is written was read in this step or before it)
      if (k >= bound) {
        const int to = left + __builtin_popcountll(mask & ((uint64_t(1) << lane) - 1));
        lk[to] = k;
        lt[to] = tok;
      }
      left += __builtin_popcountll(mask);
      __syncthreads();
    }
    for (int i = lane; i < left; i += kWave) {
      const uint32_t k = lk[i];
      const int64_t tok = lt[i];
      int place = 0;
      for (int j = 0; j < left; ++j) place += (lk[j] > k || (lk[j] == k && lt[j] < tok)) ? 1 : 0;
      if (place < a.top) put(place, k, tok);
    }
    fill(left);
  }
}

// ---------------------------------------------------------------------------
// gradient: dx_j = g ([j = token] - p_j) - h p_j (log p_j + H),  p_j = exp(x_j - lse).  Element by element, bound by memory
// (16384 x 32000 bf16: 318 us, what a copy of as many bytes takes 301).  A thread takes one vector, of rows that begin anywhere
// two, whose first and last lines of memory two workgroups share; us with 64 / 128 / 256 threads: 16384 x 32000 bf16 343 / 330 /
// 333, 4096 x 32000 fp32 159 / 168 / 164; ragged 8192 x 50257 bf16 one vector 335 / - / 284, two - / - / 273.
// ---------------------------------------------------------------------------
struct LogprobBwdArgs {
  const void* logits;
  const int64_t* tokens;
  const float *lse, *entropy, *g, *h;
  void* out;
  int64_t x_pitch, out_pitch, ignored_index, vocab_start;
  int cols, seg, segs;   // a workgroup takes `seg` columns of a row, a row has `segs` workgroups
  uint16_t threads;
};
static_assert(sizeof(LogprobBwdArgs) <= kCheapArgs, "");

template <typename T, bool RAGGED, bool ENTROPY>
__global__ __launch_bounds__(256)
void token_logprob_bwd_kernel(LogprobBwdArgs a) {
  constexpr int VEC = VecIO<T>::N, U = RAGGED ? 2 : 1;
  const int t = int(threadIdx.x), threads = a.threads;
  const uint32_t row = blockIdx.x / uint32_t(a.segs);
  const int first = int(blockIdx.x - row * uint32_t(a.segs)) * a.seg, cols = min(a.seg, a.cols - first);
  T* const outr = static_cast<T*>(a.out) + int64_t(row) * a.out_pitch + first;
  const int64_t token = a.tokens[row];
  auto store = [&](T* at, const float* f) {
    if constexpr (RAGGED) st16_any(at, VecIO<T>::pack(f));
    else st16_stream(at, VecIO<T>::pack(f));
  };
  if (token == a.ignored_index) {   // uniform
    const PartSpan<T, RAGGED> span(outr, cols, t);
    const float zero[VEC] = {};
    for (int v = t; v < span.nvec; v += threads) store(outr + span.column(v), zero);
    if (RAGGED && span.edge >= 0) Cvt<T>::store(outr + span.edge, 0.f);
    return;
  }
  const T* const xr = static_cast<const T*>(a.logits) + int64_t(row) * a.x_pitch + first;
  const PartSpan<T, RAGGED> span(xr, cols, t);
  u32x4 raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int v = u * threads + t;
    if (v < span.nvec) raw[u] = span.load(v);
  }
  const float lse = a.lse[row], g = a.g ? a.g[row] : 0.f;
  const float h = ENTROPY ? a.h[row] : 0.f;
  // dx = p (c0 - h log p) + g [j = token],  c0 = -g - h H
  const float c0 = ENTROPY ? -fmaf(h, a.entropy[row], g) : -g;
  const int64_t local = token - a.vocab_start - first;
  const int hit = local >= 0 && local < cols ? int(local) : -1;
  auto grad = [&](float x, int col) {
    const float lp = x - lse, p = __builtin_amdgcn_exp2f(lp * kLog2e);
    float o = ENTROPY ? p * fmaf(-h, fmaxf(lp, kFarBelow), c0) : p * c0;
    return col == hit ? o + g : o;
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int v = u * threads + t;
    if (v < span.nvec) {
      float f[VEC];
      const int c = span.column(v);
      VecIO<T>::unpack(raw[u], f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = grad(f[j], c + j);
      store(outr + c, f);
    }
  }
  if (RAGGED && span.edge >= 0) Cvt<T>::store(outr + span.edge, grad(Cvt<T>::load(xr + span.edge), span.edge));
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// How a forward call is laid out: `splits` parts of `seg` columns (whole vectors of 16 bytes), `threads` per workgroup.
// Parts, one launch and the launch that merges them / one launch, us: where rows are fewer than compute units and a part still
// has 2048 vectors (bf16, 8 parts, 1 row of 50257 5.5 / 6.4, of 131072 6.1 / 10.1; 4 parts, 64 rows of 131072 8.8 / 12.5; not
// for 256 rows: 16.3 / 13.7); with alternatives 32768 (the lists cost as much again: 1 row of 50257 with 20, 4 parts 17.4 / 10.4;
// of 131072 fp32, 8 parts 16.8 / 14.9).
// Threads: what fills the chip with rows wants small workgroups, some 32 vectors a thread, which come and go independently
// (16384 x 32000 bf16 with 64 / 128 / 256 / 512 threads 168 / 164 / 159 / 187 us, with 8 alternatives 195 / 179 / 180 / 218;
// 8192 x 50257 131 / 137 / 130 / 150 and 170 / 156 / 144 / 166; 16384 x 12565 68 / 69 / 81 / 121 and 95 / 87 / 111 / 163; 16384
// x 4000 fp16 29 / 30 / 45 / 82 and, from 128 on, 45 / 67 / 126).  Fewer rows than compute units: as many as have 4 vectors.
struct LogprobPlan {
  int splits, seg, threads;
};
static int pow2_at_least(int64_t n) {
  int p = 64;
  while (p < n && p < 512) p *= 2;
  return p;
}
static LogprobPlan plan_logprob(int64_t rows, int64_t cols, int vec, int64_t top) {
  LogprobPlan p;
  const int64_t nvec = (cols + vec - 1) / vec, cus = device_cu_count();
  p.splits = 1;
  const int64_t part = top ? 32768 : 2048;   // vectors
  if (nvec >= 2 * part)
    p.splits = int(std::max<int64_t>(1, std::min<int64_t>({nvec / part, cus / std::max<int64_t>(rows, 1), kMaxSplits})));
  const int64_t per = (nvec + p.splits - 1) / p.splits;
  p.seg = int(std::min<int64_t>(per * vec, 0x7fffffff));
  p.splits = int((cols + p.seg - 1) / p.seg);
  p.threads = rows * p.splits <= cus ? std::max(128, pow2_at_least(per / 4)) : std::min(256, std::max(top ? 128 : 64, pow2_at_least(per / 32)));
  return p;
}
static size_t logprob_workspace(const LogprobPlan& p, int64_t rows, int top) {
  return p.splits == 1 ? 0 : size_t(p.splits) * size_t(rows) * (size_t(top) * 12 + 16);
}

// (a wavefront per row of few: it reads the parts side by side; 64 rows of 8 parts without alternatives 5.6 us instead of 12.7)
static int launch_combine(const LogprobCombineArgs& a, hipStream_t s) {
  if (a.top || a.rows <= 1024) {
    const int64_t at_once = int64_t(1) << 25;   // a launch's threads fit 32 bits
    for (int64_t r = 0; r < a.rows; r += at_once) {
      LogprobCombineArgs b = a;   // rows stays: it is the step between the parts
      b.stats += r; b.tokens += r;
      if (b.logprob) b.logprob += r;
      if (b.entropy) b.entropy += r;
      if (b.lse) b.lse += r;
      if (b.out_stats) b.out_stats += r;
      if (b.top) { b.in_value += r * b.top; b.in_token += r * b.top; b.top_value += r * b.top; b.top_token += r * b.top; }
      HK_LAUNCH((token_logprob_combine_kernel<true>), dim3(unsigned(std::min(at_once, a.rows - r))), dim3(64),
                size_t(a.n) * a.top * 12, s, b);
    }
  } else {
    HK_LAUNCH((token_logprob_combine_kernel<false>), dim3(unsigned((a.rows + 255) / 256)), dim3(256), 0, s, a);
  }
  return launch_check("token_logprob_combine_kernel");
}

static bool is_row_dtype(int dtype) { return dtype == HK_FLOAT32 || dtype == HK_BFLOAT16 || dtype == HK_FLOAT16; }

// rows of a forward call on one device: final values, or (stats != null) the statistics of a shard
static int logprob_forward(const char* name, int dtype, const void* logits, int64_t pitch, const int64_t* tokens,
                           float* logprob, float* entropy, float* lse, float* stats, float* top_value,
                           int64_t* top_token, int64_t top, int64_t rows, int64_t cols, int64_t vocab_start,
                           int64_t ignored_index, void* workspace, size_t workspace_bytes, hkStream_t stream) {
  HK_REQUIRE(is_row_dtype(dtype), HK_ERR_UNSUPPORTED, "%s: not implemented for dtype %d", name, dtype);
  HK_REQUIRE(rows >= 0 && cols >= 1 && top >= 0, HK_ERR_INVALID, "%s: bad shape [%lld, %lld], %lld alternatives", name,
             (long long)rows, (long long)cols, (long long)top);
  HK_REQUIRE(top <= kMaxTop, HK_ERR_INVALID, "%s: at most %d alternatives, %lld asked for", name, kMaxTop, (long long)top);
  HK_REQUIRE(rows <= 0x7fffffffLL && cols <= 0x7ffffff0LL, HK_ERR_INVALID, "%s: rows and columns must fit 31 bits", name);
  if (rows == 0) return HK_OK;
  HK_REQUIRE(logits && tokens && (stats || logprob || entropy || lse || top), HK_ERR_INVALID, "%s: null input/output", name);
  HK_REQUIRE(top == 0 || (top_value && top_token), HK_ERR_INVALID, "%s: null alternatives", name);
  HK_REQUIRE(pitch >= cols, HK_ERR_INVALID, "%s: row pitch %lld below %lld columns", name, (long long)pitch, (long long)cols);
  const int vec = int(16 / dtype_size(dtype));
  const LogprobPlan p = plan_logprob(rows, cols, vec, top);
  const size_t need = logprob_workspace(p, rows, int(top));
  HK_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), HK_ERR_WORKSPACE,
             "%s: workspace of %zu bytes needed, %zu given", name, need, workspace_bytes);
  HK_REQUIRE(need == 0 || (reinterpret_cast<uintptr_t>(workspace) & 7u) == 0, HK_ERR_INVALID,
             "%s: the workspace must lie on an 8-byte boundary", name);
  hipStream_t s = as_hip(stream);
  const bool parts = p.splits > 1;
  LogprobArgs a{};
  a.logits = logits; a.tokens = tokens; a.x_pitch = pitch; a.ignored_index = ignored_index; a.vocab_start = vocab_start;
  a.rows = int(rows); a.cols = int(cols); a.seg = p.seg; a.threads = uint16_t(p.threads); a.top = uint16_t(top);
  a.logprob = logprob; a.entropy = entropy; a.lse = lse; a.top_value = top_value; a.top_token = top_token;
  float* part_stats = nullptr;
  if (parts) {   // tokens first: they are the widest
    const size_t lists = size_t(p.splits) * size_t(rows) * size_t(top);
    a.top_token = static_cast<int64_t*>(workspace);
    a.top_value = reinterpret_cast<float*>(a.top_token + lists);
    part_stats = a.top_value + lists;
    a.logprob = part_stats;
  } else if (stats) {
    a.logprob = stats;
  }
  const bool ragged = cols % vec != 0 || !aligned16(logits) || pitch % vec != 0;
  const bool mode1 = parts || stats;
  // (a part per row and grid line: 65535 rows at a time; a launch's threads fit 32 bits)
  const int64_t at_once = mode1 ? 65535 : (int64_t(1) << 31) / p.threads;
  HK_REQUIRE(!parts || rows <= at_once, HK_ERR_INVALID, "%s: too many rows in parts", name);
  for (int64_t r = 0; r < rows; r += at_once) {
    LogprobArgs b = a;
    // a.rows stays: it is the step between the statistics; what lies per row moves on
    const int64_t n = std::min(at_once, rows - r);
    b.logits = static_cast<const char*>(logits) + r * pitch * int64_t(dtype_size(dtype));
    b.tokens = tokens + r;
    if (a.logprob) b.logprob = a.logprob + r;
    if (a.entropy) b.entropy = a.entropy + r;
    if (a.lse) b.lse = a.lse + r;
    if (top && r) { b.top_value = a.top_value + r * top; b.top_token = a.top_token + r * top; }
    const dim3 grid = mode1 ? dim3(unsigned(p.splits), unsigned(n)) : dim3(unsigned(n));
    const dim3 block{unsigned(p.threads)};
    // (the slots that rows of this length use)
    const int64_t rounds = (p.seg / vec + p.threads * 32 / vec - 1) / (p.threads * 32 / vec) + 1;
    const size_t lds = top ? size_t(std::min<int64_t>(kMaxSlots, rounds)) * p.threads * sizeof(float) : 0;
    profile_before(s);
#define HK_LP(T, RAGGED, MODE, TOP) HK_LAUNCH((token_logprob_kernel<T, RAGGED, MODE, TOP>), grid, block, lds, s, b)
#define HK_LP_TOP(T, RAGGED, MODE) do { if (top) HK_LP(T, RAGGED, MODE, true); else HK_LP(T, RAGGED, MODE, false); } while (0)
#define HK_LP_MODE(T, RAGGED) do { if (mode1) HK_LP_TOP(T, RAGGED, 1); else HK_LP_TOP(T, RAGGED, 0); } while (0)
#define HK_LP_TYPE(T) do { if (ragged) HK_LP_MODE(T, true); else HK_LP_MODE(T, false); } while (0)
    if (dtype == HK_FLOAT32) HK_LP_TYPE(float);
    else if (dtype == HK_BFLOAT16) HK_LP_TYPE(bf16);
    else HK_LP_TYPE(fp16);
#undef HK_LP_TYPE
#undef HK_LP_MODE
#undef HK_LP_TOP
#undef HK_LP
    profile_after(s);
    const int rc = launch_check("token_logprob_kernel");
    if (rc != HK_OK) return rc;
  }
  if (!parts) return HK_OK;
  LogprobCombineArgs c{};
  c.stats = part_stats; c.in_value = a.top_value; c.in_token = a.top_token; c.tokens = tokens;
  c.logprob = logprob; c.entropy = entropy; c.lse = lse; c.out_stats = stats;
  c.top_value = top_value; c.top_token = top_token; c.ignored_index = ignored_index; c.vocab_size = cols;
  c.rows = int(rows); c.n = uint16_t(p.splits); c.top = uint16_t(top);
  return launch_combine(c, s);
}

} // namespace hk

using namespace hk;

extern "C" {

int hk_token_logprob_workspace_bytes(int dtype, int64_t rows, int64_t cols, int64_t top, size_t* bytes) {
  HK_REQUIRE(is_row_dtype(dtype), HK_ERR_UNSUPPORTED, "hk_token_logprob_workspace_bytes: not implemented for dtype %d", dtype);
  HK_REQUIRE(bytes && rows >= 0 && cols >= 1 && top >= 0 && top <= kMaxTop && rows <= 0x7fffffffLL && cols <= 0x7ffffff0LL,
             HK_ERR_INVALID, "hk_token_logprob_workspace_bytes: bad argument");
  *bytes = rows == 0 ? 0 : logprob_workspace(plan_logprob(rows, cols, int(16 / dtype_size(dtype)), top), rows, int(top));
  return HK_OK;
}

int hk_token_logprob_fwd(int dtype, const void* logits, int64_t logits_pitch, const int64_t* tokens, float* logprob,
                         float* entropy, float* lse, float* top_logprob, int64_t* top_token, int64_t top, int64_t rows,
                         int64_t cols, int64_t ignored_index, void* workspace, size_t workspace_bytes, hkStream_t stream) {
  return logprob_forward("hk_token_logprob_fwd", dtype, logits, logits_pitch, tokens, logprob, entropy, lse, nullptr,
                         top_logprob, top_token, top, rows, cols, 0, ignored_index, workspace, workspace_bytes, stream);
}

int hk_vocab_parallel_logprob_stats(int dtype, const void* logits, int64_t logits_pitch, const int64_t* tokens, float* stats,
                                    float* top_value, int64_t* top_token, int64_t top, int64_t rows, int64_t cols,
                                    int64_t vocab_start, int64_t ignored_index, void* workspace, size_t workspace_bytes,
                                    hkStream_t stream) {
  HK_REQUIRE(stats || rows == 0, HK_ERR_INVALID, "hk_vocab_parallel_logprob_stats: null output");
  HK_REQUIRE(vocab_start >= 0, HK_ERR_INVALID, "hk_vocab_parallel_logprob_stats: negative vocab_start");
  return logprob_forward("hk_vocab_parallel_logprob_stats", dtype, logits, logits_pitch, tokens, nullptr, nullptr, nullptr,
                         stats, top_value, top_token, top, rows, cols, vocab_start, ignored_index, workspace,
                         workspace_bytes, stream);
}

int hk_vocab_parallel_logprob_combine(const float* stats, const float* top_values, const int64_t* top_tokens, int64_t nshards,
                                      const int64_t* tokens, int64_t ignored_index, int64_t vocab_size, float* logprob,
                                      float* entropy, float* lse, float* top_logprob, int64_t* top_token, int64_t top,
                                      int64_t rows, hkStream_t stream) {
  HK_REQUIRE(rows >= 0 && rows <= 0x7fffffffLL && nshards >= 1 && top >= 0, HK_ERR_INVALID,
             "hk_vocab_parallel_logprob_combine: bad shape");
  HK_REQUIRE(nshards <= kMaxShards && top <= kMaxTop, HK_ERR_INVALID,
             "hk_vocab_parallel_logprob_combine: at most %d shards and %d alternatives", kMaxShards, kMaxTop);
  if (rows == 0) return HK_OK;
  HK_REQUIRE(stats && tokens && (logprob || entropy || lse || top), HK_ERR_INVALID,
             "hk_vocab_parallel_logprob_combine: null input/output");
  HK_REQUIRE(top == 0 || (top_values && top_tokens && top_logprob && top_token), HK_ERR_INVALID,
             "hk_vocab_parallel_logprob_combine: null alternatives");
  LogprobCombineArgs c{};
  c.stats = stats; c.in_value = top_values; c.in_token = top_tokens; c.tokens = tokens;
  c.logprob = logprob; c.entropy = entropy; c.lse = lse; c.top_value = top_logprob; c.top_token = top_token;
  c.ignored_index = ignored_index; c.vocab_size = vocab_size;
  c.rows = int(rows); c.n = uint16_t(nshards); c.top = uint16_t(top);
  return launch_combine(c, as_hip(stream));
}

int hk_token_logprob_bwd(int dtype, const void* logits, int64_t logits_pitch, const int64_t* tokens, const float* lse,
                         const float* entropy, const float* grad_logprob, const float* grad_entropy, void* dlogits,
                         int64_t dlogits_pitch, int64_t rows, int64_t cols, int64_t vocab_start, int64_t ignored_index,
                         hkStream_t stream) {
  HK_REQUIRE(is_row_dtype(dtype), HK_ERR_UNSUPPORTED, "hk_token_logprob_bwd: not implemented for dtype %d", dtype);
  HK_REQUIRE(rows >= 0 && cols >= 0 && rows <= 0x7fffffffLL && cols <= 0x7ffffff0LL && vocab_start >= 0, HK_ERR_INVALID,
             "hk_token_logprob_bwd: bad shape");
  if (rows == 0 || cols == 0) return HK_OK;
  HK_REQUIRE(logits && tokens && lse && dlogits && (grad_logprob || grad_entropy), HK_ERR_INVALID,
             "hk_token_logprob_bwd: null input/output");
  HK_REQUIRE(!grad_entropy || entropy, HK_ERR_INVALID, "hk_token_logprob_bwd: grad_entropy needs the rows' entropy");
  HK_REQUIRE(logits_pitch >= cols && dlogits_pitch >= cols, HK_ERR_INVALID, "hk_token_logprob_bwd: row pitch below the columns");
  const int vec = int(16 / dtype_size(dtype));
  const bool ragged = cols % vec != 0 || !aligned16(logits) || !aligned16(dlogits) || logits_pitch % vec != 0 ||
                      dlogits_pitch % vec != 0;
  LogprobBwdArgs a{};
  a.logits = logits; a.tokens = tokens; a.lse = lse; a.entropy = entropy; a.g = grad_logprob; a.h = grad_entropy; a.out = dlogits;
  a.x_pitch = logits_pitch; a.out_pitch = dlogits_pitch; a.ignored_index = ignored_index; a.vocab_start = vocab_start;
  a.cols = int(cols);
  const int threads = ragged ? 256 : dtype == HK_FLOAT32 ? 64 : 128;
  a.threads = uint16_t(threads);
  a.seg = (ragged ? 2 : 1) * threads * vec;
  a.segs = int((cols + a.seg - 1) / a.seg);
  hipStream_t s = as_hip(stream);
  const int64_t at_once = std::max<int64_t>(1, (int64_t(1) << 31) / (int64_t(a.segs) * threads));   // a launch's threads fit 32 bits
  for (int64_t r = 0; r < rows; r += at_once) {
    const int64_t n = std::min(at_once, rows - r);
    LogprobBwdArgs b = a;
    const int64_t es = int64_t(dtype_size(dtype));
    b.logits = static_cast<const char*>(logits) + r * logits_pitch * es;
    b.out = static_cast<char*>(dlogits) + r * dlogits_pitch * es;
    b.tokens += r; b.lse += r;
    if (b.entropy) b.entropy += r;
    if (b.g) b.g += r;
    if (b.h) b.h += r;
    const dim3 grid{unsigned(n * a.segs)}, block{unsigned(threads)};
    profile_before(s);
#define HK_LP(T, RAGGED) \
  do { if (grad_entropy) HK_LAUNCH((token_logprob_bwd_kernel<T, RAGGED, true>), grid, block, 0, s, b); \
       else HK_LAUNCH((token_logprob_bwd_kernel<T, RAGGED, false>), grid, block, 0, s, b); } while (0)
#define HK_LP_TYPE(T) do { if (ragged) HK_LP(T, true); else HK_LP(T, false); } while (0)
    if (dtype == HK_FLOAT32) HK_LP_TYPE(float);
    else if (dtype == HK_BFLOAT16) HK_LP_TYPE(bf16);
    else HK_LP_TYPE(fp16);
#undef HK_LP_TYPE
#undef HK_LP
    profile_after(s);
    const int rc = launch_check("token_logprob_bwd_kernel");
    if (rc != HK_OK) return rc;
  }
  return HK_OK;
}

} // extern "C"
