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
constexpr float kNegInf = -__builtin_huge_valf();
// differences of logits are cut here where they enter a product: exp() of it is 0, and 0 * -inf would be NaN
constexpr float kFarBelow = -1e4f;
constexpr int kMaxTop = 32;          // alternatives of a row
constexpr int kMaxShards = 64;       // lists that one wavefront merges
constexpr int kMaxCandidates = 512;

struct LogprobTuple {   // (m, S, W)
  static constexpr int K = 3;
  float v[3];
  static __device__ __forceinline__ LogprobTuple identity() { return LogprobTuple{{kNegInf, 0.f, 0.f}}; }
  static __device__ __forceinline__ float finite_or_zero(float m) { return m == kNegInf ? 0.f : m; }
  // this relative to the maximum mg (finite; or +inf, which ends in NaN)
  __device__ __forceinline__ void rebase(float mg) {
    const float d = fmaxf(v[0] - mg, kFarBelow), f = __builtin_amdgcn_exp2f(d * kLog2e);
    v[2] = f * fmaf(d, v[1], v[2]);
    v[1] *= f;
  }
  static __device__ __forceinline__ LogprobTuple merge(LogprobTuple a, LogprobTuple b) {
    const float m = fmaxf(a.v[0], b.v[0]), mg = finite_or_zero(m);
    a.rebase(mg);
    b.rebase(mg);
    return LogprobTuple{{m, a.v[1] + b.v[1], a.v[2] + b.v[2]}};
  }
  // N more elements, taken against the new maximum
  template <int N>
  __device__ __forceinline__ void add(const float* f) {
    float m = v[0];
    if constexpr (N == 1) {
      m = fmaxf(m, f[0]);
    } else {
      static_assert(N % 2 == 0, "pairs of elements per max3");
#pragma unroll
      for (int e = 0; e < N; e += 2) m = max3(m, f[e], f[e + 1]);
    }
    const float mg = finite_or_zero(m);
    rebase(mg);
    v[0] = m;
    float s[2] = {v[1], 0.f}, w[2] = {v[2], 0.f};
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = f[e] - mg, x = __builtin_amdgcn_exp2f(d * kLog2e);
      s[e & 1] += x;
      w[e & 1] = fmaf(x, fmaxf(d, kFarBelow), w[e & 1]);
    }
    v[1] = s[0] + s[1];
    v[2] = w[0] + w[1];
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

// MODE 0: one workgroup per row, final values.  MODE 1: workgroup (part, row) leaves the statistics and the alternatives
// of a part of the row.  TOP: with alternatives.
template <typename T, bool RAGGED, int MODE, bool TOP>
__global__ __launch_bounds__(1024, 8)
void token_logprob_kernel(LogprobArgs a) {
  constexpr int VEC = VecIO<T>::N, U = sizeof(T) == 2 ? 4 : 8;
  __shared__ float red[kMaxWaves * 3];
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
  int v = 0;
#pragma nounroll
  for (; v + U * threads <= span.nvec; v += U * threads) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = span.load(v + u * threads + t);
    float f[U * VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) VecIO<T>::unpack(raw[u], &f[u * VEC]);
    p.template add<U * VEC>(f);
  }
  if (v < span.nvec) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw[u] = neg_inf_vec<T>();
      if (v + u * threads + t < span.nvec) raw[u] = span.load(v + u * threads + t);
    }
    float f[U * VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) VecIO<T>::unpack(raw[u], &f[u * VEC]);
    p.template add<U * VEC>(f);
  }
  if constexpr (RAGGED) p.template add<1>(&edge);

  [[maybe_unused]] const float mine = p.v[0];   // the maximum of this thread's elements
  p = group_allreduce_tuple(p, red, 0, nwaves);
  const float log_s = logf(p.v[1]), lse = p.v[0] + log_s;
  if (t == 0) {
    const int64_t local = token - a.vocab_start - first;
    const bool inside = local >= 0 && local < cols;
    const float picked = inside ? Cvt<T>::load(xr + local) : 0.f;
    if constexpr (MODE) {
      stats[0] = p.v[0];
      stats[a.rows] = p.v[1];
      stats[2 * int64_t(a.rows)] = p.v[2];
      stats[3 * int64_t(a.rows)] = picked;
    } else {
      if (a.logprob) a.logprob[row] = inside ? (picked - p.v[0]) - log_s : __builtin_nanf("");
      if (a.entropy) a.entropy[row] = log_s - p.v[2] / p.v[1];
      if (a.lse) a.lse[row] = lse;
    }
  }

  if constexpr (TOP) {
    // The k-th largest of 64 groups' maxima (lane l of every wavefront) is a lower bound of the row's k-th largest value:
    // its leading bits by bisection.  The threads whose maximum reaches it read their elements again and put those that
    // reach it into a list, some k + k^2 / 128 of them in any order; a candidate's place in the order is the number of
    // candidates before it.
    constexpr int kBits = sizeof(T) == 4 ? 24 : std::is_same<T, bf16>::value ? 16 : 20;
    __shared__ float lane_max[kMaxWaves][kWave];
    __shared__ uint32_t cand_key[kMaxCandidates];
    __shared__ int cand_col[kMaxCandidates];
    __shared__ uint32_t count;
    const int lane = t & 63;
    lane_max[t >> 6][lane] = mine;
    if (t == 0) count = 0;
    __syncthreads();
    float g = kNegInf;
    for (int w = 0; w < nwaves; ++w) g = fmaxf(g, lane_max[w][lane]);
    const uint32_t gk = order_key(g);
    uint32_t bound = 0;
#pragma unroll
    for (int b = 31; b >= 32 - kBits; --b) {
      const uint32_t at = bound | (1u << b);
      if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(gk >= at)) >= int(a.top)) bound = at;
    }
    bound = max(bound, kKeyNegInf + 1);          // an element of -inf is no alternative
    auto offer = [&](float f, int col) {
      const uint32_t k = order_key(f);
      if (k >= bound && f == f) {
        const uint32_t i = atomicAdd(&count, 1u);   // the order does not matter
        if (i < kMaxCandidates) { cand_key[i] = k; cand_col[i] = col; }
      }
    };
    auto each = [&](auto fn) {   // fn(element, column in the part) over this thread's elements
      for (int w = t; w < span.nvec; w += threads) {
        float f[VEC];
        VecIO<T>::unpack(span.load_again(w), f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) fn(f[j], span.column(w) + j);
      }
      if (RAGGED && span.edge >= 0) fn(edge, span.edge);
    };
    if (order_key(mine) >= bound) each(offer);
    __syncthreads();
    const int n = int(count);
    const bool none = MODE == 0 && !(fabsf(lse) < __builtin_huge_valf());   // no probabilities: no alternatives
    const float base = MODE ? 0.f : lse;
    const int64_t number0 = a.vocab_start + first;
    if (t < a.top && (none || t >= n)) {
      top_value[t] = none ? __builtin_nanf("") : kNegInf;
      top_token[t] = -1;
    }
    if (none) return;
    auto put = [&](int place, uint32_t key, int col) {
      const float f = u2f(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
      top_value[place] = f - base;
      top_token[place] = number0 + col;
    };
    if (n <= kMaxCandidates) {
      for (int i = t; i < n; i += threads) {
        const uint32_t k = cand_key[i];
        const int c = cand_col[i];
        int place = 0;
        for (int j = 0; j < n; ++j) place += (cand_key[j] > k || (cand_key[j] == k && cand_col[j] < c)) ? 1 : 0;
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
      each([&](float f, int col) {
        const uint32_t k = order_key(f);
        const bool behind = k < last_key || (k == last_key && col > last_col);
        if (f == f && behind && (k > best || (k == best && col < best_col))) { best = k; best_col = col; }
      });
      __syncthreads();   // count, the candidates and the last round's result are read
      if (t == 0) { count = 0; cand_col[0] = 0x7fffffff; }
      __syncthreads();
      atomicMax(&count, best);
      __syncthreads();
      if (best == count) atomicMin(&cand_col[0], best_col);
      __syncthreads();
      last_key = count;
      last_col = cand_col[0];
      if (t == 0) put(place, last_key, last_col);
    }
  }
}

// ---------------------------------------------------------------------------
// Parts of rows merged: stats [n, 4, rows], alternatives [n, rows, top], sorted lists.  A wavefront per row with
// alternatives (lane i holds the head of list i), a thread per row without.  Final values (logprob, entropy, lse), or,
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

template <bool TOP>
__global__ __launch_bounds__(TOP ? 64 : 256)
void token_logprob_combine_kernel(LogprobCombineArgs a) {
  extern __shared__ __align__(16) unsigned char lists[];   // TOP: int64_t [n * top], then float [n * top]
  const int row = TOP ? int(blockIdx.x) : int(blockIdx.x) * 256 + int(threadIdx.x);
  if (row >= a.rows) return;
  const int lane = TOP ? int(threadIdx.x) : 0;
  const int64_t R = a.rows;
  const int64_t token = a.tokens[row];
  const bool ignored = token == a.ignored_index;
  LogprobTuple p = LogprobTuple::identity();
  float picked = 0.f;
  if constexpr (TOP) {
    if (lane < a.n) {
      const float* s = a.stats + lane * 4 * R + row;
      p = LogprobTuple{{s[0], s[R], s[2 * R]}};
      picked = s[3 * R];
    }
    p = wave_allreduce_tuple(p);
    SumTuple<1> one{{picked}};
    picked = wave_allreduce_tuple(one).v[0];
  } else {
    for (int k = 0; k < a.n; ++k) {
      const float* s = a.stats + k * 4 * R + row;
      p = LogprobTuple::merge(p, LogprobTuple{{s[0], s[R], s[2 * R]}});
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
  if constexpr (TOP) {
    int64_t* lt = reinterpret_cast<int64_t*>(lists);
    float* lv = reinterpret_cast<float*>(lt + a.n * a.top);
    const int total = a.n * a.top;
    for (int i = lane; i < total; i += kWave) {
      const int64_t at = (int64_t(i / a.top) * R + row) * a.top + i % a.top;
      lv[i] = a.in_value[at];
      lt[i] = a.in_token[at];
    }
    __syncthreads();
    const bool none = !ignored && !a.out_stats && !(fabsf(lse) < __builtin_huge_valf());
    const float base = a.out_stats ? 0.f : lse;
    int head = 0;
    for (int place = 0; place < a.top; ++place) {
      const bool have = !none && !ignored && lane < a.n && head < a.top && lt[lane * a.top + head] >= 0;
      const float v = have ? lv[lane * a.top + head] : kNegInf;
      const int64_t tok = have ? lt[lane * a.top + head] : 0x7fffffffffffffffLL;
      const float best = wave_allreduce_tuple(MaxTuple{{v}}).v[0];
      int64_t winner = have && v == best ? tok : 0x7fffffffffffffffLL;
#pragma unroll
      for (int s = 1; s < kWave; s *= 2) {
        const int64_t o = __shfl_xor(winner, s, kWave);
        winner = o < winner ? o : winner;
      }
      const bool found = winner != 0x7fffffffffffffffLL;   // uniform
      if (have && tok == winner && v == best) ++head;
      if (lane == 0) {
        a.top_value[int64_t(row) * a.top + place] = found ? best - base : none ? __builtin_nanf("") : kNegInf;
        a.top_token[int64_t(row) * a.top + place] = found ? winner : -1;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// gradient: dx_j = g ([j = token] - p_j) - h p_j (log p_j + H),  p_j = exp(x_j - lse)
// ---------------------------------------------------------------------------
struct LogprobBwdArgs {
  const void* logits;
  const int64_t* tokens;
  const float *lse, *entropy, *g, *h;
  void* out;
  int64_t x_pitch, out_pitch, ignored_index, vocab_start;
  int cols, seg, segs;   // a workgroup takes `seg` columns of a row, a row has `segs` workgroups
};
static_assert(sizeof(LogprobBwdArgs) <= kCheapArgs, "");

constexpr int kBwdThreads = 256;

template <typename T, bool RAGGED, bool ENTROPY>
__global__ __launch_bounds__(kBwdThreads)
void token_logprob_bwd_kernel(LogprobBwdArgs a) {
  constexpr int VEC = VecIO<T>::N;
  const int t = int(threadIdx.x);
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
    for (int v = t; v < span.nvec; v += kBwdThreads) store(outr + span.column(v), zero);
    if (RAGGED && span.edge >= 0) Cvt<T>::store(outr + span.edge, 0.f);
    return;
  }
  const T* const xr = static_cast<const T*>(a.logits) + int64_t(row) * a.x_pitch + first;
  const PartSpan<T, RAGGED> span(xr, cols, t);
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
  for (int v = t; v < span.nvec; v += kBwdThreads) {
    float f[VEC];
    const int c = span.column(v);
    VecIO<T>::unpack(span.load(v), f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = grad(f[j], c + j);
    store(outr + c, f);
  }
  if (RAGGED && span.edge >= 0) Cvt<T>::store(outr + span.edge, grad(Cvt<T>::load(xr + span.edge), span.edge));
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// How a forward call is laid out: `splits` parts of `seg` columns (whole vectors of 16 bytes), `threads` per workgroup.
struct LogprobPlan {
  int splits, seg, threads;
};
static LogprobPlan plan_logprob(int64_t rows, int64_t cols, int vec) {
  LogprobPlan p;
  const int64_t nvec = (cols + vec - 1) / vec;
  p.splits = 1;
  const int64_t want = 2 * int64_t(device_cu_count());
  if (rows < want) {
    const int64_t most = std::min<int64_t>(kMaxShards, (nvec + 1023) / 1024);
    p.splits = int(std::max<int64_t>(1, std::min(most, want / std::max<int64_t>(rows, 1))));
  }
  const int64_t per = (nvec + p.splits - 1) / p.splits;
  p.seg = int(std::min<int64_t>(per * vec, 0x7fffffff));
  p.splits = int((cols + p.seg - 1) / p.seg);
  p.threads = int(std::min<int64_t>(1024, std::max<int64_t>(64, ((per + 3) / 4 + 63) / 64 * 64)));
  return p;
}
static size_t logprob_workspace(const LogprobPlan& p, int64_t rows, int top) {
  return p.splits == 1 ? 0 : size_t(p.splits) * size_t(rows) * (size_t(top) * 12 + 16);
}

static int launch_combine(const LogprobCombineArgs& a, hipStream_t s) {
  if (a.top) {
    HK_LAUNCH((token_logprob_combine_kernel<true>), dim3(unsigned(a.rows)), dim3(64), size_t(a.n) * a.top * 12, s, a);
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
  const LogprobPlan p = plan_logprob(rows, cols, vec);
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
  // (a part per row and grid line: 65535 rows at a time)
  const int64_t at_once = mode1 ? 65535 : rows;
  HK_REQUIRE(!parts || rows <= at_once, HK_ERR_INVALID, "%s: too many rows in parts", name);
  for (int64_t r = 0; r < rows; r += at_once) {
    LogprobArgs b = a;
    // a.rows stays: it is the step between the statistics; what lies per row moves on
    const int64_t n = std::min(at_once, rows - r);
    b.logits = static_cast<const char*>(logits) + r * pitch * int64_t(dtype_size(dtype));
    b.tokens = tokens + r;
    if (mode1) b.logprob = a.logprob + r;
    if (top && r) { b.top_value = a.top_value + r * top; b.top_token = a.top_token + r * top; }
    const dim3 grid = mode1 ? dim3(unsigned(p.splits), unsigned(n)) : dim3(unsigned(n));
    const dim3 block{unsigned(p.threads)};
    profile_before(s);
#define HK_LP(T, RAGGED, MODE, TOP) HK_LAUNCH((token_logprob_kernel<T, RAGGED, MODE, TOP>), grid, block, 0, s, b)
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
  *bytes = rows == 0 ? 0 : logprob_workspace(plan_logprob(rows, cols, int(16 / dtype_size(dtype))), rows, int(top));
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
  const int64_t nvec = (cols + vec - 1) / vec;
  const int64_t parts = (nvec + 4 * kBwdThreads - 1) / (4 * kBwdThreads), per = (nvec + parts - 1) / parts;
  a.seg = int(std::min<int64_t>(per * vec, 0x7fffffff));
  a.segs = int((cols + a.seg - 1) / a.seg);
  hipStream_t s = as_hip(stream);
  const int64_t at_once = std::max<int64_t>(1, 0x7fffffffLL / a.segs);   // workgroups of a launch fit 31 bits
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
    const dim3 grid{unsigned(n * a.segs)}, block{unsigned(kBwdThreads)};
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
