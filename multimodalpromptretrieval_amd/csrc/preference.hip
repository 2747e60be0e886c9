// preference.hip — log-probabilities of label sequences and the preference loss of paired answers,
// with their gradients.  For sequence s over T positions with labels y (negative: ignored):
//   lse(x) = m + log sum exp(x - m),      lp_s = sum_t [y >= 0] (x[t, y_t] - lse(x[t]))
//   margin_p = beta ((lp_p - lp_{P+p}) - (ref_p - ref_{P+p}))          (p < P, chosen | rejected)
//   loss = 1/P sum_p -(1 - eps) log sigmoid(margin_p) - eps log sigmoid(-margin_p)
//   dx[s, t, :] = dlp_s (onehot(y_t) - softmax(x[t]));   an ignored position's row: 0, x unread
// Bound by memory: the forward reads the logits of the labelled positions once, the backward reads
// them again and writes every row.  The softmax statistics (m and 1 / sum, fp32) are kept from the
// forward; log-probabilities are summed in 64 bits, so the difference of two long answers keeps its
// digits.  A label >= V gives NaN.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ops.h"

namespace mpr {
namespace {

constexpr int LP_THREADS = 256;
constexpr int LP_MAX_SPLIT = 16;

struct LpArgs {
  const void* labels;
  int labels64;
  int64_t ls;           // label row stride
  int64_t xs, xt;       // logits strides: sequence, position
  int64_t S, T, V;
  int split;
};

__device__ __forceinline__ int64_t lp_label(const LpArgs& a, int64_t s, int64_t t) {
  return a.labels64 ? static_cast<const int64_t*>(a.labels)[s * a.ls + t]
                    : (int64_t)static_cast<const int32_t*>(a.labels)[s * a.ls + t];
}

// running maximum and sum of exp(x - maximum)
struct MaxSum {
  float m, s;
};
__device__ __forceinline__ float exp_from(float x, float m) {
  return __expf(x - (m == -INFINITY ? 0.f : m));
}
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b) {
  const float m = fmaxf(a.m, b.m);
  return {m, a.s * exp_from(a.m, m) + b.s * exp_from(b.m, m)};
}

// what a stats launch leaves: per part of a row, or per row in one part
union LpStat {
  MaxSum* part;
  double* lp;
};
// log softmax at a value v of a row, the terms in fp32, their difference in 64 bits
__device__ __forceinline__ double lp_row(float v, MaxSum c) {
  return (double)(v - c.m) - (double)logf(c.s);
}

// stat[row * split + part] = the maximum and sum over the part's columns; where a row is one part, what
// becomes of them: row_stat and the label's log-probability (0 where it is ignored).  Bound by the read of the
// labelled rows: 8192 rows of 32128 in bf16, five eighths of them labelled (329 MB), 48 us, 6.9 TB/s
// (part of them from the caches); 320 rows of 32101 in fp32 7 us.
template <class T>
__global__ __launch_bounds__(LP_THREADS) void lp_stats_kernel(const T* __restrict__ x, LpArgs a,
                                                              LpStat stat,
                                                              MaxSum* __restrict__ row_stat) {
  constexpr int N = VEC16<T>, U = 4;
  __shared__ MaxSum red[LP_THREADS / 64];
  const int64_t row = blockIdx.x, s = row / a.T, t = row % a.T;
  const int64_t y = lp_label(a, s, t);
  if (y < 0) {
    if (a.split == 1 && threadIdx.x == 0) stat.lp[row] = 0.0;
    return;
  }
  const T* xr = x + s * a.xs + t * a.xt;
  const float at_label = y < a.V ? to_f<T>(xr[y]) : NAN;
  const int64_t nv = a.V / N, per = cdiv(nv, a.split);
  const int64_t lo = blockIdx.y * per, hi = min(nv, lo + per);
  MaxSum c = {-INFINITY, 0.f};
  int64_t i = lo + threadIdx.x;
  const auto step = [&](auto whole) {  // U accesses at once; not whole: those that there are
    float v[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (decltype(whole)::value || i + u * LP_THREADS < hi)
        load_f<T, N>(xr + (i + u * LP_THREADS) * N, v[u]);
      else
#pragma unroll
        for (int e = 0; e < N; ++e) v[u][e] = -INFINITY;
    }
    float m = c.m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) m = fmaxf(m, v[u][e]);
    float sum = c.s * exp_from(c.m, m);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) sum += exp_from(v[u][e], m);
    c = {m, sum};
  };
  for (; i + (U - 1) * LP_THREADS < hi; i += U * LP_THREADS) step(std::true_type{});
  if (i < hi) step(std::false_type{});
  if (blockIdx.y == gridDim.y - 1)
    for (int64_t j = nv * N + threadIdx.x; j < a.V; j += LP_THREADS) {
      const float v = to_f<T>(xr[j]), m = fmaxf(c.m, v);
      c = {m, c.s * exp_from(c.m, m) + exp_from(v, m)};
    }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1)
    c = join(c, MaxSum{__shfl_xor(c.m, off, 64), __shfl_xor(c.s, off, 64)});
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < LP_THREADS / 64; ++w) c = join(c, red[w]);
    if (a.split == 1) {
      row_stat[row] = {c.m, 1.f / c.s};
      stat.lp[row] = lp_row(at_label, c);
    } else {
      stat.part[row * a.split + blockIdx.y] = c;
    }
  }
}

// A thread's share of lp_s in 64 bits, of positions t0, t0 + step, ...; where rows are in parts,
// row_stat[row] = (m, 1 / sum) for the backward
template <class T>
__device__ double lp_share(const T* x, const LpArgs& a, const LpStat& stat, MaxSum* row_stat,
                           int64_t s, int t0, int step) {
  double lp = 0.0;
  if (a.split == 1) {
#pragma unroll 8
    for (int64_t t = t0; t < a.T; t += step) lp += stat.lp[s * a.T + t];
    return lp;
  }
  for (int64_t t = t0; t < a.T; t += step) {
    const int64_t y = lp_label(a, s, t);
    if (y < 0) continue;
    const int64_t row = s * a.T + t;
    const float v = y < a.V ? to_f<T>(x[s * a.xs + t * a.xt + y]) : NAN;
    MaxSum c = stat.part[row * a.split];
    for (int i = 1; i < a.split; ++i) c = join(c, stat.part[row * a.split + i]);
    row_stat[row] = {c.m, 1.f / c.s};
    lp += lp_row(v, c);
  }
  return lp;
}

// lp_s, a block for each
template <class T>
__global__ __launch_bounds__(256) void lp_sequence_kernel(const T* x, LpArgs a, LpStat stat,
                                                          MaxSum* row_stat, float* logps,
                                                          double* logps64) {
  __shared__ double red[4];
  const int64_t s = blockIdx.x;
  const double part = wave_add(lp_share(x, a, stat, row_stat, s, threadIdx.x, 256));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = part;
  __syncthreads();
  if (threadIdx.x == 0) {
    const double lp = (red[0] + red[1]) + (red[2] + red[3]);
    logps[s] = (float)lp;
    logps64[s] = lp;
  }
}

// The pairs of the batch by one block of 1024: loss, and dlp of every sequence for a loss gradient
// of 1.
__device__ __forceinline__ void lp_pairs(const double* lp, const float* ref, int64_t P, double beta,
                                         double eps, float* loss, float* dlp) {
  __shared__ double red[16];
  double sum = 0.0;
  for (int64_t p = threadIdx.x; p < P; p += 1024) {
    const double m = beta * ((lp[p] - lp[P + p]) - ((double)ref[p] - (double)ref[P + p]));
    // -log sigmoid(m) = log(1 + exp(-|m|)) + max(-m, 0);  -log sigmoid(-m) is m more.  An answer with
    // a token that the model rules out has an infinite margin: the term of weight 0 is left out, and
    // the two of a negative margin are one (0 inf and inf - inf would be NaN)
    sum += log1p(exp(-fabs(m))) + (m > 0.0 ? (eps == 0.0 ? 0.0 : eps * m) : (eps - 1.0) * m);
    const double g = beta / (double)P * (eps - 1.0 / (1.0 + exp(m)));
    dlp[p] = (float)g;
    dlp[P + p] = (float)-g;
  }
  sum = wave_add(sum);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) sum += red[w];
    loss[0] = (float)(sum / (double)P);
  }
}

__global__ __launch_bounds__(1024) void lp_pairs_kernel(const double* lp, const float* ref,
                                                        int64_t P, double beta, double eps,
                                                        float* loss, float* dlp) {
  lp_pairs(lp, ref, P, beta, eps, loss, dlp);
}

// Few sequences of few positions: both in one launch, a wave for each sequence in turn (16 sequences of
// 20: 5 us, and a launch of 3.4 us of host time less).
constexpr int LP_FEW = 64;
constexpr int64_t LP_FEW_ROWS = 16384;
template <class T>
__global__ __launch_bounds__(1024) void lp_few_kernel(const T* x, LpArgs a, LpStat stat,
                                                      MaxSum* row_stat, float* logps,
                                                      const float* ref, double beta, double eps,
                                                      float* loss, float* dlp) {
  __shared__ double lp64[LP_FEW];
  const int lane = threadIdx.x & 63;
  for (int s = threadIdx.x >> 6; s < a.S; s += 16) {
    const double lp = wave_add(lp_share(x, a, stat, row_stat, s, lane, 64));
    if (lane == 0) {
      logps[s] = (float)lp;
      lp64[s] = lp;
    }
  }
  __syncthreads();
  lp_pairs(lp64, ref, a.S / 2, beta, eps, loss, dlp);
}

// dx, a block per row (and part of it).  Bound by memory: labelled rows are read again, every row is
// written; the exponentials hide behind that.  The 8192 rows above (329 MB in, 526 MB out) 150 us, 5.7
// TB/s, with stores that pass the caches by (29 us more without: they push out logits still to be read).
template <class T, bool STREAM>
__global__ __launch_bounds__(LP_THREADS) void lp_grad_kernel(const T* __restrict__ x, LpArgs a,
                                                             const MaxSum* __restrict__ row_stat,
                                                             const float* __restrict__ dlp,
                                                             const float* __restrict__ mult,
                                                             T* __restrict__ dx) {
  constexpr int N = VEC16<T>;
  const int64_t row = blockIdx.x, s = row / a.T, t = row % a.T;
  const int64_t y = lp_label(a, s, t);
  T* dr = dx + row * a.V;
  const int64_t nv = a.V / N, per = cdiv(nv, gridDim.y);
  const int64_t lo = blockIdx.y * per, hi = min(nv, lo + per);
  const bool rest = blockIdx.y == gridDim.y - 1;
  if (y < 0) {
    const float z[N] = {};
    for (int64_t i = lo + threadIdx.x; i < hi; i += LP_THREADS) store_f<T, N, STREAM>(dr + i * N, z);
    if (rest)
      for (int64_t j = nv * N + threadIdx.x; j < a.V; j += LP_THREADS) dr[j] = from_f<T>(0.f);
    return;
  }
  const T* xr = x + s * a.xs + t * a.xt;
  const MaxSum st = row_stat[row];
  const float m = st.m == -INFINITY ? 0.f : st.m;
  float g = mult ? dlp[s] * mult[0] : dlp[s];
  if (y >= a.V) g = NAN;
  const float f = -g * st.s;
  for (int64_t i = lo + threadIdx.x; i < hi; i += LP_THREADS) {
    float v[N];
    load_f<T, N>(xr + i * N, v);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = f * __expf(v[e] - m);
    const int64_t at = y - i * N;
    if (at >= 0 && at < N)
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] += e == at ? g : 0.f;
    store_f<T, N, STREAM>(dr + i * N, v);
  }
  if (rest)
    for (int64_t j = nv * N + threadIdx.x; j < a.V; j += LP_THREADS)
      dr[j] = from_f<T>(f * __expf(to_f<T>(xr[j]) - m) + (j == y ? g : 0.f));
}

struct LpPlan {
  int64_t rows, stat, row_stat, lp64, bytes;
  int split;
};

// Parts of a row: enough blocks for the chip where there are few rows, LP_PART columns at least.
constexpr int64_t LP_BLOCKS = 2048, LP_PART = 4096;

LpPlan lp_plan(int64_t S, int64_t T, int64_t V) {
  LpPlan p;
  p.rows = S * T;
  int64_t k = p.rows ? LP_BLOCKS / p.rows : 1;
  k = std::min<int64_t>(k, std::min<int64_t>(LP_MAX_SPLIT, V / LP_PART));
  p.split = (int)std::max<int64_t>(1, k);
  p.lp64 = 0;
  p.stat = p.lp64 + 8 * S;
  p.bytes = p.stat + 8 * p.rows * p.split;
  return p;
}

int lp_check(const char* what, int32_t dtype, int64_t S, int64_t T, int64_t V, int64_t xs,
             int64_t xt, int64_t ls) {
  MPR_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype code %d", what, (int)dtype);
  MPR_REQUIRE(S >= 0 && T >= 0 && S < (int64_t)1 << 31 && T < (int64_t)1 << 31 &&
                  S * T <= MAX_GRID_X,
              "%s: %lld sequences of %lld positions", what, (long long)S, (long long)T);
  MPR_REQUIRE(V >= 1 && V < (int64_t)1 << 31, "%s: a vocabulary of %lld", what, (long long)V);
  MPR_REQUIRE(xs >= 0 && xt >= 0 && ls >= 0, "%s: negative stride", what);
  return MPR_OK;
}

}  // namespace
}  // namespace mpr

using namespace mpr;

extern "C" {

int mpr_logps_workspace(int64_t S, int64_t T, int64_t V, int64_t* bytes) {
  return ops_call("logps_workspace", [&]() -> int {
    MPR_TRY(lp_check("logps_workspace", 0, S, T, V, 0, 0, 0));
    MPR_REQUIRE(bytes, "logps_workspace: null pointer");
    *bytes = lp_plan(S, T, V).bytes;
    return MPR_OK;
  });
}

int mpr_logps_fwd(const void* logits, int32_t dtype, int64_t S, int64_t T, int64_t V, int64_t xs,
                  int64_t xt, const void* labels, int32_t labels64, int64_t ls, float* logps,
                  float* row_stat, const float* ref, double beta, double label_smoothing,
                  float* loss, float* dlogps, void* ws, int64_t ws_bytes, void* stream) {
  return ops_call("logps_fwd", [&]() -> int {
    MPR_TRY(lp_check("logps_fwd", dtype, S, T, V, xs, xt, ls));
    MPR_REQUIRE(!loss || (S > 0 && S % 2 == 0 && ref && dlogps),
                "logps_fwd: a loss needs pairs, reference log-probabilities and dlogps");
    if (S == 0) return MPR_OK;
    const LpPlan p = lp_plan(S, T, V);
    MPR_REQUIRE(logps && (T == 0 || (logits && labels && row_stat)), "logps_fwd: null pointer");
    MPR_REQUIRE(ws && ws_bytes >= p.bytes, "logps_fwd: workspace of %lld bytes, %lld needed",
                (long long)ws_bytes, (long long)p.bytes);
    hipStream_t s = op_stream(stream);
    char* w = static_cast<char*>(ws);
    LpStat stat;
    stat.part = reinterpret_cast<MaxSum*>(w + p.stat);
    const bool few = loss && S <= LP_FEW && p.rows <= LP_FEW_ROWS;
    double* lp64 = reinterpret_cast<double*>(w + p.lp64);
    const LpArgs a{labels, labels64, ls, xs, xt, S, T, V, p.split};
    MPR_TRY(by_dtype(dtype, [&](auto z) -> int {
      using X = decltype(z);
      const X* x = static_cast<const X*>(logits);
      if (p.rows) {
        lp_stats_kernel<X><<<dim3((unsigned)p.rows, p.split), LP_THREADS, 0, s>>>(
            x, a, stat, reinterpret_cast<MaxSum*>(row_stat));
        MPR_LAUNCHED();
      }
      if (few) {
        lp_few_kernel<X><<<1, 1024, 0, s>>>(x, a, stat, reinterpret_cast<MaxSum*>(row_stat), logps,
                                            ref, beta, label_smoothing, loss, dlogps);
        MPR_LAUNCHED();
        return MPR_OK;
      }
      lp_sequence_kernel<X><<<dim3((unsigned)S), 256, 0, s>>>(
          x, a, stat, reinterpret_cast<MaxSum*>(row_stat), logps, lp64);
      MPR_LAUNCHED();
      return MPR_OK;
    }));
    if (!loss || few) return MPR_OK;
    lp_pairs_kernel<<<1, 1024, 0, s>>>(lp64, ref, S / 2, beta, label_smoothing, loss, dlogps);
    MPR_LAUNCHED();
    return MPR_OK;
  });
}

int mpr_logps_bwd(const void* logits, int32_t dtype, int64_t S, int64_t T, int64_t V, int64_t xs,
                  int64_t xt, const void* labels, int32_t labels64, int64_t ls,
                  const float* row_stat, const float* dlogps, const float* mult, void* dlogits,
                  void* stream) {
  return ops_call("logps_bwd", [&]() -> int {
    MPR_TRY(lp_check("logps_bwd", dtype, S, T, V, xs, xt, ls));
    if (S * T == 0) return MPR_OK;
    MPR_REQUIRE(logits && labels && row_stat && dlogps && dlogits, "logps_bwd: null pointer");
    const LpPlan p = lp_plan(S, T, V);
    const LpArgs a{labels, labels64, ls, xs, xt, S, T, V, p.split};
    return by_dtype(dtype, [&](auto z) -> int {
      using X = decltype(z);
      const auto grad = p.rows * V * (int64_t)sizeof(X) >= STREAM_BYTES ? lp_grad_kernel<X, true>
                                                                          : lp_grad_kernel<X, false>;
      grad<<<dim3((unsigned)p.rows, p.split), LP_THREADS, 0, op_stream(stream)>>>(
          static_cast<const X*>(logits), a, reinterpret_cast<const MaxSum*>(row_stat), dlogps,
          mult, static_cast<X*>(dlogits));
      MPR_LAUNCHED();
      return MPR_OK;
    });
  });
}

}  // extern "C"
