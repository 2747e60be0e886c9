// gradclip.hip — the global L2 norm of many tensors and their clipping to it:
//   norm = sqrt(sum_i sum_j g_i[j]^2),  c = min(1, max_norm / (norm + eps)),  out_i = c g_i.
// What bounds it is memory: every gradient is read for the norm, and read again and written once
// the norm is known.  The squares are summed in 64 bits (gradients of 1e-30 or 1e+30 neither
// vanish nor overflow; a conversion and an fma per element hide behind the loads).
//
// Tensors are cut into chunks of CHUNK elements counted from each tensor's own start, a block per
// chunk, so every partial sum and their order depend on the sizes alone and the norm is the same
// bits wherever the tensors lie.  The table of tensors goes by value in the kernel's arguments
// (CLIP_TABLE of them a launch): a captured graph replays it with nothing to keep alive.
#include <algorithm>
#include <vector>

#include "ops.h"

namespace mpr {
namespace {

constexpr int CHUNK = 32768;
constexpr int CLIP_TABLE = 120;  // 32 bytes each: within the 4 KB of kernel arguments
constexpr int CLIP_THREADS = 256;

struct ClipTable {
  const void* in[CLIP_TABLE];
  void* out[CLIP_TABLE];
  int64_t n[CLIP_TABLE];
  int32_t chunk0[CLIP_TABLE + 1];  // chunks before tensor i (within this launch)
  int32_t types[CLIP_TABLE];       // in | out << 4
  int32_t count;
};

struct ClipState {  // the head of the workspace
  float coef;
  float pad[3];
};

__device__ __forceinline__ int clip_find(const ClipTable& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.chunk0[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <class T>
__device__ __forceinline__ double clip_sumsq(const T* x, int64_t n, int t, int threads) {
  constexpr int V = VEC16<T>;
  double s = 0.0;
  const int64_t nv = n / V;
  for (int64_t i = t; i < nv; i += threads) {
    float f[V];
    load_f<T, V>(x + i * V, f);
#pragma unroll
    for (int e = 0; e < V; ++e) s = fma((double)f[e], (double)f[e], s);
  }
  for (int64_t i = nv * V + t; i < n; i += threads) {
    const double f = to_f<T>(x[i]);
    s = fma(f, f, s);
  }
  return s;
}

__device__ __forceinline__ double clip_sumsq_of(int type, const void* p, int64_t at, int64_t n,
                                                int t, int threads) {
  if (type == MPR_F32) return clip_sumsq(static_cast<const float*>(p) + at, n, t, threads);
  if (type == MPR_BF16) return clip_sumsq(static_cast<const bf16*>(p) + at, n, t, threads);
  return clip_sumsq(static_cast<const f16*>(p) + at, n, t, threads);
}

template <class T, class U>
__device__ __forceinline__ void clip_scale(const T* x, U* y, int64_t n, float c, int t,
                                           int threads) {
  constexpr int V = VEC16<T>;
  const int64_t nv = n / V;
  for (int64_t i = t; i < nv; i += threads) {
    float f[V];
    load_f<T, V>(x + i * V, f);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] *= c;
    store_f<U, V>(y + i * V, f);
  }
  for (int64_t i = nv * V + t; i < n; i += threads) y[i] = from_f<U>(to_f<T>(x[i]) * c);
}

template <class T>
__device__ __forceinline__ void clip_scale_to(int type, const T* x, void* y, int64_t at, int64_t n,
                                              float c, int t, int threads) {
  if (type == MPR_F32) clip_scale(x + at, static_cast<float*>(y) + at, n, c, t, threads);
  else if (type == MPR_BF16) clip_scale(x + at, static_cast<bf16*>(y) + at, n, c, t, threads);
  else clip_scale(x + at, static_cast<f16*>(y) + at, n, c, t, threads);
}

__device__ __forceinline__ void clip_scale_of(int types, const void* x, void* y, int64_t at,
                                              int64_t n, float c, int t, int threads) {
  const int in = types & 15, out = types >> 4;
  if (in == MPR_F32) clip_scale_to(out, static_cast<const float*>(x), y, at, n, c, t, threads);
  else if (in == MPR_BF16) clip_scale_to(out, static_cast<const bf16*>(x), y, at, n, c, t, threads);
  else clip_scale_to(out, static_cast<const f16*>(x), y, at, n, c, t, threads);
}

// the sum of a block's values in a fixed order, in thread 0
template <int THREADS>
__device__ __forceinline__ double block_sum(double v, double* red) {
  const int t = threadIdx.x;
  v = wave_add(v);
  if ((t & 63) == 0) red[t >> 6] = v;
  __syncthreads();
  double s = 0.0;
  if (t == 0)
    for (int w = 0; w < THREADS / 64; ++w) s += red[w];
  return s;
}

__device__ __forceinline__ float clip_coef(double norm, double max_norm, double eps) {
  const double c = max_norm / (norm + eps);  // a NaN norm gives NaN: the gradients show it
  return c > 1.0 ? 1.f : (float)c;
}

__global__ __launch_bounds__(CLIP_THREADS) void clip_norm_kernel(ClipTable tab, double* partial) {
  __shared__ double red[CLIP_THREADS / 64];
  const int c = blockIdx.x, i = clip_find(tab, c);
  const int64_t at = (int64_t)(c - tab.chunk0[i]) * CHUNK;
  const int64_t n = min((int64_t)CHUNK, tab.n[i] - at);
  const double s = block_sum<CLIP_THREADS>(
      clip_sumsq_of(tab.types[i] & 15, tab.in[i], at, n, threadIdx.x, CLIP_THREADS), red);
  if (threadIdx.x == 0) partial[c] = s;
}

__global__ __launch_bounds__(1024) void clip_finish_kernel(const double* partial, int64_t n,
                                                           double max_norm, double eps,
                                                           float* norm, ClipState* st) {
  __shared__ double red[16];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += partial[i];
  s = block_sum<1024>(s, red);
  if (threadIdx.x == 0) {
    const double r = sqrt(s);
    norm[0] = (float)r;
    st->coef = clip_coef(r, max_norm, eps);
  }
}

// The chunks from the last to the first: the norm's pass left the last ones in the caches.  222 M
// gradients (two thirds fp32, the others bf16) into an fp32 buffer: three launches of 114 us, 4.75 TB/s
// read and written together, after 58 us each for the norm, 4.2 TB/s.
__global__ __launch_bounds__(CLIP_THREADS) void clip_scale_kernel(ClipTable tab,
                                                                  const ClipState* st) {
  const float coef = st->coef;
  const int c = gridDim.x - 1 - blockIdx.x, i = clip_find(tab, c);
  if (coef == 1.f && tab.in[i] == tab.out[i]) return;  // in place below the limit: unchanged
  const int64_t at = (int64_t)(c - tab.chunk0[i]) * CHUNK;
  const int64_t n = min((int64_t)CHUNK, tab.n[i] - at);
  clip_scale_of(tab.types[i], tab.in[i], tab.out[i], at, n, coef, threadIdx.x, CLIP_THREADS);
}

// Few values: one block does it all, a wave per unit of ONE_UNIT of them (three launches cost more
// than the reads: 9000 values in 8 tensors 15 us with the host's part, 26 with three).
constexpr int ONE_UNIT = 1024, ONE_UNITS = 128;
__global__ __launch_bounds__(1024) void clip_one_kernel(ClipTable tab, int units, int scale,
                                                        double max_norm, double eps, float* norm) {
  __shared__ double red[16];
  __shared__ float coef;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double s = 0.0;
  for (int u = wave; u < units; u += 16) {
    const int i = clip_find(tab, u);
    const int64_t at = (int64_t)(u - tab.chunk0[i]) * ONE_UNIT;
    const int64_t n = min((int64_t)ONE_UNIT, tab.n[i] - at);
    s += clip_sumsq_of(tab.types[i] & 15, tab.in[i], at, n, lane, 64);
  }
  s = block_sum<1024>(s, red);
  if (threadIdx.x == 0) {
    const double r = sqrt(s);
    norm[0] = (float)r;
    coef = clip_coef(r, max_norm, eps);
  }
  __syncthreads();
  for (int u = wave; scale && u < units; u += 16) {
    const int i = clip_find(tab, u);
    if (coef == 1.f && tab.in[i] == tab.out[i]) continue;
    const int64_t at = (int64_t)(u - tab.chunk0[i]) * ONE_UNIT;
    const int64_t n = min((int64_t)ONE_UNIT, tab.n[i] - at);
    clip_scale_of(tab.types[i], tab.in[i], tab.out[i], at, n, coef, lane, 64);
  }
}

struct Span {
  uintptr_t a, b;
};

// The rest of the tensors' table from item `i` on, at most CLIP_TABLE tensors; returns the next.
int clip_fill(ClipTable& tab, const int64_t* desc, int n, int i, int64_t* chunks,
              int chunk = CHUNK) {
  int64_t c = 0;
  tab.count = 0;
  for (; i < n && tab.count < CLIP_TABLE; ++i) {
    const int64_t* d = desc + 5 * (int64_t)i;
    if (d[1] == 0) continue;
    const int64_t own = cdiv(d[1], chunk);
    if (c + own > MAX_GRID_X) break;
    const int k = tab.count++;
    tab.in[k] = reinterpret_cast<const void*>(d[0]);
    tab.n[k] = d[1];
    tab.out[k] = reinterpret_cast<void*>(d[3]);
    tab.types[k] = (int32_t)(d[2] | (d[4] << 4));
    tab.chunk0[k] = (int32_t)c;
    c += own;
  }
  tab.chunk0[tab.count] = (int32_t)c;
  *chunks = c;
  return i;
}

int64_t clip_chunks(const int64_t* desc, int n) {
  int64_t c = 0;
  for (int i = 0; i < n; ++i) c += cdiv(desc[5 * (int64_t)i + 1], CHUNK);
  return c;
}

// scale: outputs are wanted.  The norm alone reads, and what it reads may overlap.
int clip_check(int n, const int64_t* desc, bool scale) {
  std::vector<Span> spans;
  if (scale) spans.reserve(2 * (size_t)n);
  for (int i = 0; i < n; ++i) {
    const int64_t* d = desc + 5 * (int64_t)i;
    MPR_REQUIRE(d[1] >= 0 && d[1] <= (int64_t)1 << 37, "clip_grads: tensor %d has %lld values", i,
                (long long)d[1]);
    MPR_REQUIRE(d[2] >= 0 && d[2] <= 2 && (!d[3] || (d[4] >= 0 && d[4] <= 2)),
                "clip_grads: tensor %d has dtype codes %lld, %lld", i, (long long)d[2],
                (long long)d[4]);
    if (d[1] == 0) continue;
    MPR_REQUIRE(d[0], "clip_grads: tensor %d is null", i);
    if (!scale) continue;
    MPR_REQUIRE(d[3], "clip_grads: tensor %d has no output", i);
    MPR_REQUIRE(d[3] != d[0] || d[4] == d[2],
                "clip_grads: tensor %d is clipped in place into another type", i);
    const uintptr_t a = (uintptr_t)d[0], o = (uintptr_t)d[3];
    spans.push_back({a, a + (size_t)d[1] * (d[2] == MPR_F32 ? 4 : 2)});
    if (o != a) spans.push_back({o, o + (size_t)d[1] * (d[4] == MPR_F32 ? 4 : 2)});
  }
  std::sort(spans.begin(), spans.end(), [](const Span& x, const Span& y) { return x.a < y.a; });
  for (size_t i = 1; i < spans.size(); ++i)
    MPR_REQUIRE(spans[i].a >= spans[i - 1].b,
                "clip_grads: tensors overlap in memory (the same one twice?)");
  return MPR_OK;
}

}  // namespace
}  // namespace mpr

using namespace mpr;

extern "C" {

int mpr_clip_workspace(int32_t n, const int64_t* desc, int64_t* bytes) {
  return ops_call("clip_workspace", [&]() -> int {
    MPR_REQUIRE(n >= 0 && (n == 0 || desc) && bytes, "clip_workspace: %d tensors", n);
    *bytes = (int64_t)sizeof(ClipState) + 8 * clip_chunks(desc, n);
    return MPR_OK;
  });
}

int mpr_clip_grads(int32_t n, const int64_t* desc, double max_norm, double eps, float* norm,
                   void* ws, int64_t ws_bytes, void* stream) {
  return ops_call("clip_grads", [&]() -> int {
    MPR_REQUIRE(n >= 0 && (n == 0 || desc), "clip_grads: %d tensors", n);
    bool scale = false;
    for (int i = 0; i < n; ++i) scale = scale || desc[5 * (int64_t)i + 3];
    MPR_TRY(clip_check(n, desc, scale));
    MPR_REQUIRE(norm, "clip_grads: no place for the norm");
    const int64_t chunks = clip_chunks(desc, n);
    MPR_REQUIRE(ws && ws_bytes >= (int64_t)sizeof(ClipState) + 8 * chunks,
                "clip_grads: workspace of %lld bytes, %lld needed", (long long)ws_bytes,
                (long long)((int64_t)sizeof(ClipState) + 8 * chunks));
    hipStream_t s = op_stream(stream);
    ClipState* st = static_cast<ClipState*>(ws);
    double* partial = reinterpret_cast<double*>(st + 1);
    ClipTable tab;
    int64_t done = 0, c = 0;
    if (chunks <= ONE_UNITS && clip_fill(tab, desc, n, 0, &c, ONE_UNIT) == n && c <= ONE_UNITS) {
      clip_one_kernel<<<1, 1024, 0, s>>>(tab, (int)c, scale, max_norm, eps, norm);
      MPR_LAUNCHED();
      return MPR_OK;
    }
    std::vector<int> first;  // the tensor that each launch begins with
    for (int i = 0; i < n;) {
      const int from = i;
      i = clip_fill(tab, desc, n, i, &c);
      if (c == 0) continue;
      first.push_back(from);
      clip_norm_kernel<<<dim3((unsigned)c), CLIP_THREADS, 0, s>>>(tab, partial + done);
      MPR_LAUNCHED();
      done += c;
    }
    clip_finish_kernel<<<1, 1024, 0, s>>>(partial, chunks, max_norm, eps, norm, st);
    MPR_LAUNCHED();
    if (!scale) return MPR_OK;  // the norm alone
    for (size_t k = first.size(); k-- > 0;) {
      clip_fill(tab, desc, n, first[k], &c);
      clip_scale_kernel<<<dim3((unsigned)c), CLIP_THREADS, 0, s>>>(tab, st);
      MPR_LAUNCHED();
    }
    return MPR_OK;
  });
}

}  // extern "C"
