// embed.hip — the scaled embedding lookup and its gradient by sorted tokens.
//   out[i, :] = scale * W[ids[i], :]           dW[v, :] = scale * sum_{i: ids[i] = v} dout[i, :]
// Both are bound by memory: the lookup writes n rows and reads at most V, the gradient reads n
// rows and writes V.  The gradient needs the positions of each token together: they are sorted by
// token with a stable radix sort (so a token's rows are summed in the order of their positions, and
// two runs give the same bits), then each wave sums a window of the sorted positions.  A token
// whose rows cross windows (padding, a full stop) is finished by a second kernel from the
// windows' fp32 partial sums, in window order.
//
// An id outside [0, V) reads nothing: its output row is NaN, and it has no gradient.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ops.h"

namespace mpr {
namespace {

// ---- lookup --------------------------------------------------------------------------------------
// Bound by the writes of n rows (the table's rows that repeat come from the caches).  A wave copies
// LOOKUP_ROWS rows side by side, each lane 16 bytes of each, so that the gathers of one hide those of
// the others.  262144 rows of 1024 in bf16 (537 MB out, streamed past the caches) 146 us, 3.7 TB/s of
// writes alone; 8992 rows of 768 in fp32 10 us, 2.8 TB/s.
constexpr int LOOKUP_ROWS = 4;  // rows a wave has in flight

template <class T, class I, bool STREAM>
__global__ __launch_bounds__(256) void embed_lookup_kernel(const T* __restrict__ table, int64_t V,
                                                           int64_t ld, const I* __restrict__ ids,
                                                           int64_t n, int d, float scale,
                                                           T* __restrict__ out) {
  constexpr int N = VEC16<T>;
  const int lane = threadIdx.x & 63, nv = d / N;
  for (int64_t r0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * LOOKUP_ROWS; r0 < n;
       r0 += (int64_t)gridDim.x * 4 * LOOKUP_ROWS) {
    int64_t id[LOOKUP_ROWS];
#pragma unroll
    for (int r = 0; r < LOOKUP_ROWS; ++r) {
      id[r] = r0 + r < n ? (int64_t)ids[r0 + r] : -1;
      if (id[r] < 0 || id[r] >= V) id[r] = -1;
    }
    for (int c = lane; c < nv; c += 64) {
      float x[LOOKUP_ROWS][N];
#pragma unroll
      for (int r = 0; r < LOOKUP_ROWS; ++r) {
        if (id[r] >= 0) {
          load_f<T, N>(table + id[r] * ld + (int64_t)c * N, x[r]);
#pragma unroll
          for (int e = 0; e < N; ++e) x[r][e] *= scale;
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) x[r][e] = NAN;
        }
      }
#pragma unroll
      for (int r = 0; r < LOOKUP_ROWS; ++r)
        if (r0 + r < n) store_f<T, N, STREAM>(out + (r0 + r) * d + (int64_t)c * N, x[r]);
    }
    for (int c = nv * N + lane; c < d; c += 64)
      for (int r = 0; r < LOOKUP_ROWS; ++r)
        if (r0 + r < n)
          out[(r0 + r) * d + c] =
              from_f<T>(id[r] >= 0 ? to_f<T>(table[id[r] * ld + c]) * scale : NAN);
  }
}

// ---- stable radix sort of (token, position) ------------------------------------------------------
// Digits of at most 8 bits, least significant first.  Each pass: every block counts the digits of
// its run of tiles, then ranks and moves them: an item's place is the number of items with a
// smaller digit, plus those of its digit in earlier blocks, tiles, waves and lanes.  Keys that take
// no gradient (the padding index, ids outside the table) become V and sort behind every row.
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WAVES = SORT_THREADS / 64;
constexpr int SORT_ITEMS = 2;  // per thread
constexpr int SORT_TILE = SORT_THREADS * SORT_ITEMS;
constexpr int SORT_BLOCKS = 256;
constexpr int SORT_ONE = 16 * SORT_THREADS;  // positions that one launch sorts
constexpr int DIGITS = 256;

struct SortPlan {
  int64_t tiles_per_block;
  int blocks, passes, bits;  // digit bits
};

SortPlan sort_plan(int64_t n, int64_t V) {
  SortPlan p;
  const int64_t tiles = cdiv(n, SORT_TILE);
  p.tiles_per_block = cdiv(tiles, SORT_BLOCKS);
  p.blocks = (int)cdiv(tiles, p.tiles_per_block);
  int bits = 1;
  while (bits < 32 && (V >> bits)) ++bits;  // keys 0 .. V
  p.passes = (bits + 7) / 8;
  p.bits = (bits + p.passes - 1) / p.passes;
  return p;
}

// The token of position i as a key of the first pass.
template <class I>
__device__ __forceinline__ uint32_t first_key(const I* ids, int64_t i, int64_t V, int64_t pad) {
  const int64_t id = (int64_t)ids[i];
  return id < 0 || id >= V || id == pad ? (uint32_t)V : (uint32_t)id;
}

struct KeySrc {  // the items of a pass: the ids themselves, or an earlier pass's output
  const void* ids;
  int ids64;
  int64_t V, pad;
  const uint32_t *key, *pos;
};

__device__ __forceinline__ uint32_t key_at(const KeySrc& s, int64_t i) {
  if (s.key) return s.key[i];
  return s.ids64 ? first_key(static_cast<const int64_t*>(s.ids), i, s.V, s.pad)
                 : first_key(static_cast<const int32_t*>(s.ids), i, s.V, s.pad);
}

__global__ __launch_bounds__(SORT_THREADS) void sort_count_kernel(KeySrc src, int64_t n,
                                                                  int64_t tiles_per_block,
                                                                  int shift, int bits,
                                                                  uint32_t* hist) {
  __shared__ uint32_t cnt[DIGITS];
  const int t = threadIdx.x;
  if (t < DIGITS) cnt[t] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * tiles_per_block * SORT_TILE;
  const int64_t hi = min(n, lo + tiles_per_block * SORT_TILE);
  const uint32_t mask = (1u << bits) - 1;
  for (int64_t i = lo + t; i < hi; i += SORT_THREADS)
    atomicAdd(&cnt[(key_at(src, i) >> shift) & mask], 1u);
  __syncthreads();
  if (t < DIGITS) hist[(int64_t)blockIdx.x * DIGITS + t] = cnt[t];
}

// The exclusive sums of the first 256 threads' values (every thread of the block calls it).
__device__ __forceinline__ uint32_t scan_digits(uint32_t v, uint32_t* part) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  uint32_t s = v;
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t x = __shfl_up(s, off, 64);
    if (lane >= off) s += x;
  }
  if (wave < 4 && lane == 63) part[wave] = s;
  __syncthreads();
  for (int w = 0; w < 4; ++w)
    if (w < wave && wave < 4) s += part[w];
  return s - v;
}

// The rank of an item among those of its digit that this wave has met, this round's lower lanes
// included; cnt: the wave's counts.  Lanes run in lockstep: every lane reads the count before the
// first lane of its digit raises it (the fences keep the compiler from moving the accesses).
__device__ __forceinline__ uint32_t digit_rank(uint32_t* cnt, uint32_t dig, bool in, int bits,
                                               int lane) {
  uint64_t same = __ballot(in);  // the lanes that hold this digit
  for (int b = 0; b < bits; ++b) {
    const uint64_t m = __ballot((dig >> b) & 1);
    same &= (dig >> b) & 1 ? m : ~m;
  }
  const uint32_t old = in ? *(volatile uint32_t*)&cnt[dig] : 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const uint64_t below = same & ((1ull << lane) - 1);
  if (in && below == 0) *(volatile uint32_t*)&cnt[dig] = old + (uint32_t)__popcll(same);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  return old + (uint32_t)__popcll(below);
}

// Up to ITEMS * SORT_THREADS positions in one launch: block b sorts the tokens [b range, (b + 1)
// range) by itself.  It reads every id, counts those below its range (which says where its part of
// the result begins) and keeps its own in the order of their positions; one counting pass over
// `range` digits then ranks them.  Reading 16384 ids in 128 blocks costs less than the launches
// that sharing them would take: 8992 ids 13 us against 28 us for the two passes below.
constexpr int RANGE_MAX = 1024;
template <int ITEMS>
__global__ __launch_bounds__(SORT_THREADS) void sort_range_kernel(KeySrc src, int n, uint32_t range,
                                                                  int bits, uint32_t* key_out,
                                                                  uint32_t* pos_out) {
  __shared__ uint32_t item[ITEMS * SORT_THREADS];  // token - lo (16 bits), position (14 bits)
  __shared__ uint32_t wcnt[SORT_WAVES][RANGE_MAX];
  __shared__ uint32_t mine[SORT_WAVES], less[SORT_WAVES], part[SORT_WAVES];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const uint32_t lo = blockIdx.x * range, hi = min(lo + range, (uint32_t)src.V + 1);
  uint32_t key[ITEMS], n_mine = 0, n_less = 0;
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const int i = (wave * ITEMS + r) * 64 + lane;
    key[r] = i < n ? key_at(src, i) : ~0u;
  }
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    n_less += (uint32_t)__popcll(__ballot(key[r] < lo));
    n_mine += (uint32_t)__popcll(__ballot(key[r] >= lo && key[r] < hi));
  }
  if (lane == 0) {
    mine[wave] = n_mine;
    less[wave] = n_less;
  }
  for (uint32_t d = lane; d < range; d += 64) wcnt[wave][d] = 0;
  __syncthreads();
  uint32_t base = 0, total = 0, at = 0;
  for (int w = 0; w < SORT_WAVES; ++w) {
    base += less[w];
    if (w < wave) at += mine[w];
    total += mine[w];
  }
  if (total == 0) return;
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const bool in = key[r] >= lo && key[r] < hi;
    const uint64_t m = __ballot(in);
    if (in)
      item[at + (uint32_t)__popcll(m & ((1ull << lane) - 1))] =
          (key[r] - lo) << 16 | (uint32_t)((wave * ITEMS + r) * 64 + lane);
    at += (uint32_t)__popcll(m);
  }
  __syncthreads();
  const int rounds = (int)((total + SORT_THREADS - 1) / SORT_THREADS);
  uint32_t mark[ITEMS];  // an item's place among those of its token
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const uint32_t i = (uint32_t)((wave * rounds + r) * 64 + lane);
    const bool in = r < rounds && i < total;
    mark[r] = r < rounds ? digit_rank(wcnt[wave], in ? item[i] >> 16 : 0, in, bits, lane) : 0;
  }
  __syncthreads();
  uint32_t count = 0;  // of token lo + t
  if (t < (int)range)
    for (int w = 0; w < SORT_WAVES; ++w) count += wcnt[w][t];
  uint32_t sum = count;
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t x = __shfl_up(sum, off, 64);
    if (lane >= off) sum += x;
  }
  if (lane == 63) part[wave] = sum;
  __syncthreads();
  uint32_t first = base + sum - count;
  for (int w = 0; w < wave; ++w) first += part[w];
  if (t < (int)range)
    for (int w = 0; w < SORT_WAVES; ++w) {
      const uint32_t c = wcnt[w][t];
      wcnt[w][t] = first;
      first += c;
    }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const uint32_t i = (uint32_t)((wave * rounds + r) * 64 + lane);
    if (r < rounds && i < total) {
      const uint32_t x = item[i], to = wcnt[wave][x >> 16] + mark[r];
      key_out[to] = lo + (x >> 16);
      pos_out[to] = x & 0xFFFF;
    }
  }
}

__global__ __launch_bounds__(SORT_THREADS) void sort_move_kernel(KeySrc src, int64_t n,
                                                                 int64_t tiles_per_block,
                                                                 int shift, int bits,
                                                                 const uint32_t* hist,
                                                                 uint32_t* key_out,
                                                                 uint32_t* pos_out) {
  __shared__ uint32_t base[DIGITS];                // next place of each digit
  __shared__ uint32_t part[4];
  __shared__ uint32_t wcnt[SORT_WAVES][DIGITS];    // per wave: items of the digit, then their base
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const uint32_t mask = (1u << bits) - 1;
  // each digit's items in the blocks before this one, and in all (four threads a digit)
  uint32_t before = 0, total = 0;
#pragma unroll 8
  for (int b = t / DIGITS; b < (int)gridDim.x; b += SORT_THREADS / DIGITS) {
    const uint32_t h = hist[(int64_t)b * DIGITS + t % DIGITS];
    if (b < (int)blockIdx.x) before += h;
    total += h;
  }
  (&wcnt[0][0])[2 * t] = before;
  (&wcnt[0][0])[2 * t + 1] = total;
  __syncthreads();
  if (t < DIGITS)
    for (int q = 1; q < SORT_THREADS / DIGITS; ++q) {
      before += (&wcnt[0][0])[2 * (t + q * DIGITS)];
      total += (&wcnt[0][0])[2 * (t + q * DIGITS) + 1];
    }
  const uint32_t smaller = scan_digits(total, part);
  if (t < DIGITS) base[t] = smaller + before;
  const int64_t lo = (int64_t)blockIdx.x * tiles_per_block * SORT_TILE;
  const int64_t hi = min(n, lo + tiles_per_block * SORT_TILE);
  for (int64_t tile = lo; tile < hi; tile += SORT_TILE) {
    for (int i = t; i < SORT_WAVES * DIGITS; i += SORT_THREADS) (&wcnt[0][0])[i] = 0;
    __syncthreads();
    uint32_t key[SORT_ITEMS], pos[SORT_ITEMS], rank[SORT_ITEMS];
#pragma unroll
    for (int r = 0; r < SORT_ITEMS; ++r) {
      const int64_t i = tile + ((int64_t)wave * SORT_ITEMS + r) * 64 + lane;
      const bool in = i < hi;
      key[r] = in ? key_at(src, i) : 0;
      pos[r] = in ? (src.pos ? src.pos[i] : (uint32_t)i) : 0;
      rank[r] = digit_rank(wcnt[wave], (key[r] >> shift) & mask, in, bits, lane);
    }
    __syncthreads();
    if (t < DIGITS) {
      uint32_t at = base[t];
      for (int w = 0; w < SORT_WAVES; ++w) {
        const uint32_t c = wcnt[w][t];
        wcnt[w][t] = at;
        at += c;
      }
      base[t] = at;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < SORT_ITEMS; ++r) {
      const int64_t i = tile + ((int64_t)wave * SORT_ITEMS + r) * 64 + lane;
      if (i < hi) {
        const uint32_t at = wcnt[wave][(key[r] >> shift) & mask] + rank[r];
        key_out[at] = key[r];
        pos_out[at] = pos[r];
      }
    }
    __syncthreads();
  }
}

// ---- sums ----------------------------------------------------------------------------------------
constexpr int ZERO_ROWS = 16;  // table rows a wave looks up among the sorted tokens
constexpr int SUM_AHEAD = 8;   // rows a wave has in flight

struct SumArgs {
  const uint32_t *key, *pos;
  int64_t n, V, ld;
  int d, win, slabs;
  float scale;
  int64_t wins, zero_blocks;
  float *head, *tail;  // [wins][d]: the window's share of a run that began before it / goes on
};

template <class T, int N>
__device__ __forceinline__ void sum_flush(const SumArgs& a, T* dw, int64_t w, uint32_t key,
                                          bool from_before, bool goes_on, int64_t col, bool act,
                                          float (&acc)[N]) {
  if (!act || key >= (uint32_t)a.V) return;
  if (from_before || goes_on) {
    store_f<float, N>((from_before ? a.head : a.tail) + w * a.d + col, acc);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] *= a.scale;
    store_f<T, N>(dw + (int64_t)key * a.d + col, acc);
  }
}

// Blocks [0, zero_blocks): the rows of dW without a token become zero (a wave looks its rows up in
// the sorted keys, ZERO_ROWS at a time).  The others: a wave per window of `win` sorted positions and
// slab of 64 accesses of N columns, the rows' loads SUM_AHEAD ahead of their additions.  Bound by the
// reads of dout: 262144 rows of 1024 in bf16, 30 % of them padding that is skipped (376 MB in, 66 MB
// out), 102 us, 4.3 TB/s; 8992 rows of 768 in fp32 (28 MB in, 99 MB out) 19 us, 6.6 TB/s.
template <class T, int N>
__global__ __launch_bounds__(256) void embed_sum_kernel(const T* __restrict__ dout, SumArgs a,
                                                        T* __restrict__ dw) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  if (blockIdx.x < a.zero_blocks) {
    for (int64_t r0 = ((int64_t)blockIdx.x * 4 + wave) * ZERO_ROWS; r0 < a.V;
         r0 += a.zero_blocks * 4 * ZERO_ROWS) {
      const int64_t row = r0 + lane;
      bool empty = false;
      if (lane < ZERO_ROWS && row < a.V) {
        int64_t lo = 0, hi = a.n;  // the first sorted position with key >= row
        while (lo < hi) {
          const int64_t mid = (lo + hi) >> 1;
          if (a.key[mid] < (uint32_t)row) lo = mid + 1; else hi = mid;
        }
        empty = lo == a.n || a.key[lo] != (uint32_t)row;
      }
      const uint64_t todo = __ballot(empty);
      for (int r = 0; r < ZERO_ROWS; ++r) {
        if (!((todo >> r) & 1)) continue;
        T* o = dw + (r0 + r) * a.d;
        float z[N] = {};
        for (int c = lane * N; c + N <= a.d; c += 64 * N) store_f<T, N>(o + c, z);
      }
    }
    return;
  }
  const int64_t unit = (blockIdx.x - a.zero_blocks) * 4 + wave;
  const int64_t w = unit / a.slabs;
  if (w >= a.wins) return;
  const int64_t col = ((int64_t)(unit % a.slabs) * 64 + lane) * N;
  const int64_t lo = w * a.win, hi = min(a.n, lo + a.win);
  const uint32_t first = a.key[lo], last = a.key[hi - 1];
  if (first >= (uint32_t)a.V) return;  // behind the last row
  const bool before = lo > 0 && a.key[lo - 1] == first;
  const bool after = hi < a.n && a.key[hi] == last;
  const bool act = col + N <= a.d;
  float acc[N] = {};
  uint32_t cur = first;
  bool run_before = before;
  for (int64_t base = lo; base < hi; base += 64) {
    const int m = (int)min((int64_t)64, hi - base);
    const uint32_t mykey = lane < m ? a.key[base + lane] : 0;
    const uint32_t mypos = lane < m ? a.pos[base + lane] : 0;
    for (int j0 = 0; j0 < m; j0 += SUM_AHEAD) {
      typename Vec<T, N>::type x[SUM_AHEAD];
#pragma unroll
      for (int j = 0; j < SUM_AHEAD; ++j) {
        const int at = min(j0 + j, m - 1);
        const int64_t p = (uint32_t)__builtin_amdgcn_readlane((int)mypos, at);
        if (act) x[j] = *reinterpret_cast<const typename Vec<T, N>::type*>(dout + p * a.ld + col);
      }
#pragma unroll
      for (int j = 0; j < SUM_AHEAD; ++j) {
        if (j0 + j >= m) break;
        const uint32_t k = (uint32_t)__builtin_amdgcn_readlane((int)mykey, j0 + j);
        if (k != cur) {
          sum_flush<T, N>(a, dw, w, cur, run_before, false, col, act, acc);
#pragma unroll
          for (int e = 0; e < N; ++e) acc[e] = 0.f;
          cur = k;
          run_before = false;
        }
        if (act) {
#pragma unroll
          for (int e = 0; e < N; ++e) acc[e] += vec_f<T, N>(x[j], e);
        }
      }
    }
  }
  sum_flush<T, N>(a, dw, w, cur, run_before, after, col, act, acc);
}

// A run that crosses windows: the tail of the window where it begins, then the heads of the
// following ones.  A block per window and 256 columns (4 a lane); the waves take the windows in turn.
// Bound by the latency of the longest run: 8992 rows, a fifth of them one token, 6.5 us.
constexpr int JOIN_AHEAD = 8;
template <class T, int N>
__global__ __launch_bounds__(256) void embed_join_kernel(SumArgs a, T* __restrict__ dw) {
  __shared__ float red[4][64][N];
  const int64_t w = blockIdx.x;
  const int64_t hi = (w + 1) * a.win;
  if (hi >= a.n) return;
  const uint32_t key = a.key[hi - 1];
  if (key >= (uint32_t)a.V || a.key[hi] != key) return;
  const int64_t lo = w * a.win;
  if (a.key[lo] == key && lo > 0 && a.key[lo - 1] == key) return;  // began before
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the windows w + 1 .. w + m begin with the key
  int64_t m = 1;
  for (;;) {
    const int64_t at = (w + 1 + m + lane) * a.win;
    const uint64_t same = __ballot(at < a.n && a.key[at < a.n ? at : 0] == key);
    if (same == ~0ull) {
      m += 64;
      continue;
    }
    m += __ffsll((unsigned long long)~same) - 1;
    break;
  }
  const int col = (blockIdx.y * 64 + lane) * N;
  float s[N] = {};
  if (col < a.d) {
    const float* h = a.head + (w + 1) * a.d + col;
    int64_t i = wave;
    for (; i + 4 * (JOIN_AHEAD - 1) < m; i += 4 * JOIN_AHEAD) {
      float x[JOIN_AHEAD][N];
#pragma unroll
      for (int j = 0; j < JOIN_AHEAD; ++j) load_f<float, N>(h + (i + 4 * j) * a.d, x[j]);
#pragma unroll
      for (int j = 0; j < JOIN_AHEAD; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) s[e] += x[j][e];
    }
    for (; i < m; i += 4) {
      float x[N];
      load_f<float, N>(h + i * a.d, x);
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] += x[e];
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) red[wave][lane][e] = s[e];
  __syncthreads();
  if (wave == 0 && col < a.d) {
    load_f<float, N>(a.tail + w * a.d + col, s);
#pragma unroll
    for (int e = 0; e < N; ++e)
      s[e] = (s[e] + ((red[0][lane][e] + red[1][lane][e]) + (red[2][lane][e] + red[3][lane][e]))) *
             a.scale;
    store_f<T, N>(dw + (int64_t)key * a.d + col, s);
  }
}

// ---- host ----------------------------------------------------------------------------------------
struct EmbedGrad {
  SortPlan sort;
  int64_t key[2], pos[2], hist, head, tail, bytes;  // offsets into the workspace
  int64_t wins;
  int win, slabs;
};

int64_t align256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// Window: the largest of 256 .. 8 positions that still gives SUM_WAVES waves (a longer window leaves
// fewer partial sums of the runs that cross windows; fewer waves leave memory idle).
constexpr int64_t SUM_WAVES = 4096;
constexpr int64_t ZERO_BLOCKS = (int64_t)1 << 20;  // tables of more than 2^26 rows: several turns each
constexpr int64_t SUM_GRID = ((int64_t)1 << 24) - 1;  // less than 2^32 threads in blocks of 256

EmbedGrad embed_plan(int64_t n, int64_t V, int d, int vec) {
  EmbedGrad p;
  p.sort = sort_plan(n, V);
  p.slabs = (int)cdiv(d, 64 * (int64_t)vec);
  p.win = 8;
  for (int w : {256, 128, 64, 32, 16})
    if (n / w * p.slabs >= SUM_WAVES) {
      p.win = w;
      break;
    }
  p.wins = cdiv(n, p.win);
  int64_t at = 0;
  for (int i = 0; i < 2; ++i) {
    p.key[i] = at; at += align256(4 * n);
    p.pos[i] = at; at += align256(4 * n);
  }
  p.hist = at; at += align256(4 * (int64_t)DIGITS * p.sort.blocks);
  p.head = at; at += align256(4 * p.wins * d);
  p.tail = at; at += align256(4 * p.wins * d);
  p.bytes = at;
  return p;
}

int embed_vec(int32_t dtype, int d) {
  const int v = dtype == MPR_F32 ? 4 : 8;
  return d % v ? 1 : v;
}

int64_t sum_blocks(const SumArgs& a) { return a.zero_blocks + cdiv(a.wins * a.slabs, 4); }

template <class T, int N>
int embed_sums(const void* dout, const SumArgs& a, void* dw, hipStream_t s) {
  const int64_t blocks = sum_blocks(a);
  embed_sum_kernel<T, N><<<dim3((unsigned)blocks), 256, 0, s>>>(static_cast<const T*>(dout), a,
                                                                 static_cast<T*>(dw));
  MPR_LAUNCHED();
  constexpr int J = N == 1 ? 1 : 4;  // (N > 1: d is a multiple of it)
  embed_join_kernel<T, J><<<dim3((unsigned)a.wins, (unsigned)cdiv(a.d, 64 * J)), 256, 0, s>>>(
      a, static_cast<T*>(dw));
  MPR_LAUNCHED();
  return MPR_OK;
}

int embed_check(const char* what, int32_t dtype, int64_t n, int64_t V, int32_t d) {
  MPR_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype code %d", what, (int)dtype);
  MPR_REQUIRE(n >= 0 && n < (int64_t)1 << 31, "%s: %lld ids", what, (long long)n);
  MPR_REQUIRE(V >= 1 && V < (int64_t)1 << 31, "%s: a table of %lld rows", what, (long long)V);
  MPR_REQUIRE(d >= 1 && d <= 1 << 21, "%s: rows of %d", what, (int)d);
  return MPR_OK;
}

}  // namespace
}  // namespace mpr

using namespace mpr;

extern "C" {

int mpr_embed_lookup(const void* table, int32_t dtype, int64_t V, int64_t ld, const void* ids,
                     int32_t ids64, int64_t n, int32_t d, float scale, void* out, void* stream) {
  return ops_call("embed_lookup", [&]() -> int {
    MPR_TRY(embed_check("embed_lookup", dtype, n, V, d));
    MPR_REQUIRE(ld >= d || V == 1, "embed_lookup: row stride %lld < %d", (long long)ld, (int)d);
    if (n == 0) return MPR_OK;
    MPR_REQUIRE(table && ids && out, "embed_lookup: null pointer");
    return by_dtype(dtype, [&](auto z) -> int {
      using T = decltype(z);
      const dim3 grid((unsigned)std::min<int64_t>(cdiv(n, 4 * LOOKUP_ROWS), MAX_GRID_X));
      const bool stream_out = n * d * (int64_t)sizeof(T) >= STREAM_BYTES;
      const auto launch = [&](auto id, auto st) {
        typedef decltype(id) I;
        embed_lookup_kernel<T, I, decltype(st)::value><<<grid, 256, 0, op_stream(stream)>>>(
            static_cast<const T*>(table), V, ld, static_cast<const I*>(ids), n, d, scale,
            static_cast<T*>(out));
      };
      if (ids64 && stream_out) launch(int64_t{}, std::true_type{});
      else if (ids64) launch(int64_t{}, std::false_type{});
      else if (stream_out) launch(int32_t{}, std::true_type{});
      else launch(int32_t{}, std::false_type{});
      MPR_LAUNCHED();
      return MPR_OK;
    });
  });
}

int mpr_embed_grad_workspace(int32_t dtype, int64_t n, int64_t V, int32_t d, int64_t* bytes) {
  return ops_call("embed_grad_workspace", [&]() -> int {
    MPR_TRY(embed_check("embed_grad_workspace", dtype, n, V, d));
    MPR_REQUIRE(bytes, "embed_grad_workspace: null pointer");
    *bytes = n ? embed_plan(n, V, d, embed_vec(dtype, d)).bytes : 0;
    return MPR_OK;
  });
}

int mpr_embed_grad(const void* dout, int32_t dtype, int64_t ld, const void* ids, int32_t ids64,
                   int64_t n, int64_t V, int32_t d, float scale, int64_t padding_idx, void* dtable,
                   void* ws, int64_t ws_bytes, void* stream) {
  return ops_call("embed_grad", [&]() -> int {
    MPR_TRY(embed_check("embed_grad", dtype, n, V, d));
    MPR_REQUIRE(ld >= d || n <= 1, "embed_grad: row stride %lld < %d", (long long)ld, (int)d);
    MPR_REQUIRE(dtable && (n == 0 || (dout && ids)), "embed_grad: null pointer");
    const int vec = embed_vec(dtype, d);
    hipStream_t s = op_stream(stream);
    EmbedGrad p{};
    SumArgs a{};
    a.n = n; a.V = V; a.ld = ld; a.d = d; a.scale = scale;
    a.win = 1; a.slabs = 1;
    a.zero_blocks = std::min(cdiv(V, 4 * ZERO_ROWS), ZERO_BLOCKS);
    if (n) {
      p = embed_plan(n, V, d, vec);
      MPR_REQUIRE(ws && ws_bytes >= p.bytes, "embed_grad: workspace of %lld bytes, %lld needed",
                  (long long)ws_bytes, (long long)p.bytes);
      a.win = p.win; a.wins = p.wins; a.slabs = p.slabs;
      MPR_REQUIRE(sum_blocks(a) <= SUM_GRID && a.wins <= SUM_GRID, "embed_grad: too many positions");
      char* w = static_cast<char*>(ws);
      uint32_t* key[2] = {reinterpret_cast<uint32_t*>(w + p.key[0]),
                          reinterpret_cast<uint32_t*>(w + p.key[1])};
      uint32_t* pos[2] = {reinterpret_cast<uint32_t*>(w + p.pos[0]),
                          reinterpret_cast<uint32_t*>(w + p.pos[1])};
      uint32_t* hist = reinterpret_cast<uint32_t*>(w + p.hist);
      KeySrc src{ids, ids64, V, padding_idx, nullptr, nullptr};
      const int64_t range = std::max<int64_t>(64, cdiv(V + 1, 128));
      const bool one = n <= SORT_ONE && range <= RANGE_MAX;
      if (one) {
        int bits = 1;
        while ((int64_t)1 << bits < range) ++bits;
        const auto sort = n <= 4 * SORT_THREADS ? sort_range_kernel<4> : sort_range_kernel<16>;
        sort<<<dim3((unsigned)cdiv(V + 1, range)), SORT_THREADS, 0, s>>>(
            src, (int)n, (uint32_t)range, bits, key[0], pos[0]);
        MPR_LAUNCHED();
        src.key = key[0];
        src.pos = pos[0];
      }
      for (int i = 0; !one && i < p.sort.passes; ++i) {
        const int shift = i * p.sort.bits;
        sort_count_kernel<<<p.sort.blocks, SORT_THREADS, 0, s>>>(src, n, p.sort.tiles_per_block,
                                                                 shift, p.sort.bits, hist);
        MPR_LAUNCHED();
        sort_move_kernel<<<p.sort.blocks, SORT_THREADS, 0, s>>>(src, n, p.sort.tiles_per_block,
                                                                shift, p.sort.bits, hist,
                                                                key[i & 1], pos[i & 1]);
        MPR_LAUNCHED();
        src.key = key[i & 1];
        src.pos = pos[i & 1];
      }
      a.key = src.key; a.pos = src.pos;
      a.head = reinterpret_cast<float*>(w + p.head);
      a.tail = reinterpret_cast<float*>(w + p.tail);
    }
    return by_dtype(dtype, [&](auto z) -> int {
      using T = decltype(z);
      if (n == 0) {  // every row is empty
        embed_sum_kernel<T, 1><<<dim3((unsigned)a.zero_blocks), 256, 0, s>>>(
            static_cast<const T*>(dout), a, static_cast<T*>(dtable));
        MPR_LAUNCHED();
        return MPR_OK;
      }
      return vec == 1 ? embed_sums<T, 1>(dout, a, dtable, s)
                      : embed_sums<T, VEC16<T>>(dout, a, dtable, s);
    });
  });
}

}  // extern "C"
