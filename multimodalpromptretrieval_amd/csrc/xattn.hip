// xattn.hip — attention of queries to another sequence's states (an encoder's), forward and
// backward, for key / value heads that groups of query heads share.  Per (batch, key head), the
// queries of its group are the rows r = g Lq + i (g < G = H / Hkv, i < Lq):
//   S = scale q k^T,  P = softmax over the keys that the mask keeps,  O = P v;  no key kept: O = 0
//   dV = P^T dO,  dS = P (dO v^T - rowsum(dO O)),  dQ = scale dS k,  dK = scale dS^T q
// The softmax runs in one pass over the keys with a running maximum and sum (fp32, base 2), and
// the backward computes P again from the saved row statistic lse2 = max + log2(sum), so nothing of
// size Lq x Lk is kept.  A row of all shared heads of a group lies in one tile, so K and V are read
// once for the group and dK, dV sum the heads in registers: no atomics, the same bits every run.
//
// Matrix products: bf16 inputs on v_mfma_f32_32x32x16_bf16, float inputs on v_mfma_f32_32x32x2_f32
// (exact fp32 products).  Half is for single tokens only: it has no matrix-core variant here, and the
// caller computes it in float.  The products are arranged so that a tile's scores come out of the matrix
// core in the lane order in which the next product takes them (scores transposed: lane = row, registers
// = keys): probabilities go from one product to the next in registers, never through LDS.  P and dS
// are rounded to bf16 as operands of the second products, as the inputs are; sums stay fp32.  Two
// things keep the backward's differences dP - rowsum(dO O) exact where a row has few keys and they
// cancel: the forward divides by the sum of the rounded P (its weights then add up to 1), and it
// keeps what rounding takes off O for that row sum.
//
// Masked keys count for nothing whatever they hold (NaN, infinities): they are staged as zeros.  A row
// of kept keys that all score -inf has no softmax: its sum is 0 as that of a row without a key is, and
// what tells them apart is whether a key was there (NONE_FINITE); O and the saved statistic are NaN.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ops.h"

namespace mpr {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr int NW = 4;  // waves of a block (of the tiled kernels)

struct XArgs {
  const void *q, *k, *v, *dout, *o;
  const uint8_t* keep;
  int64_t q_bs, q_ls, q_hs, k_bs, k_ls, k_hs, v_bs, v_ls, v_hs, keep_bs, do_bs, do_ls, do_hs;
  int B, H, Hkv, G, Lq, Lk, D;
  int R;             // rows of a key head: G Lq
  uint64_t lq_mul;   // r / Lq = r lq_mul >> lq_shift for r < 2^30
  int lq_shift;
  int tiles, splits, per_split;  // blocks along the tiled axis, and shares of the other one
  int longest_first;  // the batch entries in the order of their lengths
  float c;           // scale log2(e), above 0
  float slack;       // how far scores may pass the running maximum: 8 / c
  float scale;
  void* out;         // forward: [B, Lq, H, D]
  void* rest;        // bf16 only, may be null: what rounding took off out
  const void* o_rest;
  float* lse;        // [B, H, Lq]: max + log2(sum) of the scaled scores in base 2
  float* delta;      // [B, H, Lq]
  float *part, *part2;  // splits' shares
  float* part_ms;    // [split][B Hkv R][2]: running maximum and sum
  void *dq, *dk, *dv;
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// In the place of a share's sum: it has keys, and every score is -inf.  (The share's maximum is -inf,
// so beside others it weighs 0 like any other value.)
constexpr float NONE_FINITE = -1.f;
// what a row's sum l of 0 makes of its output and of its statistic
__device__ __forceinline__ float inv_sum(float l, bool some) {
  return l == 0.f ? (some ? NAN : 0.f) : 1.f / l;
}
__device__ __forceinline__ float lse_of(float m, float l, bool some) {
  return l == 0.f ? (some ? NAN : -INFINITY) : m + log2f(l);
}

// ---- the two matrix cores ------------------------------------------------------------------------
// LDS tiles hold rows of DP elements in 16-byte pieces; piece c of row r lies at piece c ^ swz(r):
// eight rows of one piece, and four rows of two neighbouring pieces, then cover all the banks, which
// is what a row read and a column read ask for at a time.
__device__ __forceinline__ int swz(int r) { return ((r & 3) << 1) | ((r >> 2) & 1); }

// A chunk is the contraction of one call (two pieces); frag: a lane's share of it.  Lane l holds
// index l & 31 of the operand's own axis; its half h = l >> 5 of the contraction.
//   row(p, r0, c): operand rows r0 .. r0 + 31 lie as rows of LDS, chunk c of their columns
//   col(p, k0, m0): the contraction runs over rows k0 .. of LDS, in the order in which a product's
//                   result holds its rows (result register r of half h is row 8 (r / 4) + 4 h +
//                   r % 4); the operand's own axis is the columns m0 .. m0 + 31
struct MmaBf16 {
  typedef bf16 elem;
  typedef bf16x8 frag;
  static constexpr int CHUNK = 16;
  // ds_read_tr16_b64: 16 lanes read 4 rows of 16 elements and each gets a column of them
  template <int DP>
  static __device__ __forceinline__ frag col(const elem* p, int k0, int m0, int lane) {
    const int i = lane & 15, g = lane >> 4;
    const int r = 4 * (g >> 1) + (i >> 2);  // (k0 is a multiple of 8: it does not enter swz)
    const int sw = (2 * (g & 1) + ((i & 3) >> 1)) ^ swz(r), m8 = m0 >> 3;
    const elem* a = p + r * DP + ((sw ^ (m8 & 7)) << 3) + 4 * (i & 1) + k0 * DP + ((m8 & ~7) << 3);
    typedef __attribute__((address_space(3))) s16x4* lds4;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)a);
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(a + 8 * DP));
    const s16x8 z = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(frag, z);
  }
  static __device__ __forceinline__ frag pack(const f32x16& x, int c) {
    frag f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (bf16)x[8 * c + j];
    return f;
  }
  static __device__ __forceinline__ float sum(frag f, float s) {  // s + its elements
    typedef bf16 pair __attribute__((ext_vector_type(2)));
    const pair one = {(bf16)1.f, (bf16)1.f};
#pragma unroll
    for (int j = 0; j < 8; j += 2)
      s = __builtin_amdgcn_fdot2_f32_bf16(pair{f[j], f[j + 1]}, one, s, false);
    return s;
  }
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

struct MmaF32 {
  typedef float elem;
  typedef f32x4 frag;
  static constexpr int CHUNK = 8;
  template <int DP>
  static __device__ __forceinline__ frag col(const elem* p, int k0, int m0, int lane) {
    const int h = lane >> 5, x = ((lane & 31) >> 2) ^ h;  // m0 is a multiple of 32: 8 pieces
    const elem* a = p + 4 * h * DP + (lane & 3);
    frag f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = a[((x ^ (2 * j)) << 2) + (k0 + j) * DP + m0];
    return f;
  }
  static __device__ __forceinline__ frag pack(const f32x16& x, int c) {
    return frag{x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]};
  }
  static __device__ __forceinline__ float sum(frag f, float s) {
    return s + ((f[0] + f[1]) + (f[2] + f[3]));
  }
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

template <class M>
constexpr int PIECE = 16 / (int)sizeof(typename M::elem);  // elements

template <class M, int DP>
__device__ __forceinline__ typename M::frag row_frag(const typename M::elem* p, int r0, int c,
                                                     int lane) {
  const int r = lane & 31, x = (lane >> 5) ^ swz(r);
  return *reinterpret_cast<const typename M::frag*>(
      p + r * DP + (x ^ (2 * c & 7)) * PIECE<M> + r0 * DP + (2 * c & ~7) * PIECE<M>);
}

// The compiler keeps the order across this point.  Below, operands are read from LDS AHEAD calls before
// the matrix core takes them, in the order written: left to itself it reads each where it is used,
// and every call waits out LDS's latency.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }
constexpr int AHEAD = 4;

// acc += the chunks' products of the LDS rows r0 .. r0 + 31 with f (one or two such sums side by
// side: neighbouring calls do not wait for each other's result)
template <class M, int DP>
__device__ __forceinline__ void rows_mma(const typename M::elem* p, int r0,
                                         const typename M::frag (&f)[DP / M::CHUNK], f32x16& acc,
                                         int lane) {
  constexpr int NC = DP / M::CHUNK, A = AHEAD < NC ? AHEAD : NC;
  typename M::frag x[A];
#pragma unroll
  for (int c = 0; c < A; ++c) x[c] = row_frag<M, DP>(p, r0, c, lane);
  in_order();
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    acc = M::mma(x[c % A], f[c], acc);
    if (c + A < NC) x[c % A] = row_frag<M, DP>(p, r0, c + A, lane);
    in_order();
  }
}
template <class M, int DP, class F1, class F2>
__device__ __forceinline__ void rows_mma2(const typename M::elem* p1, const typename M::elem* p2,
                                          int r0, F1 f1, F2 f2, f32x16& acc1, f32x16& acc2,
                                          int lane) {
  constexpr int NC = DP / M::CHUNK, A = DP == 128 ? AHEAD / 2 : AHEAD;
  typename M::frag x[A], y[A], g[A];
#pragma unroll
  for (int c = 0; c < A; ++c) {
    x[c] = row_frag<M, DP>(p1, r0, c, lane);
    y[c] = row_frag<M, DP>(p2, r0, c, lane);
    g[c] = f2(c);
  }
  in_order();
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    acc1 = M::mma(x[c % A], f1(c), acc1);
    acc2 = M::mma(y[c % A], g[c % A], acc2);
    if (c + A < NC) {
      x[c % A] = row_frag<M, DP>(p1, r0, c + A, lane);
      y[c % A] = row_frag<M, DP>(p2, r0, c + A, lane);
      g[c % A] = f2(c + A);
    }
    in_order();
  }
}
// acc[d] += (columns 32 d .. of LDS rows k0 .. k0 + 31, transposed) x s, s a result of 32 x 32; the
// sum of this lane's s, as the product takes them (rounded).  FINE: s in two parts, its rounding and
// what that takes off it, each multiplied: s to 16 bits instead of 8.
template <class M, int DP, bool FINE = false>
__device__ __forceinline__ float cols_mma(const typename M::elem* p, int k0, const f32x16& s,
                                          f32x16 (&acc)[DP / 32], int lane) {
  constexpr int ND = DP / 32, PC = 32 / M::CHUNK, NI = ND * PC, A = AHEAD < NI ? AHEAD : NI;
  typename M::frag x[A], f[PC], g[FINE ? PC : 1];
  const auto get = [&](int i) {
    return M::template col<DP>(p, k0 + i / ND * M::CHUNK, i % ND * 32, lane);
  };
#pragma unroll
  for (int i = 0; i < A; ++i) x[i] = get(i);
  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < PC; ++c) {
    f[c] = M::pack(s, c);
    sum = M::sum(f[c], sum);
    if constexpr (FINE) {
      constexpr int N = M::CHUNK / 2;
#pragma unroll
      for (int j = 0; j < N; ++j) g[c][j] = (typename M::elem)(s[N * c + j] - (float)f[c][j]);
      sum = M::sum(g[c], sum);
    }
  }
  in_order();
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    acc[i % ND] = M::mma(x[i % A], f[i / ND], acc[i % ND]);
    if constexpr (FINE) acc[i % ND] = M::mma(x[i % A], g[i / ND], acc[i % ND]);
    if (i + A < NI) x[i % A] = get(i + A);
    in_order();
  }
  return sum;
}

// the row (0 .. 31) that result register r of this lane's half holds
__device__ __forceinline__ int acc_row(int r, int lane) {
  return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
}

// a value's pair in the other half of the wave: f(own, other's) in both
template <class F>
__device__ __forceinline__ float halves(float x, F f) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return f(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

template <int CTRL>
__device__ __forceinline__ float permuted(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// the sum over neighbouring groups of LPR lanes, in all of them (no LDS: lane permutations)
template <int LPR>
__device__ __forceinline__ float group_add(float x) {
  x += permuted<0xB1>(x);   // lane ^ 1
  x += permuted<0x4E>(x);   // lane ^ 2
  x += permuted<0x141>(x);  // mirrored in 8: the other four
  if constexpr (LPR >= 16) x += permuted<0x140>(x);  // mirrored in 16: the other eight
  if constexpr (LPR == 32) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
  }
  return x;
}

// ---- staging -------------------------------------------------------------------------------------
// A tile of ROWS rows from memory straight to LDS (no registers in between): starts the reads; they
// have landed after landed() and a barrier.  A wave's call writes 64 neighbouring pieces, so the
// permutation of a row's pieces is in what each lane reads.  Rows past `last` read that row: what they
// hold meets only zeros (patch()) or masked scores.  Pieces past column D read `zeros` (another piece
// of the row would not do: an infinity there times the other operand's zero is NaN).  at(r): the
// row's first element.
__device__ const f32x4 zeros = {0.f, 0.f, 0.f, 0.f};
template <class E, int DP, int ROWS, class At>
__device__ __forceinline__ void stage(E* lds, int64_t r0, int64_t last, int D, At at, int wave,
                                      int lane) {
  constexpr int N = 16 / (int)sizeof(E), CH = DP / N, CNT = ROWS * CH / (64 * NW);
  static_assert(ROWS * CH % (64 * NW) == 0, "whole calls a wave");
#pragma unroll
  for (int i = 0; i < CNT; ++i) {
    const int first = (i * NW + wave) * 64, slot = first + lane, r = slot / CH;
    const int c = ((slot % CH) ^ swz(r)) * N;
    const E* from = at(min(r0 + r, last)) + c;
    from = c < D ? from : reinterpret_cast<const E*>(&zeros);
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void*)from,
        (__attribute__((address_space(3))) void*)(lds + first * N), 16, 0, 0);
  }
}
// this wave's reads into LDS are done (before the barrier that shows them to the others)
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// zeros in the rows of a staged tile whose bit is 0
template <class E, int DP, int ROWS>
__device__ __forceinline__ void patch(E* lds, const uint32_t* words, int t) {
  constexpr int N = 16 / (int)sizeof(E), CH = DP / N;
  for (int p = t; p < ROWS * CH; p += 64 * NW) {
    const int r = p / CH;
    if (!((words[r >> 5] >> (r & 31)) & 1))
      *reinterpret_cast<f32x4*>(lds + p * N) = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// a wave's 32 rows as second operands in registers: frag c = contraction chunk c of row lane & 31
template <class T, class M, int DP>
__device__ __forceinline__ void load_rows(typename M::frag (&f)[DP / M::CHUNK], const T* row,
                                          bool in, int D, int lane) {
  constexpr int N = M::CHUNK / 2;
#pragma unroll
  for (int c = 0; c < DP / M::CHUNK; ++c) {
    const int d = c * M::CHUNK + N * (lane >> 5);
#pragma unroll
    for (int e = 0; e < N; ++e) f[c][e] = (typename M::elem)0.f;
    if (in && d < D) {
      const typename Vec<T, N>::type v =
          *reinterpret_cast<const typename Vec<T, N>::type*>(row + d);
#pragma unroll
      for (int e = 0; e < N; ++e) f[c][e] = (typename M::elem)v[e];
    }
  }
}

// The keys of a block in spans of SPAN: words[i] has a bit for each of the 32 keys from k0 + 32 i
// that exists (k < end) and that the mask keeps.  Whole tiles without one are passed over.
constexpr int SPAN = 4096, SPAN_UNIT = 128;  // SPAN_UNIT: a multiple of every tile
__device__ __forceinline__ void span_words(uint32_t* words, const uint8_t* keep, int64_t k0,
                                           int64_t end, int t, int threads) {
  const int n = (int)min((int64_t)SPAN, (end - k0 + SPAN_UNIT - 1) / SPAN_UNIT * SPAN_UNIT);
  for (int i = t; i < n; i += threads) {  // n and threads are multiples of 64: whole waves
    const int64_t k = k0 + i;
    const uint64_t on = __ballot(k < end && (!keep || keep[k]));
    if ((t & 63) == 0) {
      words[i >> 5] = (uint32_t)on;
      words[(i >> 5) + 1] = (uint32_t)(on >> 32);
    }
  }
}
// the keys that a span of n (words in LDS) has, the same in every lane
__device__ __forceinline__ int span_keys(const uint32_t* words, int n, int lane) {
  static_assert(SPAN / 32 == 128, "two words a lane");
  const int all = (n + SPAN_UNIT - 1) / SPAN_UNIT * (SPAN_UNIT / 32);
  const int own = (lane < all ? __popc(words[lane]) : 0) +
                  (lane + 64 < all ? __popc(words[lane + 64]) : 0);
  const float sum = halves(group_add<32>((float)own), [](float x, float y) { return x + y; });
  return __builtin_amdgcn_readfirstlane((int)sum);
}
template <int KT>
__device__ __forceinline__ int next_tile(const uint32_t* words, int at, int last) {
  for (; at < last; at += KT) {
    uint32_t any = 0;
#pragma unroll
    for (int u = 0; u < KT / 32; ++u) any |= words[at / 32 + u];
    if (any) break;
  }
  return at;
}

// [DP x 32 result, transposed] -> rows of 4-element runs: f(d, 4 values)
template <int DP, class F>
__device__ __forceinline__ void for_runs(const f32x16 (&acc)[DP / 32], int lane, F f) {
#pragma unroll
  for (int t = 0; t < DP / 32; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float x[4] = {acc[t][4 * r], acc[t][4 * r + 1], acc[t][4 * r + 2], acc[t][4 * r + 3]};
      f(32 * t + 8 * r + 4 * (lane >> 5), x);
    }
}

// A wave's accumulator to LDS and back (another wave's, lane for lane)
template <int NT>
__device__ __forceinline__ void acc_out(float* lds, const f32x16 (&acc)[NT], int lane) {
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<f32x4*>(lds + ((t * 4 + r) * 64 + lane) * 4) =
          f32x4{acc[t][4 * r], acc[t][4 * r + 1], acc[t][4 * r + 2], acc[t][4 * r + 3]};
}
template <int NT>
__device__ __forceinline__ void acc_join(const float* lds, f32x16 (&acc)[NT], float own,
                                         float other, int lane) {
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(lds + ((t * 4 + r) * 64 + lane) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][4 * r + e] = acc[t][4 * r + e] * own + x[e] * other;
    }
}

// N values of the output, and what rounding takes off them
template <class T, int N>
__device__ __forceinline__ void store_out(const XArgs& a, int64_t at, const float (&x)[N]) {
  store_f<T, N>(static_cast<T*>(a.out) + at, x);
  if (a.rest) {
    float y[N];
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = x[e] - to_f<T>(from_f<T>(x[e]));
    store_f<T, N>(static_cast<T*>(a.rest) + at, y);
  }
}

struct RowAt {  // row r of (b, key head): its query head and position
  int h, i;
};
__device__ __forceinline__ RowAt row_at(const XArgs& a, int hk, int r) {
  const int g = (int)((uint64_t)(uint32_t)r * a.lq_mul >> a.lq_shift);
  return {hk * a.G + g, r - g * a.Lq};
}

// Which (tile, split, batch, key head) a block computes.  Blocks go round robin over the 8 XCDs; the
// tiles of one split of a key head read the same keys, so they are given to one XCD and its L2, and
// neighbouring key heads to different XCDs: the heads of a batch entry have its length in common, and
// with whole entries on an XCD the longest one's would keep the others waiting.
struct Job {
  int tile, split, b, hk;
  int64_t bh;
};
__device__ __forceinline__ Job job_of(const XArgs& a) {
  const uint32_t groups = gridDim.x / a.tiles, even = groups / 8 * 8, at = blockIdx.x;
  uint32_t group;
  Job j;
  if (at < even * a.tiles) {
    const uint32_t i = at / 8;
    group = i / a.tiles * 8 + at % 8;
    j.tile = i % a.tiles;
  } else {
    const uint32_t i = at - even * a.tiles;
    group = even + i / a.tiles;
    j.tile = i % a.tiles;
  }
  j.split = group % a.splits;
  j.bh = group / a.splits;
  j.b = (int)(j.bh / a.Hkv);
  j.hk = (int)(j.bh % a.Hkv);
  return j;
}

// The same with the longest batch entries first, where their masks tell them apart: blocks that begin
// together should take equally long, and the last ones to begin be short.  16 samples of a mask are
// enough to order by, and any order gives the same results.  (8 x 12 heads, 997 x 2011 keys, lengths
// of a quarter to all of them, D = 64 bf16: 55, 63 and 67 us in three orders given, 48, 51 and 62 so; 32 x
// 12 heads, 512 x 2011 115 and 101; D = 128 the same either way.)
constexpr int ORDER_MOST = 64, ORDER_SAMPLES = 16;
__device__ __forceinline__ Job job_longest_first(const XArgs& a, int t) {
  Job j = job_of(a);
  if (!a.longest_first) return j;
  __shared__ int kept[ORDER_MOST], chosen;
  constexpr int AT_ONCE = 64 * NW / ORDER_SAMPLES;
  const int sample = t % ORDER_SAMPLES;
  const int64_t key = (int64_t)a.Lk * (2 * sample + 1) / (2 * ORDER_SAMPLES);
#pragma unroll
  for (int i = 0; i < ORDER_MOST / AT_ONCE; ++i) {
    const int b = i * AT_ONCE + t / ORDER_SAMPLES;
    const uint64_t on = __ballot(b < a.B && a.keep[b * a.keep_bs + key]);
    if (sample == 0)
      kept[b] = __popc((uint32_t)(on >> (t & 63 & ~(ORDER_SAMPLES - 1))) & ((1u << ORDER_SAMPLES) - 1));
  }
  __syncthreads();
  if (t < a.B) {
    int before = 0;
    for (int b = 0; b < a.B; ++b) before += kept[b] > kept[t] || (kept[b] == kept[t] && b < t);
    if (before == j.b) chosen = t;
  }
  __syncthreads();
  j.b = chosen;
  j.bh = (int64_t)j.b * a.Hkv + j.hk;
  return j;
}

// The block's waves: WR of them along the rows (32 each), NW / WR along the staged keys, KT at a time.
// OCC: waves a SIMD is to hold, which is what its registers are shared by.  Tiles are staged into one
// buffer while the other is computed, where two fit.
template <class M, int DP, int WR>
struct Shape {
  typedef typename M::elem E;
  static constexpr bool HALF = sizeof(E) == 2;
  static constexpr int WK = NW / WR;
  static constexpr int KT = HALF && WR == NW ? 64 : 32 * WK;
  static constexpr int NU = KT / 32 / WK;  // a wave's 32-key products in a tile
  static constexpr int FWD_OCC = HALF && DP == 64 ? 3 : 2;
  static constexpr int BWD_OCC = HALF || (DP == 64 && WR == NW) ? 2 : 1;
  static constexpr int TILE = KT * DP;  // elements of K, and of V
  static constexpr int BUFS = 4 * TILE * (int)sizeof(E) <= 131072 ? 2 : 1;
  static constexpr int JOIN = (NW - WR) * (DP * 32 + 128) * 4;  // bytes, at the end
  static constexpr int BYTES = 2 * TILE * (int)sizeof(E) > JOIN ? 2 * TILE * (int)sizeof(E) : JOIN;
};

// Runs over the live tiles of the block's keys [k_lo, k_hi): for each, compute(K, V, the tile's
// words).  ZERO_K: masked keys' rows of K become zeros as V's do.  ready: the words of the first span are
// there already.
template <class T, class M, int DP, int WR, bool ZERO_K, class KAt, class VAt, class F>
__device__ __forceinline__ void for_tiles(char* lds0, char* lds1, uint32_t* words,
                                          const uint8_t* keep, int64_t k_lo, int64_t k_hi, int D,
                                          KAt k_at, VAt v_at, int t, int wave, int lane, bool ready,
                                          F compute) {
  typedef Shape<M, DP, WR> S;
  typedef typename M::elem E;
  constexpr int KT = S::KT;
  for (int64_t base = k_lo; base < k_hi; base += SPAN) {
    if (base > k_lo || !ready) {
      __syncthreads();
      span_words(words, keep, base, k_hi, t, 64 * NW);
      __syncthreads();
    }
    const int last = (int)min((int64_t)SPAN, k_hi - base);
    const auto load = [&](char* lds, int at) {
      E* k = reinterpret_cast<E*>(lds);
      stage<E, DP, KT>(k, base + at, k_hi - 1, D, k_at, wave, lane);
      stage<E, DP, KT>(k + S::TILE, base + at, k_hi - 1, D, v_at, wave, lane);
    };
    const auto take = [&](char* lds, int at) {
      E* k = reinterpret_cast<E*>(lds);
      uint32_t all = ~0u;
#pragma unroll
      for (int u = 0; u < KT / 32; ++u) all &= words[at / 32 + u];
      if (all != ~0u) {  // the same for every wave
        if (ZERO_K) patch<E, DP, KT>(k, words + at / 32, t);
        patch<E, DP, KT>(k + S::TILE, words + at / 32, t);
        __syncthreads();
      }
      compute(k, k + S::TILE, words + at / 32);
    };
    int at = next_tile<KT>(words, 0, last);
    if (at >= last) continue;
    load(lds0, at);
    landed();
    __syncthreads();
    if constexpr (S::BUFS == 2) {
      for (;;) {
        const int b = next_tile<KT>(words, at + KT, last);
        if (b < last) load(lds1, b);
        take(lds0, at);
        if (b >= last) break;
        landed();
        __syncthreads();
        at = next_tile<KT>(words, b + KT, last);
        if (at < last) load(lds0, at);
        take(lds1, b);
        if (at >= last) break;
        landed();
        __syncthreads();
      }
    } else {
      for (;;) {
        take(lds0, at);
        at = next_tile<KT>(words, at + KT, last);
        if (at >= last) break;
        __syncthreads();
        load(lds0, at);
        landed();
        __syncthreads();
      }
    }
  }
}

// ---- forward -------------------------------------------------------------------------------------
// The running maximum follows the scores only when they pass it by more than 8 (in base 2): until
// then exponentials up to 2^8 share the old base, and the sums need no rescaling.
// FINE: P to 16 bits as an operand (bf16).  Where one key carries a row, P's rounding reaches the output
// and the backward's row sum at full size, where many do it averages out: at 2 keys, gradients 1.7
// times as far off as their own rounding takes them, 1.45 times with P to 16 bits.  So few keys are
// multiplied FINE (2048 rows x 256 keys, 96 heads of 64: 42 us against 36), and what counts are those
// that the mask keeps, however far a batch is padded.
//
// What bounds it are the matrix cores and the vector work of the exponentials (16 a lane for each 32 x 32
// scores), which overlap little: at D = 128 the matrix pipes are busy 40 % of the cycles and the
// vector pipes 45 %, at D = 64 30 and 60 %.  32 rows a wave hold Q, the scores and the sums in registers
// with two waves a SIMD (three at D = 64); four waves along the rows read a staged tile of 64 keys four
// times.  4 x 16 heads over 4, 1024 x 4096 keys, D = 128 in bf16, in a graph, 154 to 174 us (790 to 890
// TFLOP/s; profiled, where passes stand apart, 186 on average and 173 at least), D = 64 103 us
// (670); in fp32, whose products take 16 times as long and hide the rest, 1030 us and 562 us (133 and
// 122 of 154 TFLOP/s).
template <class T, class M, int DP, int WR, bool FINE>
__device__ __forceinline__ void xattn_fwd_block(const XArgs& a, const Job& j, const uint8_t* keep,
                                                char* lds, char* lds1, uint32_t* words, int t,
                                                int lane, int wave, bool ready) {
  typedef Shape<M, DP, WR> S;
  typedef typename M::elem E;
  constexpr int WK = S::WK, NU = S::NU, NC = DP / M::CHUNK;
  const int wr = wave % WR, wk = wave / WR;
  const int row = (j.tile * WR + wr) * 32 + (lane & 31);
  const bool in = row < a.R;
  const RowAt ra = row_at(a, j.hk, in ? row : 0);
  const T* k = static_cast<const T*>(a.k) + j.b * a.k_bs + j.hk * a.k_hs;
  const T* v = static_cast<const T*>(a.v) + j.b * a.v_bs + j.hk * a.v_hs;
  const auto k_at = [&](int64_t r) { return k + r * a.k_ls; };
  const auto v_at = [&](int64_t r) { return v + r * a.v_ls; };
  typename M::frag q[NC];
  load_rows<T, M, DP>(q, static_cast<const T*>(a.q) + j.b * a.q_bs + ra.i * a.q_ls + ra.h * a.q_hs,
                      in, a.D, lane);
  f32x16 acc[DP / 32] = {};
  float m = -INFINITY, l = 0.f;  // of the unscaled scores
  bool some = false;             // the block's share has a key
  const int64_t k_lo = (int64_t)j.split * a.per_split, k_hi = min((int64_t)a.Lk, k_lo + a.per_split);
  for_tiles<T, M, DP, WR, false>(lds, lds1, words, keep, k_lo, k_hi, a.D, k_at, v_at, t, wave, lane,
                                 ready, [&](const E* ks, const E* vs, const uint32_t* on) {
      some = true;
      const int u0 = wk * NU;
      uint32_t bits[NU], any = 0, all = ~0u;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        bits[u] = __builtin_amdgcn_readfirstlane(on[u0 + u]);
        any |= bits[u];
        all &= bits[u];
      }
      if (any == 0) return;  // none of this wave's keys
      f32x16 s[NU];
      float top = m;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        s[u] = f32x16{};
        rows_mma<M, DP>(ks, 32 * (u0 + u), q, s[u], lane);
      }
      if (all != ~0u) {
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[u][r] = (bits[u] >> acc_row(r, lane)) & 1 ? s[u][r] : -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
      top = halves(top, [](float x, float y) { return fmaxf(x, y); });
      if (__ballot(top > m + a.slack)) {
        const float alpha = top == -INFINITY ? 1.f : exp2_fast((m - top) * a.c);
        m = top;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] *= alpha;
      }
      const float zero = m == -INFINITY ? 0.f : -m * a.c;
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[u][r] = exp2_fast(fmaf(s[u][r], a.c, zero));
#pragma unroll
      for (int u = 0; u < NU; ++u) l += cols_mma<M, DP, FINE>(vs, 32 * (u0 + u), s[u], acc, lane);
  });
  l = halves(l, [](float x, float y) { return x + y; });
  if constexpr (WK > 1) {  // the waves along the keys
    __syncthreads();
    float* join = reinterpret_cast<float*>(lds);
    constexpr int SLOT = DP * 32 + 128;
    if (wk) {
      float* o = join + ((wk - 1) * WR + wr) * SLOT;
      acc_out(o, acc, lane);
      o[DP * 32 + lane] = m;
      o[DP * 32 + 64 + lane] = l;
    }
    __syncthreads();
    if (wk) return;
    for (int w = 0; w < WK - 1; ++w) {
      const float* o = join + (w * WR + wr) * SLOT;
      const float m2 = o[DP * 32 + lane], l2 = o[DP * 32 + 64 + lane], top = fmaxf(m, m2);
      const float x = top == -INFINITY ? 1.f : exp2_fast((m - top) * a.c);
      const float y = top == -INFINITY ? 1.f : exp2_fast((m2 - top) * a.c);
      acc_join(o, acc, x, y, lane);
      l = l * x + l2 * y;
      m = top;
    }
  }
  if (!in) return;
  if (a.splits > 1) {
    const int64_t at = ((int64_t)j.split * a.B * a.Hkv + j.bh) * a.R + row;
    float* o = a.part + at * a.D;
    for_runs<DP>(acc, lane, [&](int d, const float (&x)[4]) {
      if (d < a.D) store_f<float, 4>(o + d, x);
    });
    if (lane < 32) {
      a.part_ms[2 * at] = m * a.c;
      a.part_ms[2 * at + 1] = some && l == 0.f ? NONE_FINITE : l;
    }
    return;
  }
  const float inv = inv_sum(l, some);
  const int64_t at = (((int64_t)j.b * a.Lq + ra.i) * a.H + ra.h) * a.D;
  for_runs<DP>(acc, lane, [&](int d, const float (&x)[4]) {
    const float y[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
    if (d < a.D) store_out<T, 4>(a, at + d, y);
  });
  if (lane < 32 && a.lse)
    a.lse[((int64_t)j.b * a.H + ra.h) * a.Lq + ra.i] = lse_of(m * a.c, l, some);
}

constexpr int FINE_KEYS = 256;
template <class T, class M, int DP, int WR>
__global__ __launch_bounds__(64 * NW, (Shape<M, DP, WR>::FWD_OCC)) void xattn_fwd_kernel(XArgs a) {
  typedef Shape<M, DP, WR> S;
  __shared__ __align__(16) char lds[S::BYTES];
  __shared__ __align__(16) char lds1[S::BUFS == 2 ? S::BYTES : 16];
  __shared__ uint32_t words[SPAN / 32];
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const Job j = job_longest_first(a, t);
  const uint8_t* keep = a.keep ? a.keep + j.b * a.keep_bs : nullptr;
  bool fine = a.Lk <= FINE_KEYS, ready = false;
  if constexpr (std::is_same_v<T, bf16>) {
    if (keep && !fine) {
      // a share of a long row may hold half of FINE_KEYS by itself: it is split at 256 keys at least
      const int most = a.splits > 1 ? FINE_KEYS / 2 : FINE_KEYS;
      const int64_t k_lo = (int64_t)j.split * a.per_split;
      const int64_t k_hi = min((int64_t)a.Lk, k_lo + a.per_split);
      int kept = 0;
      for (int64_t base = k_lo; base < k_hi && kept <= most; base += SPAN) {
        __syncthreads();
        span_words(words, keep, base, k_hi, t, 64 * NW);
        __syncthreads();
        kept += span_keys(words, (int)min((int64_t)SPAN, k_hi - base), lane);
        ready = base == k_lo;
      }
      fine = kept <= most;
    }
    if (fine) {
      xattn_fwd_block<T, M, DP, WR, true>(a, j, keep, lds, lds1, words, t, lane, wave, ready);
      return;
    }
  }
  xattn_fwd_block<T, M, DP, WR, false>(a, j, keep, lds, lds1, words, t, lane, wave, ready);
}

// The splits of a row: rescaled to their common maximum and summed in order.  A wave per row, whose
// lanes read the splits' statistics side by side and then AHEAD of their rows at a time: the time is
// the latency of these reads (1024 rows of 4 splits 4.8 us; one split after the other 8.7).
template <class T>
__global__ __launch_bounds__(256) void xattn_join_kernel(XArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t rows = (int64_t)a.B * a.Hkv * a.R;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= rows) return;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2* ms = reinterpret_cast<const f32x2*>(a.part_ms);
  constexpr int AHEAD = 8;
  const f32x2 none = {-INFINITY, 0.f};
  const f32x2 first = lane < a.splits ? ms[lane * rows + at] : none;
  float m = first[0];
  for (int s = lane + 64; s < a.splits; s += 64) m = fmaxf(m, ms[s * rows + at][0]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[2] = {0.f, 0.f};
  bool some = false;
  for (int s0 = 0; s0 < a.splits; s0 += 64) {  // a lane per split, for its weight
    const int n = min(64, a.splits - s0);
    const f32x2 x = s0 == 0 ? first : lane < n ? ms[(s0 + lane) * rows + at] : none;
    some = some || __ballot(x[1] == NONE_FINITE);
    const float w = exp2_fast(x[0] - base);
    l += wave_add(w * x[1]);
    for (int s = 0; s < n; s += AHEAD) {
      float y[AHEAD][2];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int d = lane + 64 * j;
          y[u][j] = s + u < n && d < a.D ? a.part[((s0 + s + u) * rows + at) * a.D + d] : 0.f;
        }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const float f = __shfl(w, min(s + u, n - 1), 64);
#pragma unroll
        for (int j = 0; j < 2; ++j) o[j] += f * y[u][j];
      }
    }
  }
  const int64_t bh = at / a.R;
  const int b = (int)(bh / a.Hkv), hk = (int)(bh % a.Hkv);
  const RowAt ra = row_at(a, hk, (int)(at % a.R));
  const float inv = inv_sum(l, some);
  const int64_t to = (((int64_t)b * a.Lq + ra.i) * a.H + ra.h) * a.D;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int d = lane + 64 * j;
    const float y[1] = {o[j] * inv};
    if (d < a.D) store_out<T, 1>(a, to + d, y);
  }
  if (lane == 0 && a.lse)
    a.lse[((int64_t)b * a.H + ra.h) * a.Lq + ra.i] = lse_of(m, l, some);
}

// ---- a few rows (single tokens) ------------------------------------------------------------------
// The keys and values are read once and that is all the time there is: no matrix core, and LDS only
// for the mask's bits and the end.  LPR lanes read a key's row, 16 bytes each, so a wave reads 64 /
// LPR keys at a time; each such group of lanes keeps its own running maximum, sum and output share
// of every row (the maximum moves as the tiled kernel's does), and they are joined when the keys are
// done.  The wave's next FEW_AHEAD reads are on their way while the present ones are computed.  32 x 8 key heads of 4 rows, 8192 keys, D = 128 in
// bf16: 190 us, 5.7 TB/s (with every lane taking every row's exponential 199, and 184 against 163 for
// ragged lengths, where the longest head's blocks are bound by their vector work); 16 x 12 heads, 562
// keys, D = 64 in fp32 9.6 us, half of it until the first keys are there.  (Reading the first keys
// before the mask is known made masked batches slower, 66 us against 60.)
constexpr int FEW_WAVES = 8, FEW_AHEAD = 4;

// f over the lanes that hold the same column of neighbouring groups of LPR, in all of them
template <int LPR, class F>
__device__ __forceinline__ float across(float x, F f) {
  if constexpr (LPR == 8) x = f(x, permuted<0x128>(x));  // turned by 8 within 16: lane ^ 8
  if constexpr (LPR <= 16) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = f(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
  }
  return halves(x, f);
}

// Sums of NR rows over the lanes of a group, one row to a lane: instead of NR sums in every lane, each
// exchange halves the rows that a lane goes on with, so a score's exponential is taken once for every
// 8 lanes' rows, not in each.  Row r is then held by lane lane_of<NR>(r) of every 8.
template <int NR>
constexpr int lane_of(int r) {
  return NR == 1 ? 0 : NR == 2 ? 4 * r : NR == 4 ? 4 * (r >> 1) + (r & 1)
                                                 : 4 * (r >> 2) + (r >> 1 & 1) + 2 * (r & 1);
}
template <int LPR, int NR>
__device__ __forceinline__ float row_sums(const float (&y)[NR], int lane) {
  if constexpr (NR == 1) {
    return group_add<LPR>(y[0]);
  } else {
    const bool b0 = lane & 1, b1 = lane & 2, b2 = lane & 4;
    float x, a[NR / 2];
#pragma unroll
    for (int i = 0; i < NR / 2; ++i)
      a[i] = (b2 ? y[NR / 2 + i] : y[i]) + permuted<0x141>(b2 ? y[i] : y[NR / 2 + i]);
    if constexpr (NR == 2) {
      x = a[0] + permuted<0xB1>(a[0]);
      x += permuted<0x4E>(x);
    } else if constexpr (NR == 4) {
      x = (b0 ? a[1] : a[0]) + permuted<0xB1>(b0 ? a[0] : a[1]);
      x += permuted<0x4E>(x);
    } else {
      float b[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        b[i] = (b0 ? a[2 + i] : a[i]) + permuted<0xB1>(b0 ? a[i] : a[2 + i]);
      x = (b1 ? b[1] : b[0]) + permuted<0x4E>(b1 ? b[0] : b[1]);
    }
    if constexpr (LPR >= 16) x += permuted<0x128>(x);  // lane ^ 8
    if constexpr (LPR == 32) {
      const uint32_t u = __builtin_bit_cast(uint32_t, x);
      const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
      x = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
    }
    return x;
  }
}
// and back: the value of every row in every lane of the group
template <int LPR, int NR, int R = 0>
__device__ __forceinline__ void row_values(float x, float lo, float hi, float (&all)[NR]) {
  constexpr int L = lane_of<NR>(R);
  if constexpr (LPR == 8) all[R] = permuted<(L & 3) * 0x55>(L & 4 ? hi : lo);
  else all[R] = permuted<0x150 + L>(x);  // lane L of the 16 to all of them
  if constexpr (R + 1 < NR) row_values<LPR, NR, R + 1>(x, lo, hi, all);
}
template <int LPR, int NR>
__device__ __forceinline__ void row_values(float x, int lane, float (&all)[NR]) {
  if constexpr (NR == 1) {
    all[0] = x;
  } else {
    float lo = x, hi = x;  // of 8 lanes, the lower four's values and the upper four's
    if constexpr (LPR == 8) {
      const float down = permuted<0x124>(x), up = permuted<0x12C>(x);  // from lane - 4, lane + 4
      lo = lane & 4 ? down : x;
      hi = lane & 4 ? x : up;
    }
    row_values<LPR, NR, 0>(x, lo, hi, all);
  }
}

// The dot product of two 16-byte runs (of 2-byte types in exact pair products), from `x` on.
template <class T>
__device__ __forceinline__ float dot16(const typename Vec<T, VEC16<T>>::type& a,
                                       const typename Vec<T, VEC16<T>>::type& b, float x) {
  if constexpr (sizeof(T) == 2) {
    typedef T pair __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      if constexpr (std::is_same_v<T, bf16>)
        x = __builtin_amdgcn_fdot2_f32_bf16(pair{a[e], a[e + 1]}, pair{b[e], b[e + 1]}, x, false);
      else
        x = __builtin_amdgcn_fdot2(pair{a[e], a[e + 1]}, pair{b[e], b[e + 1]}, x, false);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x = fmaf(a[e], b[e], x);
  }
  return x;
}

template <class T, int LPR, int NR>
__global__ __launch_bounds__(64 * FEW_WAVES) void xattn_few_kernel(XArgs a) {
  constexpr int N = VEC16<T>, KPI = 64 / LPR, GROUP = KPI * FEW_AHEAD, STEP = FEW_WAVES * GROUP;
  constexpr uint32_t GROUP_BITS = GROUP == 32 ? ~0u : (1u << (GROUP % 32)) - 1;
  __shared__ float so[FEW_WAVES][NR][LPR * N];
  __shared__ float sm[FEW_WAVES][NR][2];
  __shared__ uint32_t words[SPAN / 32];
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  // The first share of every head, then the second, ...: a head's last shares may lie behind its
  // length, and with its shares side by side one XCD got all the last ones.  Each share begins with
  // another head, so that a CU's blocks are of different batch entries.
  const uint32_t heads = (uint32_t)(a.B * a.Hkv);
  const int split = (int)(blockIdx.x / heads);
  const int64_t bh = (blockIdx.x % heads + (uint64_t)split * heads / a.splits) % heads;
  const int b = (int)(bh / a.Hkv), hk = (int)(bh % a.Hkv);
  const T* k = static_cast<const T*>(a.k) + b * a.k_bs + hk * a.k_hs;
  const T* v = static_cast<const T*>(a.v) + b * a.v_bs + hk * a.v_hs;
  const uint8_t* keep = a.keep ? a.keep + b * a.keep_bs : nullptr;
  const int d0 = (lane % LPR) * N, sub = lane / LPR;
  const bool act = d0 < a.D;
  typedef typename Vec<T, N>::type Run;
  Run q[NR];
  float o[NR][N], m = -INFINITY, l = 0.f;  // m, l: of the lane's row, unscaled scores
  bool some = false;                       // the wave has had a key
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    q[r] = Run{};
#pragma unroll
    for (int e = 0; e < N; ++e) o[r][e] = 0.f;
    if (r < a.R && act) {
      const RowAt ra = row_at(a, hk, r);
      q[r] = *reinterpret_cast<const Run*>(static_cast<const T*>(a.q) + b * a.q_bs +
                                           ra.i * a.q_ls + ra.h * a.q_hs + d0);
    }
  }
  struct Ahead {
    typename Vec<T, N>::type k[FEW_AHEAD], v[FEW_AHEAD];
    bool ok[FEW_AHEAD];
  };
  const int64_t k_lo = (int64_t)split * a.per_split, k_hi = min((int64_t)a.Lk, k_lo + a.per_split);
  for (int64_t base = k_lo; base < k_hi; base += SPAN) {
    __syncthreads();
    span_words(words, keep, base, k_hi, t, 64 * FEW_WAVES);
    __syncthreads();
    const int last = (int)min((int64_t)SPAN, k_hi - base);
    const auto next = [&](int g) {  // the wave's next group with a key
      while (g < last && !((words[g >> 5] >> (g & 31)) & GROUP_BITS)) g += STEP;
      return g;
    };
    const auto load = [&](Ahead& x, int g) {
#pragma unroll
      for (int u = 0; u < FEW_AHEAD; ++u) {
        const int i = g + u * KPI + sub;
        x.ok[u] = (words[i >> 5] >> (i & 31)) & 1;
        x.k[u] = x.v[u] = typename Vec<T, N>::type{};
        if (x.ok[u] && act) {
          x.k[u] = *reinterpret_cast<const typename Vec<T, N>::type*>(k + (base + i) * a.k_ls + d0);
          x.v[u] = *reinterpret_cast<const typename Vec<T, N>::type*>(v + (base + i) * a.v_ls + d0);
        }
      }
    };
    const auto take = [&](const Ahead& x) {
      some = true;
      float s[FEW_AHEAD], top = m;
#pragma unroll
      for (int u = 0; u < FEW_AHEAD; ++u) {
        float y[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) y[r] = dot16<T>(q[r], x.k[u], 0.f);
        const float z = row_sums<LPR, NR>(y, lane);
        s[u] = x.ok[u] ? z : -INFINITY;
        top = fmaxf(top, s[u]);
      }
      if (__ballot(top > m + a.slack)) {
        float alpha[NR];
        const float mine = top == -INFINITY ? 1.f : exp2_fast((m - top) * a.c);
        m = top;
        l *= mine;
        row_values<LPR, NR>(mine, lane, alpha);
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int e = 0; e < N; ++e) o[r][e] *= alpha[r];
      }
      const float zero = m == -INFINITY ? 0.f : -m * a.c;
#pragma unroll
      for (int u = 0; u < FEW_AHEAD; ++u) l += s[u] = exp2_fast(fmaf(s[u], a.c, zero));
#pragma unroll
      for (int u = 0; u < FEW_AHEAD; ++u) {
        float f[N], p[NR];
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = vec_f<T, N>(x.v[u], e);
        row_values<LPR, NR>(s[u], lane, p);
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int e = 0; e < N; ++e) o[r][e] = fmaf(p[r], f[e], o[r][e]);
      }
    };
    Ahead x, y;
    int g = next(wave * GROUP);
    if (g < last) load(x, g);
    while (g < last) {
      const int g2 = next(g + STEP);
      if (g2 < last) load(y, g2);
      take(x);
      if (g2 >= last) break;
      g = next(g2 + STEP);
      if (g < last) load(x, g);
      take(y);
    }
  }
  {  // the wave's groups of lanes
    const auto add = [](float x, float y) { return x + y; };
    const float top = across<LPR>(m, [](float x, float y) { return fmaxf(x, y); });
    const float mine = top == -INFINITY ? 1.f : exp2_fast((m - top) * a.c);
    l = across<LPR>(l * mine, add);
    float w[NR];
    row_values<LPR, NR>(mine, lane, w);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        o[r][e] = across<LPR>(o[r][e] * w[r], add);
        if (lane < LPR) so[wave][r][d0 + e] = o[r][e];
      }
      if (lane == lane_of<NR>(r)) {
        sm[wave][r][0] = top * a.c;
        sm[wave][r][1] = some && l == 0.f ? NONE_FINITE : l;
      }
    }
  }
  __syncthreads();
  for (int i = t; i < a.R * a.D; i += 64 * FEW_WAVES) {  // the block's waves
    const int r = i / a.D, d = i - r * a.D;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < FEW_WAVES; ++w) top = fmaxf(top, sm[w][r][0]);
    const float zero = top == -INFINITY ? 0.f : top;
    float x = 0.f, sum = 0.f;
    bool none_finite = false;
#pragma unroll
    for (int w = 0; w < FEW_WAVES; ++w) {
      const float f = exp2_fast(sm[w][r][0] - zero);
      x += f * so[w][r][d];
      sum += f * sm[w][r][1];
      none_finite = none_finite || sm[w][r][1] == NONE_FINITE;
    }
    if (a.splits > 1) {
      const int64_t at = ((int64_t)split * a.B * a.Hkv + bh) * a.R + r;
      a.part[at * a.D + d] = x;
      if (d == 0) {
        a.part_ms[2 * at] = top;
        a.part_ms[2 * at + 1] = none_finite && sum == 0.f ? NONE_FINITE : sum;
      }
    } else {
      const RowAt ra = row_at(a, hk, r);
      const float y[1] = {sum == 0.f ? (none_finite ? NAN : 0.f) : x / sum};
      store_out<T, 1>(a, (((int64_t)b * a.Lq + ra.i) * a.H + ra.h) * a.D + d, y);
      if (d == 0 && a.lse)
        a.lse[((int64_t)b * a.H + ra.h) * a.Lq + ra.i] = lse_of(top, sum, none_finite);
    }
  }
}

// ---- backward ------------------------------------------------------------------------------------
// delta[b, h, i] = sum_d dO O, where dQ, which computes it on its way, is not wanted: two lanes a row,
// the sums in dQ's order (the same bits).
template <class T, class M>
__global__ __launch_bounds__(256) void xattn_delta_kernel(XArgs a) {
  constexpr int N = M::CHUNK / 2;
  const int64_t row = (int64_t)blockIdx.x * 128 + (threadIdx.x >> 1);  // (b, i, h)
  const int half = threadIdx.x & 1;
  float s = 0.f;
  const bool in = row < (int64_t)a.B * a.Lq * a.H;
  const int h = (int)(row % a.H);
  const int64_t bi = row / a.H;
  const int i = (int)(bi % a.Lq), b = (int)(bi / a.Lq);
  for (const void* part : {a.o, a.o_rest})
    for (int d = N * half; part && in && d < a.D; d += M::CHUNK) {
      float x[N], y[N];
      load_f<T, N>(static_cast<const T*>(part) + row * a.D + d, x);
      load_f<T, N>(static_cast<const T*>(a.dout) + b * a.do_bs + i * a.do_ls + h * a.do_hs + d, y);
#pragma unroll
      for (int e = 0; e < N; ++e) s = fmaf(y[e], x[e], s);
    }
  s += __shfl_xor(s, 1, 64);
  if (in && half == 0) a.delta[((int64_t)b * a.H + h) * a.Lq + i] = s;
}

// dQ: WR of the block's waves along the rows (32 each), the others along the staged keys.  Scores and
// dP come from one pass over K and V by rows, dS goes on to the third product in registers, and delta
// is formed from O and dO while the first tile is on its way.  Three products for two of the forward's,
// bound as it is: 4 x 16 heads over 4, 1024 x 4096, D = 128 in bf16 207 us in a graph, 234 profiled
// (1000, 880 TFLOP/s of its 6 B H Lq Lk D, where a large product reaches 1072).
template <class T, class M, int DP, int WR>
__global__ __launch_bounds__(64 * NW, (Shape<M, DP, WR>::BWD_OCC)) void xattn_dq_kernel(XArgs a) {
  typedef Shape<M, DP, WR> S;
  typedef typename M::elem E;
  constexpr int WK = S::WK, NU = S::NU, NC = DP / M::CHUNK;
  __shared__ __align__(16) char lds[S::BYTES];
  __shared__ __align__(16) char lds1[S::BUFS == 2 ? S::BYTES : 16];
  __shared__ uint32_t words[SPAN / 32];
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6), wr = wave % WR, wk = wave / WR;
  const Job j = job_longest_first(a, t);
  const int row = (j.tile * WR + wr) * 32 + (lane & 31);
  const bool in = row < a.R;
  const RowAt ra = row_at(a, j.hk, in ? row : 0);
  const T* k = static_cast<const T*>(a.k) + j.b * a.k_bs + j.hk * a.k_hs;
  const T* v = static_cast<const T*>(a.v) + j.b * a.v_bs + j.hk * a.v_hs;
  const uint8_t* keep = a.keep ? a.keep + j.b * a.keep_bs : nullptr;
  const auto k_at = [&](int64_t r) { return k + r * a.k_ls; };
  const auto v_at = [&](int64_t r) { return v + r * a.v_ls; };
  typename M::frag q[NC], go[NC];
  load_rows<T, M, DP>(q, static_cast<const T*>(a.q) + j.b * a.q_bs + ra.i * a.q_ls + ra.h * a.q_hs,
                      in, a.D, lane);
  load_rows<T, M, DP>(go,
                      static_cast<const T*>(a.dout) + j.b * a.do_bs + ra.i * a.do_ls +
                          ra.h * a.do_hs,
                      in, a.D, lane);
  const int64_t stat = ((int64_t)j.b * a.H + ra.h) * a.Lq + ra.i;
  const float lse = in ? a.lse[stat] : -INFINITY;
  float delta = 0.f;
  for (const void* part : {a.o, a.o_rest}) {
    if (!part) continue;
    typename M::frag o[NC];
    load_rows<T, M, DP>(o,
                        static_cast<const T*>(part) + (((int64_t)j.b * a.Lq + ra.i) * a.H + ra.h) *
                                                          a.D,
                        in, a.D, lane);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < M::CHUNK / 2; ++e) delta = fmaf((float)go[c][e], (float)o[c][e], delta);
  }
  delta = halves(delta, [](float x, float y) { return x + y; });
  if (in && lane < 32 && wk == 0 && j.split == 0) a.delta[stat] = delta;
  // a row without a key (and one that does not exist) has exponents of -inf: P = 0
  const float neg = lse == -INFINITY ? -INFINITY : -lse;
  f32x16 acc[DP / 32] = {};
  const int64_t k_lo = (int64_t)j.split * a.per_split, k_hi = min((int64_t)a.Lk, k_lo + a.per_split);
  for_tiles<T, M, DP, WR, true>(lds, lds1, words, keep, k_lo, k_hi, a.D, k_at, v_at, t, wave, lane,
                                false, [&](const E* ks, const E* vs, const uint32_t* on) {
#pragma unroll
      for (int u = wk * NU; u < (wk + 1) * NU; ++u) {
        const uint32_t bits = __builtin_amdgcn_readfirstlane(on[u]);
        if (bits == 0) continue;
        f32x16 s = {}, dp = {};
        rows_mma2<M, DP>(ks, vs, 32 * u, [&](int c) { return q[c]; }, [&](int c) { return go[c]; },
                         s, dp, lane);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[r] = exp2_fast(fmaf(s[r], a.c, neg)) * (dp[r] - delta);
        if (bits != ~0u)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = (bits >> acc_row(r, lane)) & 1 ? s[r] : 0.f;
        cols_mma<M, DP>(ks, 32 * u, s, acc, lane);
      }
  });
  if constexpr (WK > 1) {
    __syncthreads();
    float* join = reinterpret_cast<float*>(lds);
    if (wk) acc_out(join + ((wk - 1) * WR + wr) * DP * 32, acc, lane);
    __syncthreads();
    if (wk) return;
    for (int w = 0; w < WK - 1; ++w)
      acc_join(join + (w * WR + wr) * DP * 32, acc, 1.f, 1.f, lane);
  }
  if (!in) return;
  if (a.splits > 1) {
    float* o = a.part + (((int64_t)j.split * a.B * a.Hkv + j.bh) * a.R + row) * a.D;
    for_runs<DP>(acc, lane, [&](int d, const float (&x)[4]) {
      if (d < a.D) store_f<float, 4>(o + d, x);
    });
    return;
  }
  T* o = static_cast<T*>(a.dq) + (((int64_t)j.b * a.Lq + ra.i) * a.H + ra.h) * a.D;
  for_runs<DP>(acc, lane, [&](int d, const float (&x)[4]) {
    const float y[4] = {x[0] * a.scale, x[1] * a.scale, x[2] * a.scale, x[3] * a.scale};
    if (d < a.D) store_f<T, 4>(o + d, y);
  });
}

// dK, dV: WC of the block's waves along the keys (32 each), the others along the staged rows, RT at a
// time, over the rows of every head that shares the keys.  K and V are operands of every product and
// dK and dV sums of all: at D = 128 V waits in LDS (V_LDS), the rest leaves two waves a SIMD in bf16
// and one in fp32.  Four products: 4 x 16 heads over 4, 1024 x 4096, D = 128 in bf16 276 us in a graph,
// 319 profiled (1000, 860 TFLOP/s of its 8 B H Lq Lk D); with dQ in fp32 3750 us, 128 of 154 TFLOP/s.
template <class M, int DP, int WC>
struct DkvShape {
  typedef typename M::elem E;
  static constexpr int WS = NW / WC;
  static constexpr int RT = sizeof(E) == 2 && DP == 64 && WC == NW ? 64 : 32 * WS;
  static constexpr int NU = RT / 32 / WS;
  static constexpr int TILE = RT * DP;  // elements of Q, and of dO
  static constexpr int BUFS = 4 * TILE * (int)sizeof(E) <= 131072 ? 2 : 1;
  static constexpr int JOIN = (NW - WC) * DP * 32 * 4;  // bytes, at the end: dK, then dV
  static constexpr int BYTES = 2 * TILE * (int)sizeof(E) > JOIN ? 2 * TILE * (int)sizeof(E) : JOIN;
  static constexpr bool V_LDS = sizeof(E) == 2 && DP == 128 && WC == NW;
};

template <class T, class M, int DP, int WC>
__global__ __launch_bounds__(64 * NW, (Shape<M, DP, WC>::BWD_OCC)) void xattn_dkv_kernel(XArgs a) {
  typedef DkvShape<M, DP, WC> S;
  typedef typename M::elem E;
  constexpr int RT = S::RT, WS = S::WS, NU = S::NU;
  constexpr int NC = DP / M::CHUNK;
  __shared__ __align__(16) char lds[S::BYTES];
  __shared__ __align__(16) char lds1[S::BUFS == 2 ? S::BYTES : 16];
  // -lse (-inf: a row without a key), then delta, of the tile's rows
  __shared__ __align__(16) float st0[2 * RT], st1[2 * RT];
  __shared__ __align__(16) char v_lds[S::V_LDS ? NW * 32 * DP * (int)sizeof(E) : 16];
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6), wc = wave % WC, ws = wave / WC;
  const Job j = job_of(a);
  const int64_t key = ((int64_t)j.tile * WC + wc) * 32 + (lane & 31);
  const bool in = key < a.Lk;
  const bool ok = in && (!a.keep || a.keep[j.b * a.keep_bs + key]);
  typename M::frag k[NC], v[NC];
  load_rows<T, M, DP>(k, static_cast<const T*>(a.k) + j.b * a.k_bs + j.hk * a.k_hs + key * a.k_ls,
                      ok, a.D, lane);
  load_rows<T, M, DP>(v, static_cast<const T*>(a.v) + j.b * a.v_bs + j.hk * a.v_hs + key * a.v_ls,
                      ok, a.D, lane);
  // V's operand: in registers, or, where those would not do for two waves a SIMD, in the wave's own
  // part of LDS (read by this wave alone: no barrier)
  typename M::frag* own = reinterpret_cast<typename M::frag*>(v_lds) + wave * NC * 64 + lane;
  if constexpr (S::V_LDS)
#pragma unroll
    for (int c = 0; c < NC; ++c) own[c * 64] = v[c];
  const auto v_frag = [&](int c) -> typename M::frag {
    if constexpr (S::V_LDS) return own[c * 64];
    else return v[c];
  };
  const T* q = static_cast<const T*>(a.q) + j.b * a.q_bs;
  const T* go = static_cast<const T*>(a.dout) + j.b * a.do_bs;
  const auto q_at = [&](int64_t r) {
    const RowAt ra = row_at(a, j.hk, (int)r);
    return q + ra.i * a.q_ls + ra.h * a.q_hs;
  };
  const auto g_at = [&](int64_t r) {
    const RowAt ra = row_at(a, j.hk, (int)r);
    return go + ra.i * a.do_ls + ra.h * a.do_hs;
  };
  f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
  const int r_lo = j.split * a.per_split, r_hi = min(a.R, r_lo + a.per_split);
  const bool live = __syncthreads_or(ok);  // a tile of padding has no gradient
  const bool mine = __ballot(ok) != 0;
  const bool whole = __ballot(ok) == ~0ull;
  float stat[2] = {-INFINITY, 0.f};
  const auto load = [&](char* to, int r0) {
    E* qs = reinterpret_cast<E*>(to);
    stage<E, DP, RT>(qs, r0, r_hi - 1, a.D, q_at, wave, lane);
    stage<E, DP, RT>(qs + S::TILE, r0, r_hi - 1, a.D, g_at, wave, lane);
    if (t < RT) {
      const bool there = r0 + t < r_hi;
      const RowAt ra = row_at(a, j.hk, there ? r0 + t : 0);
      const int64_t at = ((int64_t)j.b * a.H + ra.h) * a.Lq + ra.i;
      const float lse = there ? a.lse[at] : -INFINITY;
      stat[0] = lse == -INFINITY ? -INFINITY : -lse;
      stat[1] = there ? a.delta[at] : 0.f;
    }
  };
  const auto arrive = [&](float* st) {  // what load() began is in LDS for every wave
    if (t < RT) {
      st[t] = stat[0];
      st[RT + t] = stat[1];
    }
    landed();
    __syncthreads();
  };
  const auto take = [&](const char* from, const float* st) {
    if (!mine) return;
    const E* qs = reinterpret_cast<const E*>(from);
    const E* gs = qs + S::TILE;
#pragma unroll
    for (int u = ws * NU; u < (ws + 1) * NU; ++u) {
      f32x16 s = {}, dp = {};
      rows_mma2<M, DP>(qs, gs, 32 * u, [&](int c) { return k[c]; }, v_frag, s, dp, lane);
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int i = 32 * u + acc_row(4 * r4, lane);
        const f32x4 neg = *reinterpret_cast<const f32x4*>(&st[i]);
        const f32x4 delta = *reinterpret_cast<const f32x4*>(&st[RT + i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * r4 + e;
          s[r] = exp2_fast(fmaf(s[r], a.c, neg[e]));
          dp[r] = s[r] * (dp[r] - delta[e]);
        }
      }
      if (!whole)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[r] = ok ? s[r] : 0.f;
          dp[r] = ok ? dp[r] : 0.f;
        }
      cols_mma<M, DP>(gs, 32 * u, s, dv, lane);
      cols_mma<M, DP>(qs, 32 * u, dp, dk, lane);
    }
  };
  if (live && r_lo < r_hi) {
    load(lds, r_lo);
    arrive(st0);
    if constexpr (S::BUFS == 2) {
      for (int r0 = r_lo;;) {
        if (r0 + RT < r_hi) load(lds1, r0 + RT);
        take(lds, st0);
        if ((r0 += RT) >= r_hi) break;
        arrive(st1);
        if (r0 + RT < r_hi) load(lds, r0 + RT);
        take(lds1, st1);
        if ((r0 += RT) >= r_hi) break;
        arrive(st0);
      }
    } else {
      for (int r0 = r_lo + RT;; r0 += RT) {
        take(lds, st0);
        if (r0 >= r_hi) break;
        __syncthreads();
        load(lds, r0);
        arrive(st0);
      }
    }
  }
  if constexpr (WS > 1) {
    float* join = reinterpret_cast<float*>(lds);
    const auto join_waves = [&](f32x16 (&x)[DP / 32]) {
      __syncthreads();
      if (ws) acc_out(join + ((ws - 1) * WC + wc) * DP * 32, x, lane);
      __syncthreads();
      if (!ws)
        for (int w = 0; w < WS - 1; ++w)
          acc_join(join + (w * WC + wc) * DP * 32, x, 1.f, 1.f, lane);
    };
    join_waves(dk);
    join_waves(dv);
    if (ws) return;
  }
  if (!in) return;
  if (a.splits > 1) {
    const int64_t at = (((int64_t)j.split * a.B * a.Hkv + j.bh) * a.Lk + key) * a.D;
    for_runs<DP>(dk, lane, [&](int d, const float (&x)[4]) {
      if (d < a.D) store_f<float, 4>(a.part + at + d, x);
    });
    for_runs<DP>(dv, lane, [&](int d, const float (&x)[4]) {
      if (d < a.D) store_f<float, 4>(a.part2 + at + d, x);
    });
    return;
  }
  const int64_t at = (((int64_t)j.b * a.Lk + key) * a.Hkv + j.hk) * a.D;
  for_runs<DP>(dk, lane, [&](int d, const float (&x)[4]) {
    const float y[4] = {x[0] * a.scale, x[1] * a.scale, x[2] * a.scale, x[3] * a.scale};
    if (d < a.D) store_f<T, 4>(static_cast<T*>(a.dk) + at + d, y);
  });
  for_runs<DP>(dv, lane, [&](int d, const float (&x)[4]) {
    if (d < a.D) store_f<T, 4>(static_cast<T*>(a.dv) + at + d, x);
  });
}

// The splits' shares of a gradient, summed in order.  rows: (b, key head, r); kind 0: dQ rows,
// 1: dK and dV rows.
template <class T>
__global__ __launch_bounds__(256) void xattn_sum_kernel(XArgs a, int kind) {
  const int n = kind == 0 ? a.R : a.Lk;
  const int64_t rows = (int64_t)a.B * a.Hkv * n;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= rows * a.D) return;
  const int64_t at = i / a.D;
  const int d = (int)(i - at * a.D);
  const int64_t bh = at / n;
  const int b = (int)(bh / a.Hkv), hk = (int)(bh % a.Hkv), r = (int)(at % n);
  float x[4] = {}, y[4] = {};
  for (int s = 0; s < a.splits; ++s) {
    float f[4];
    load_f<float, 4>(a.part + s * rows * a.D + i, f);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += f[e];
    if (kind == 1) {
      load_f<float, 4>(a.part2 + s * rows * a.D + i, f);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += f[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] *= a.scale;
  if (kind == 0) {
    const RowAt ra = row_at(a, hk, r);
    store_f<T, 4>(static_cast<T*>(a.dq) + (((int64_t)b * a.Lq + ra.i) * a.H + ra.h) * a.D + d, x);
  } else {
    const int64_t o = (((int64_t)b * a.Lk + r) * a.Hkv + hk) * a.D + d;
    store_f<T, 4>(static_cast<T*>(a.dk) + o, x);
    store_f<T, 4>(static_cast<T*>(a.dv) + o, y);
  }
}

// ---- host ----------------------------------------------------------------------------------------
constexpr int FEW_ROWS = 8;  // rows of a key head that the single-token kernel takes

// Blocks along one axis and shares of the other: where the tiles alone leave the chip idle, the
// other axis is split (at least `least` of it a share, a multiple of `unit`) and joined afterwards.
struct Tiling {
  int nw = 1, tiles = 1, splits = 1, per = 0;
};
// fp32 blocks are bound by the matrix cores from start to end, so what counts is how many a CU gets:
// as many shares as leave each of the `want` CUs one block, or three where that is two blocks of a
// third each.  (4 x 8 heads, 600 x 1500, D = 128: 153 us and 556 us backward against 209 and 626 in
// one share; a block of under 512 keys a wave does not pay for the join.  A bf16 block is shorter by
// far and overlaps with others on its CU: it loses by that.)
Tiling tiling(int64_t heads, int64_t n, int64_t other, int64_t want, int64_t least, int unit,
              bool fp32 = false) {
  Tiling t;
  t.nw = n <= 32 ? 1 : n <= 64 ? 2 : NW;
  // Fewer rows a block, and more waves along the other axis: where the shares of that axis would not
  // make half the blocks wanted either (2 x 8 heads, 128 rows x 449, D = 128 fp32: 70 us with 128 rows a
  // block, 30 with 32), or where half the rows just make them (8 x 8 heads, 256 x 1024, D = 64: fp32 48
  // us against 58 in two shares, bf16 18 against 22).
  while (t.nw > 1) {
    const int64_t blocks = heads * cdiv(n, 32 * t.nw), halved = heads * cdiv(n, 16 * t.nw);
    const bool scarce = 2 * blocks * std::max<int64_t>(1, other / least) < want;
    if (!scarce && !(halved <= want && 10 * halved >= 6 * want)) break;
    t.nw /= 2;
  }
  t.tiles = (int)std::max<int64_t>(1, cdiv(n, 32 * t.nw));
  const int64_t blocks = std::max<int64_t>(1, heads * t.tiles);
  int64_t s = 2 * blocks >= want ? 1 : cdiv(want, blocks);
  if (fp32) {
    s = std::max<int64_t>(1, want / blocks);
    if (s == 1 && 3 * blocks <= 2 * want) s = 3;
    if (2 * blocks >= want && other * t.nw < 512 * NW) s = 1;
  }
  s = std::max<int64_t>(1, std::min(s, other / least));
  if (fp32 && cdiv(blocks * s, want) >= s) s = 1;  // no fewer keys for a CU than in one share
  t.per = (int)(cdiv(cdiv(std::max<int64_t>(other, 1), s), unit) * unit);
  t.splits = (int)std::max<int64_t>(1, cdiv(other, t.per));
  return t;
}

// Shares of the keys for the single-token kernel, whose blocks (one a CU at a time) come in rounds of
// CUS: the number whose rounds are over first.  A round takes as long as one block reads its keys, or,
// with more blocks than memory serves at that rate (saturated: 176 of up to 4 rows, whose times at 64,
// 128, 192 and 255 heads of 8192 keys, D = 128 bf16, are 140, 144, 162 and 205 us; 240 of more rows,
// which the vector units bind), as long as memory takes; a block's beginning and end cost about as much
// as reading 24 KB for each row (256 heads of 8 rows, 4096 keys: 117 us in one share, 130 in two, 151
// in four), the join as 48 KB.  Measured with 4 rows, 8192 keys: 96 heads in 2 shares 94 us (in 1: 142,
// in 3: 123), 128 in 2 112 (144), 160 in 3 136 (148; in 2: 176), 192 in 1 162 (in 2: 180), 320 in 4 259
// (326); 8 rows, 4096 keys: 128 in 2 76 (109), 160 in 3 100 (111; in 2: 125).
// Under a mask that reckoning does not hold (shares behind an entry's length end at once and even the
// others out), so few heads are shared until each CU has a block, or two of one or two rows, as long as
// that is more than one share: lengths of a quarter to all of 6144 keys, 4 rows, 88 heads in 3 61 us
// (in 2, the best without a mask: 72); 1 row, 176 heads in 3 88 us (in 1: 106).
constexpr int64_t CUS = 256, FEW_LEAST = 512;  // keys of a share
Tiling few_tiling(int64_t heads, int64_t R, int64_t Lk, int64_t key_bytes, bool masked) {
  const double saturated = R <= 4 ? 176 : 240, ends = 24576. * R / key_bytes;
  const int64_t most = std::max<int64_t>(1, Lk / FEW_LEAST);
  Tiling t;
  double least = 0;
  for (int rounds = 0; rounds <= 8; ++rounds) {  // the most shares of so many rounds; 0: one share
    const int64_t s = std::min(most, std::max<int64_t>(1, rounds * CUS / std::max<int64_t>(1, heads)));
    const int64_t blocks = heads * s, last = blocks % CUS;
    const double each = blocks / CUS * (CUS / saturated) + (last ? std::max(1., last / saturated) : 0.);
    const double time = each * ((double)cdiv(Lk, s) + ends) + (s > 1 ? 49152. / key_bytes : 0.);
    if (rounds && time >= least) continue;
    least = time;
    t.splits = (int)s;
  }
  const int64_t want = R <= 2 ? 2 * CUS : CUS;
  if (masked && 2 * heads < want)
    t.splits = (int)std::min(most, cdiv(want, std::max<int64_t>(1, heads)));
  t.per = (int)(cdiv(cdiv(std::max<int64_t>(Lk, 1), t.splits), 64) * 64);
  t.splits = (int)std::max<int64_t>(1, cdiv(Lk, t.per));
  return t;
}

struct XPlan {
  Tiling fwd, dq, dkv;
  bool few;
  int64_t fwd_bytes, bwd_bytes, part2, part_ms, delta;  // offsets
};

int64_t up256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// (the forward's bytes are the most that either mask or none needs)
XPlan xattn_plan(const int64_t* dims, int32_t dtype, bool masked = false) {
  const bool fp32 = dtype == MPR_F32;
  const int64_t B = dims[0], H = dims[1], Hkv = dims[2], Lq = dims[3], Lk = dims[4], D = dims[5];
  const int64_t heads = B * Hkv, R = H / Hkv * Lq;
  XPlan p;
  p.few = R <= FEW_ROWS;
  const auto forward = [&](bool m) {
    return p.few ? few_tiling(heads, R, Lk, 2 * D * (fp32 ? 4 : 2), m)
                 : tiling(heads, R, Lk, 256, 256, 128, fp32);
  };
  p.fwd = forward(masked);
  p.dq = tiling(heads, R, Lk, 256, 256, 128, fp32);
  p.dkv = tiling(heads, Lk, R, 256, 256, 128, fp32);
  const int64_t splits = std::max(p.fwd.splits, forward(!masked).splits);
  int64_t at = 0;
  if (splits > 1) at = up256(splits * heads * R * D * 4);
  p.part_ms = at;
  p.fwd_bytes = at + (splits > 1 ? splits * heads * R * 8 : 0);
  p.delta = 0;
  const int64_t base = up256(B * H * Lq * 4);
  int64_t part = p.dq.splits > 1 ? p.dq.splits * heads * R * D * 4 : 0;
  int64_t kv = p.dkv.splits > 1 ? up256(p.dkv.splits * heads * Lk * D * 4) : 0;
  p.part2 = base + kv;
  p.bwd_bytes = base + std::max(part, 2 * kv);
  return p;
}

int xattn_check(const char* what, const int64_t* dims, int32_t dtype) {
  MPR_REQUIRE(dims, "%s: no dimensions", what);
  MPR_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype code %d", what, (int)dtype);
  const int64_t B = dims[0], H = dims[1], Hkv = dims[2], Lq = dims[3], Lk = dims[4], D = dims[5];
  const int64_t most = (int64_t)1 << 30;
  MPR_REQUIRE(B >= 0 && B <= most && Lq >= 0 && Lq <= most && Lk >= 0 && Lk <= most,
              "%s: B=%lld Lq=%lld Lk=%lld", what, (long long)B, (long long)Lq, (long long)Lk);
  MPR_REQUIRE(Hkv >= 1 && H >= Hkv && H % Hkv == 0 && H <= 65536,
              "%s: %lld query heads over %lld key heads", what, (long long)H, (long long)Hkv);
  MPR_REQUIRE(D >= 8 && D <= 128 && D % 8 == 0, "%s: head dim %lld (a multiple of 8 up to 128)",
              what, (long long)D);
  MPR_REQUIRE(H / Hkv * Lq <= most && B * Hkv <= most, "%s: too many rows", what);
  const XPlan p = xattn_plan(dims, dtype);
  for (const Tiling& t : {p.fwd, p.dq, p.dkv})
    MPR_REQUIRE(B * Hkv <= MAX_GRID_X / ((int64_t)t.tiles * t.splits), "%s: too many blocks", what);
  return MPR_OK;
}

XArgs xattn_args(const void* q, const void* k, const void* v, const uint8_t* keep,
                 const int64_t* dims, const int64_t* st, float scale) {
  XArgs a{};
  a.q = q; a.k = k; a.v = v; a.keep = keep;
  a.q_bs = st[0]; a.q_ls = st[1]; a.q_hs = st[2];
  a.k_bs = st[3]; a.k_ls = st[4]; a.k_hs = st[5];
  a.v_bs = st[6]; a.v_ls = st[7]; a.v_hs = st[8];
  a.keep_bs = st[9];
  a.B = (int)dims[0]; a.H = (int)dims[1]; a.Hkv = (int)dims[2];
  a.Lq = (int)dims[3]; a.Lk = (int)dims[4]; a.D = (int)dims[5];
  a.G = a.H / a.Hkv;
  a.R = a.G * a.Lq;
  // with s = 30 + ceil(log2 Lq), ceil(2^s / Lq) Lq passes 2^s by less than Lq: exact below 2^30
  a.lq_shift = 30;
  while (((int64_t)1 << (a.lq_shift - 30)) < a.Lq) ++a.lq_shift;
  a.lq_mul = (uint64_t)cdiv((int64_t)1 << a.lq_shift, std::max(a.Lq, 1));
  a.scale = scale;
  a.c = std::max(scale * LOG2E, 1e-30f);  // scale 0: exponents of 0, whatever the scores
  a.slack = 8.f / a.c;
  return a;
}

unsigned xattn_tile(XArgs& a, const Tiling& t) {
  a.tiles = t.tiles;
  a.splits = t.splits;
  a.per_split = t.per;
  const int64_t blocks = (int64_t)a.B * a.Hkv * t.tiles * t.splits;
  a.longest_first = a.keep && a.B > 1 && a.B <= ORDER_MOST && a.Lk >= 512 && blocks > 256;
  return (unsigned)blocks;
}

// Storage type -> matrix core.
template <class T>
struct MmaOf { typedef MmaF32 type; };
template <>
struct MmaOf<bf16> { typedef MmaBf16 type; };

// Tiles go from memory to LDS in 16-byte pieces, which have to lie at multiples of 4 bytes.
bool pieces_aligned(const void* p, const int64_t* st, int32_t dtype) {
  return (uintptr_t)p % 4 == 0 && (dtype == MPR_F32 || ((st[0] | st[1] | st[2]) & 1) == 0);
}

// f(integral constant DP, integral constant NW)
template <class F>
int by_tile(int D, int nw, F&& f) {
  using std::integral_constant;
  if (D <= 64) {
    if (nw == 1) return f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (nw == 2) return f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    return f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  }
  if (nw == 1) return f(integral_constant<int, 128>{}, integral_constant<int, 1>{});
  if (nw == 2) return f(integral_constant<int, 128>{}, integral_constant<int, 2>{});
  return f(integral_constant<int, 128>{}, integral_constant<int, 4>{});
}

template <class T, int NR>
int few_rows(const XArgs& a, unsigned blocks, hipStream_t s) {
  constexpr int N = VEC16<T>;
  const dim3 grid(blocks), block(64 * FEW_WAVES);
  if (a.D <= 8 * N) xattn_few_kernel<T, 8, NR><<<grid, block, 0, s>>>(a);
  else if (N == 8 || a.D <= 16 * N) xattn_few_kernel<T, 16, NR><<<grid, block, 0, s>>>(a);
  else if constexpr (N == 4) xattn_few_kernel<T, 32, NR><<<grid, block, 0, s>>>(a);
  MPR_LAUNCHED();
  return MPR_OK;
}

template <class T>
int xattn_forward(XArgs a, const XPlan& p, hipStream_t s) {
  const unsigned blocks = xattn_tile(a, p.fwd);
  if (p.few) {
    MPR_TRY(a.R == 1 ? (few_rows<T, 1>(a, blocks, s)) : a.R == 2 ? (few_rows<T, 2>(a, blocks, s))
            : a.R <= 4 ? (few_rows<T, 4>(a, blocks, s)) : (few_rows<T, 8>(a, blocks, s)));
  } else if constexpr (!std::is_same_v<T, f16>) {
    typedef typename MmaOf<T>::type M;
    MPR_TRY(by_tile(a.D, p.fwd.nw, [&](auto dp, auto nw) -> int {
      constexpr int DP = dp, WR = nw;
      xattn_fwd_kernel<T, M, DP, WR><<<blocks, 64 * NW, 0, s>>>(a);
      MPR_LAUNCHED();
      return MPR_OK;
    }));
  }
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.B * a.Hkv * a.R;
    xattn_join_kernel<T><<<dim3((unsigned)cdiv(rows, 4)), 256, 0, s>>>(a);
    MPR_LAUNCHED();
  }
  return MPR_OK;
}

template <class T>
int xattn_backward(XArgs a, const XPlan& p, hipStream_t s) {
  typedef typename MmaOf<T>::type M;
  const int64_t rows = (int64_t)a.B * a.Lq * a.H, heads = (int64_t)a.B * a.Hkv;
  if (rows && !a.dq) {
    xattn_delta_kernel<T, M><<<dim3((unsigned)cdiv(rows, 128)), 256, 0, s>>>(a);
    MPR_LAUNCHED();
  }
  if (rows && a.dq) {
    const unsigned blocks = xattn_tile(a, p.dq);
    MPR_TRY(by_tile(a.D, p.dq.nw, [&](auto dp, auto nw) -> int {
      constexpr int DP = dp, WR = nw;
      xattn_dq_kernel<T, M, DP, WR><<<blocks, 64 * NW, 0, s>>>(a);
      MPR_LAUNCHED();
      return MPR_OK;
    }));
    if (a.splits > 1) {
      xattn_sum_kernel<T><<<dim3((unsigned)cdiv(heads * a.R * a.D, 1024)), 256, 0, s>>>(a, 0);
      MPR_LAUNCHED();
    }
  }
  if (a.Lk && a.dk) {
    const unsigned blocks = xattn_tile(a, p.dkv);
    MPR_TRY(by_tile(a.D, p.dkv.nw, [&](auto dp, auto nw) -> int {
      constexpr int DP = dp, WC = nw;
      xattn_dkv_kernel<T, M, DP, WC><<<blocks, 64 * NW, 0, s>>>(a);
      MPR_LAUNCHED();
      return MPR_OK;
    }));
    if (a.splits > 1) {
      xattn_sum_kernel<T><<<dim3((unsigned)cdiv(heads * a.Lk * a.D, 1024)), 256, 0, s>>>(a, 1);
      MPR_LAUNCHED();
    }
  }
  return MPR_OK;
}

}  // namespace
}  // namespace mpr

using namespace mpr;

extern "C" {

int mpr_xattn_workspace(const int64_t* dims, int32_t dtype, int64_t* fwd_bytes,
                        int64_t* bwd_bytes) {
  return ops_call("xattn_workspace", [&]() -> int {
    MPR_TRY(xattn_check("xattn_workspace", dims, dtype));
    MPR_REQUIRE(fwd_bytes && bwd_bytes, "xattn_workspace: null pointer");
    const XPlan p = xattn_plan(dims, dtype);
    *fwd_bytes = p.fwd_bytes;
    *bwd_bytes = p.bwd_bytes;
    return MPR_OK;
  });
}

int mpr_xattn_fwd(const void* q, const void* k, const void* v, const uint8_t* keep, int32_t dtype,
                  const int64_t* dims, const int64_t* strides, float scale, void* out, void* rest,
                  float* lse, void* ws, int64_t ws_bytes, void* stream) {
  return ops_call("xattn_fwd", [&]() -> int {
    MPR_TRY(xattn_check("xattn_fwd", dims, dtype));
    MPR_REQUIRE(strides && scale >= 0.f, "xattn_fwd: no strides, or a scale below 0");
    if (dims[0] * dims[3] == 0) return MPR_OK;
    MPR_REQUIRE(q && out && (dims[4] == 0 || (k && v)), "xattn_fwd: null pointer");
    const XPlan p = xattn_plan(dims, dtype, keep != nullptr);
    MPR_REQUIRE(p.fwd_bytes == 0 || (ws && ws_bytes >= p.fwd_bytes),
                "xattn_fwd: workspace of %lld bytes, %lld needed", (long long)ws_bytes,
                (long long)p.fwd_bytes);
    MPR_REQUIRE(p.few || dtype != MPR_F16, "xattn_fwd: float16 is for at most %d rows of a key head",
                FEW_ROWS);
    MPR_REQUIRE(p.few || dims[4] == 0 || (pieces_aligned(k, strides + 3, dtype) &&
                                          pieces_aligned(v, strides + 6, dtype)),
                "xattn_fwd: heads of k or v not at multiples of 4 bytes");
    XArgs a = xattn_args(q, k, v, keep, dims, strides, scale);
    a.out = out;
    a.rest = dtype == MPR_BF16 ? rest : nullptr;
    a.lse = lse;
    a.part = static_cast<float*>(ws);
    a.part_ms = reinterpret_cast<float*>(static_cast<char*>(ws) + p.part_ms);
    return by_dtype(dtype, [&](auto z) -> int {
      return xattn_forward<decltype(z)>(a, p, op_stream(stream));
    });
  });
}

int mpr_xattn_bwd(const void* q, const void* k, const void* v, const uint8_t* keep, int32_t dtype,
                  const int64_t* dims, const int64_t* strides, float scale, const void* out,
                  const void* rest, const float* lse, const void* dout, void* dq, void* dk, void* dv, void* ws,
                  int64_t ws_bytes, void* stream) {
  return ops_call("xattn_bwd", [&]() -> int {
    MPR_TRY(xattn_check("xattn_bwd", dims, dtype));
    MPR_REQUIRE(strides && scale >= 0.f, "xattn_bwd: no strides, or a scale below 0");
    if (dims[0] * (dims[3] + dims[4]) == 0) return MPR_OK;
    MPR_REQUIRE(dims[3] == 0 || (q && out && lse && dout), "xattn_bwd: null pointer");
    MPR_REQUIRE(dims[4] == 0 || (k && v), "xattn_bwd: null pointer");
    MPR_REQUIRE(!dk == !dv, "xattn_bwd: dk and dv are wanted together");
    const XPlan p = xattn_plan(dims, dtype);
    MPR_REQUIRE(p.bwd_bytes == 0 || (ws && ws_bytes >= p.bwd_bytes),
                "xattn_bwd: workspace of %lld bytes, %lld needed", (long long)ws_bytes,
                (long long)p.bwd_bytes);
    MPR_REQUIRE(dtype != MPR_F16, "xattn_bwd: float16 (compute in float32)");
    MPR_REQUIRE(dims[3] == 0 || dims[4] == 0 ||
                    (pieces_aligned(q, strides, dtype) && pieces_aligned(k, strides + 3, dtype) &&
                     pieces_aligned(v, strides + 6, dtype) &&
                     pieces_aligned(dout, strides + 10, dtype)),
                "xattn_bwd: heads not at multiples of 4 bytes");
    XArgs a = xattn_args(q, k, v, keep, dims, strides, scale);
    a.o = out;
    a.o_rest = dtype == MPR_BF16 ? rest : nullptr;
    a.lse = const_cast<float*>(lse);
    a.dout = dout;
    a.do_bs = strides[10]; a.do_ls = strides[11]; a.do_hs = strides[12];
    a.dq = dq; a.dk = dk; a.dv = dv;
    char* w = static_cast<char*>(ws);
    a.delta = reinterpret_cast<float*>(w + p.delta);
    a.part = reinterpret_cast<float*>(w + up256((int64_t)a.B * a.H * a.Lq * 4));
    a.part2 = reinterpret_cast<float*>(w + p.part2);
    return dtype == MPR_F32 ? xattn_backward<float>(a, p, op_stream(stream))
                            : xattn_backward<bf16>(a, p, op_stream(stream));
  });
}

}  // extern "C"
