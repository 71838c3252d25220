// A token per row of logits: temperature, top-k, top-p, min-p, and a choice by a given number.
//
// With m the row's largest logit and w_i = exp((x_i - m) / T), tokens are ranked by (x descending, index ascending).
//   top-k keeps ranks below k; top-p those whose lower ranks have at most p of the mass that top-k keeps (rank 0 always); min-p those
//   with w_i >= min_p. All three keep a prefix of the ranks, so what is kept is described by the last one: a (logit, index) pair.
//   The token is the first in index order whose kept mass, its predecessors' included, exceeds u times the whole kept mass.
// Masses are whole numbers, w_i * 2^45 rounded (64 bits), so sums do not depend on their order and atomics may add them: the same row
// always gives the same token, wherever it starts. exp is evaluated in 64 bits to 4e-11 (table of 2^(j / 16), degree 4), so a weight is off
// by that share of itself and 2^-46 of the largest (a token below that cannot be chosen), and only a border nearer than that to a sum may
// fall on its other side.
//
// A block, or a cluster of them, holds the row in shared memory; the logits are read once. A small k: the k-th largest of the threads' own
// largest is a logit that at least k tokens reach, so hardly more than k of them are gathered and the rest happens on that list. Else ranks
// are found without sorting: a histogram over 1024 steps of 1/32 in (m - x) / T brackets the last kept token - top-k exactly by counts,
// top-p by bounds on a bin's mass; one pass sums exact masses, bin by bin inside the bracket; the tokens of the one bin left are ranked
// against each other (up to 512 of them; more are counted in finer bins first, and equal ones in index order).
//
// 512 rows of 50400 bf16 logits: 107 us with top-p 0.9, 29 with top-k 40, 60 without either; one row of 50257: 12 us. Reading them takes 8 us;
// the rest is shared memory's atomics (the histogram: 6.5 a clock and SM) and the 64-bit exponentials of what may be kept. Two blocks an
// SM, so that one's waits are the other's work.
//
// Stands for the warper chain and multinomial draw of the reference's sample() (oslo/generation_utils.py:1364-1560), which sorts
// every row twice.
#include <math_constants.h>

#include "num.cuh"
#include "oslo_kernels.h"
#include "ptx.cuh"

namespace oslo {

struct SampleParams {
  const void* logits;
  const void* uniform;
  const float* temperature; const int* top_k; const float* top_p; const float* min_p;   // per row, or null: the numbers below
  long long* out;
  long long ld;
  double temperature1, top_p1, min_p1;
  int top_k1, V, slice, uniform64;
};

constexpr int SP_THREADS = 512, SP_WARPS = SP_THREADS / 32, SP_BINS = 1024, SP_LIST = 512;
constexpr float SP_STEP = 1.f / 32.f;       // bins' width in (m - x) / T: they reach 2^-46, and the last one holds only weights of 0
typedef unsigned long long u64;
#define SP_INLINE __attribute__((always_inline))      // what a lambda captures stays in registers
static_assert(SP_BINS == 2 * SP_THREADS, "a thread owns two bins");

struct SampleShared {
  double table[16];                         // 2^(j / 16): as many words as banks, so no two lanes meet in one
  union {
    u64 mass[SP_BINS];                      // bins' masses
    struct {
      u64 pair[SP_LIST];                    // a list of tokens: (logit's order, inverted index)
      u64 weight[SP_LIST];
    };
  };
  uint32_t count[SP_BINS];                  // bins' counts; before that the threads' largest logits
  u64 red[2][SP_WARPS];
  u64 xch[2][2];                            // what a block tells the others, two exchanges in turn
  u64 before;
  int found[4];
  uint32_t list_n;
};

__device__ __forceinline__ uint32_t sp_order(float x) {        // larger floats, larger numbers; -0 as 0
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float sp_value(uint32_t order) { return __uint_as_float(order ^ ((order >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ u64 sp_peer64(const void* p, int rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(map_to_cta(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t sp_peer32(const void* p, int rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_to_cta(smem_u32(p), rank)) : "memory");
  return v;
}
template <int C> __device__ __forceinline__ void sp_sync() {
  if (C == 1) __syncthreads();
  else cluster_sync_all();
}

// Every thread of the cluster gets f over all threads' values (f: a sum, a maximum, a minimum, with f(v, none) = v). `turn` alternates,
// so that a block that is ahead does not write what another still reads.
template <int C, typename F> __device__ __forceinline__ u64 sp_all(SampleShared& s, u64 v, u64 none, int& turn, F f) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, off));
  if (lane == 0) s.red[turn][warp] = v;
  __syncthreads();
  v = lane < SP_WARPS ? s.red[turn][lane] : none;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, off));
  if constexpr (C > 1) {
    if (threadIdx.x == 0) s.xch[turn][0] = v;
    cluster_sync_all();
    v = sp_peer64(&s.xch[turn][0], 0);
    for (int r = 1; r < C; ++r) v = f(v, sp_peer64(&s.xch[turn][0], r));
  }
  turn ^= 1;
  return v;
}
__device__ __forceinline__ u64 sp_add(u64 a, u64 b) { return a + b; }
__device__ __forceinline__ u64 sp_max(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 sp_min(u64 a, u64 b) { return a < b ? a : b; }
// Sum of the values of this block's threads ahead of this one; `total`: of all of them
template <typename V> __device__ __forceinline__ V sp_scan(SampleShared& s, V v, V& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  V* red = reinterpret_cast<V*>(s.red[0]);
  V sum = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const V o = __shfl_up_sync(0xffffffffu, sum, off);
    if (lane >= off) sum += o;
  }
  __syncthreads();                          // s.red may still be read
  if (lane == 31) red[warp] = sum;
  __syncthreads();
  V part = lane < SP_WARPS ? red[lane] : V(0), upto = part;
#pragma unroll
  for (int off = 1; off < SP_WARPS; off <<= 1) {
    const V o = __shfl_up_sync(0xffffffffu, upto, off);
    if (lane >= off) upto += o;
  }
  total = __shfl_sync(0xffffffffu, upto, SP_WARPS - 1);
  const V ahead = __shfl_sync(0xffffffffu, upto - part, warp);
  __syncthreads();
  return ahead + sum - v;
}

__device__ __forceinline__ float sp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A 16-byte piece of logits: its values, and a running maximum that a value that is no number spoils
template <typename T> struct Piece;
template <> struct Piece<float> {
  static constexpr int N = 4;
  typedef float Top;
  static __device__ __forceinline__ Top none() { return -CUDART_INF_F; }
  static __device__ __forceinline__ float larger(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
  }
  static __device__ __forceinline__ Top top(const uint4& p, Top t) {
    return larger(larger(t, larger(__uint_as_float(p.x), __uint_as_float(p.y))), larger(__uint_as_float(p.z), __uint_as_float(p.w)));
  }
  static __device__ __forceinline__ float value(Top t) { return t; }
  static __device__ __forceinline__ void get(const uint4& p, float (&v)[4]) {
    v[0] = __uint_as_float(p.x); v[1] = __uint_as_float(p.y); v[2] = __uint_as_float(p.z); v[3] = __uint_as_float(p.w);
  }
};
template <> struct Piece<__nv_bfloat16> {
  static constexpr int N = 8;
  typedef __nv_bfloat162 Top;
  static __device__ __forceinline__ Top none() { return __halves2bfloat162(__ushort_as_bfloat16(0xff80), __ushort_as_bfloat16(0xff80)); }
  static __device__ __forceinline__ Top two(const uint32_t& w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
  static __device__ __forceinline__ Top top(const uint4& p, Top t) {
    return __hmax2_nan(__hmax2_nan(t, __hmax2_nan(two(p.x), two(p.y))), __hmax2_nan(two(p.z), two(p.w)));
  }
  static __device__ __forceinline__ float value(Top t) { return __bfloat162float(__hmax_nan(t.x, t.y)); }
  static __device__ __forceinline__ void get(const uint4& p, float (&v)[8]) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
};
template <> struct Piece<__half> {
  static constexpr int N = 8;
  typedef __half2 Top;
  static __device__ __forceinline__ Top none() { return __halves2half2(__ushort_as_half(0xfc00), __ushort_as_half(0xfc00)); }
  static __device__ __forceinline__ Top two(const uint32_t& w) { return *reinterpret_cast<const __half2*>(&w); }
  static __device__ __forceinline__ Top top(const uint4& p, Top t) {
    return __hmax2_nan(__hmax2_nan(t, __hmax2_nan(two(p.x), two(p.y))), __hmax2_nan(two(p.z), two(p.w)));
  }
  static __device__ __forceinline__ float value(Top t) { return __half2float(__hmax_nan(__low2half(t), __high2half(t))); }
  static __device__ __forceinline__ void get(const uint4& p, float (&v)[8]) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = t.x; v[2 * i + 1] = t.y;
    }
  }
};
template <typename T> __device__ __forceinline__ T sp_lowest();      // minus infinity
template <> __device__ __forceinline__ float sp_lowest<float>() { return -CUDART_INF_F; }
template <> __device__ __forceinline__ __nv_bfloat16 sp_lowest<__nv_bfloat16>() { return __ushort_as_bfloat16(0xff80); }
template <> __device__ __forceinline__ __half sp_lowest<__half>() { return __ushort_as_half(0xfc00); }

template <typename T, int C>
__global__ void __launch_bounds__(SP_THREADS, 2) sample_kernel(const SampleParams p) {
  constexpr int PER = Piece<T>::N;
  extern __shared__ __align__(16) unsigned char sp_raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(sp_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % C, row = blockIdx.x / C;
  const int i0 = min(p.V, rank * p.slice), n = min(p.V, i0 + p.slice) - i0;   // this block's tokens
  const T* src = static_cast<const T*>(p.logits) + row * p.ld + i0;
  // Shared memory holds the row's own 16-byte pieces: `pad` places ahead of the first token and some behind the last one are minus
  // infinity. A warp's pieces lie one behind another.
  const int pad = static_cast<int>(reinterpret_cast<uintptr_t>(src) & 15) / static_cast<int>(sizeof(T));
  const int pieces = n > 0 ? (pad + n + PER - 1) / PER : 0, per_warp = (pieces + SP_WARPS - 1) / SP_WARPS;
  T* y = reinterpret_cast<T*>(sp_raw + (sizeof(SampleShared) + 15) / 16 * 16);
  for (int j = tid; j < pieces; j += SP_THREADS) {
    const int e = j * PER - pad;
    if (e >= 0 && e + PER <= n) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(y + j * PER)), "l"(src + e) : "memory");
    } else {
#pragma unroll
      for (int c = 0; c < PER; ++c) y[j * PER + c] = e + c >= 0 && e + c < n ? src[e + c] : sp_lowest<T>();
    }
  }
  const double temperature = p.temperature ? p.temperature[row] : p.temperature1, top_p = p.top_p ? p.top_p[row] : p.top_p1;
  const double min_p = p.min_p ? p.min_p[row] : p.min_p1;
  const int top_k = p.top_k ? p.top_k[row] : p.top_k1;
  const double u = p.uniform64 ? static_cast<const double*>(p.uniform)[row] : static_cast<double>(static_cast<const float*>(p.uniform)[row]);
  if (tid < 16) s.table[tid] = exp2(tid * (1.0 / 16.0));
  if (tid == 0) s.list_n = 0;
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();

  // f(value, place) for this thread's tokens; a token's place is its index in the block's part plus `pad`
  const int j0 = warp * per_warp, j1 = min(pieces, j0 + per_warp);
  auto each = [&](auto f) SP_INLINE {
    for (int j = j0 + lane; j < j1; j += 32) {
      float v[PER];
      Piece<T>::get(*reinterpret_cast<const uint4*>(y + j * PER), v);
#pragma unroll
      for (int c = 0; c < PER; ++c) f(v[c], j * PER + c);
    }
  };
  auto value = [&](int place) { return Num<T>::to(y[place]); };
  const int first = i0 - pad;                                   // a token's index is its place plus this

  // ---- the largest logit; one that is no number spoils the row
  int turn = 0;
  float mine_top;
  {
    auto t = Piece<T>::none();
    for (int j = j0 + lane; j < j1; j += 32) t = Piece<T>::top(*reinterpret_cast<const uint4*>(y + j * PER), t);
    mine_top = Piece<T>::value(t);
  }
  const u64 top = sp_all<C>(s, mine_top != mine_top ? ~0ull : static_cast<u64>(sp_order(mine_top)), 0, turn, sp_max);
  float m = sp_value(static_cast<uint32_t>(top));
  if (top == ~0ull || m == -CUDART_INF_F || !(u >= 0.0 && u < 1.0)) {         // the same for the whole cluster
    if (rank == 0 && tid == 0) p.out[row] = -1;
    sp_sync<C>();                                               // nobody leaves while another reads its shared memory
    return;
  }
  if (!(temperature > 0.0) || top_k == 1 || !(top_p > 0.0) || min_p != min_p) {      // the first of the largest
    u64 best = ~0ull;
    each([&](float v, int at) {
      if (v == m) best = sp_min(best, first + at);
    });
    best = sp_all<C>(s, best, ~0ull, turn, sp_min);
    if (rank == 0 && tid == 0) p.out[row] = static_cast<long long>(best);
    sp_sync<C>();
    return;
  }
  if (m == CUDART_INF_F) {                                      // infinities share everything: 0, and minus infinity elsewhere
    for (int j = tid; j < pieces * PER; j += SP_THREADS) y[j] = value(j) == m ? Num<T>::from(0.f) : sp_lowest<T>();
    m = 0.f;
    mine_top = mine_top == CUDART_INF_F ? 0.f : -CUDART_INF_F;
    __syncthreads();
  }

  // what lies outside these is as good as they are, and nothing below overflows
  const double limited = fmin(fmax(temperature, 1e-30), 1e30);
  if (fabs(static_cast<double>(m)) > 1e6 * limited) {
    // 32-bit steps at m may be wider than any weight reaches (below, the least logit that has one is a 32-bit number), and m the lowest value
    // there is, which masks write. Differences from m stand for such logits: exact up to half of m or twice it, and of no weight beyond
    for (int j = tid; j < pieces * PER; j += SP_THREADS) y[j] = Num<T>::from(value(j) - m);
    mine_top = Num<T>::to(Num<T>::from(mine_top - m));
    m = 0.f;
    __syncthreads();
  }
  const double inv_t = 1.0 / limited, md = static_cast<double>(m), steps = inv_t * 23.083120654223414;             // 16 / ln 2
  const float per_bin = static_cast<float>(inv_t / SP_STEP), share = static_cast<float>(top_p);
  const float least_v = __double2float_rd(fmax(md - 32.0 * limited, -3.0e38));
  auto depth = [&](float v) { return (m - v) * per_bin; };      // bin `b` is [b, b + 1)
  // w 2^45 as a whole number: 0 from 32 T below the largest on (2^45 exp(-32) < 1 / 2)
  auto weight = [&](float v) SP_INLINE -> u64 {
    const double d = static_cast<double>(fmaxf(v, least_v)) - md;
    const double z = fma(d, steps, 6755399441055744.0);         // rounded by adding 1.5 * 2^52
    const int k = __double2loint(z);
    const double r = fma(d, steps, -(z - 6755399441055744.0));  // in 16ths of an octave, at most a half
    // exp(r ln 2 / 16) to (0.0217)^5 / 120
    const double e = fma(fma(fma(fma(r, 1.4676100322919429e-07, 1.3550807779497455e-05), r, 0.00093838479280898709), r, 0.04332169878499658), r, 1.0);
    const double b = s.table[k & 15];
    const double scaled = __hiloint2double(__double2hiint(b) + (((k >> 4) + 45) << 20), __double2loint(b));
    return __double_as_longlong(fma(scaled, e, 4503599627370496.0)) & 0xfffffffffffffull;
  };
  // f(value, weight, place) for this thread's tokens from `bar` to `roof` (and others, should that be easier), 32 tokens of it at a time.
  // Few of them: a lane takes two at once, one pair after another while any lane of its warp has some; many (over half of some lane's; 12 and
  // 24 of 32 do as well): four of a piece at once. 512 rows of 50400 bf16 logits, top-p 0.9: 7 us less than where lanes meet after every
  // piece; with no filter, where all are weighed, 2 us more.
  constexpr int BATCH = 32 / PER;                               // pieces
  auto weigh = [&](float bar, float roof, auto f) SP_INLINE {
    for (int jb = j0 + lane; jb - lane < j1; jb += 32 * BATCH) {
      uint32_t mask = 0;
#pragma unroll
      for (int q = 0; q < BATCH; ++q) {
        const int j = jb + 32 * q;
        if (j >= j1) continue;
        float v[PER];
        Piece<T>::get(*reinterpret_cast<const uint4*>(y + j * PER), v);
#pragma unroll
        for (int c = 0; c < PER; ++c) mask |= v[c] >= bar && v[c] <= roof ? 1u << (q * PER + c) : 0u;
      }
      if (__any_sync(0xffffffffu, __popc(mask) > 16)) {
#pragma unroll 1
        for (int q = 0; q < BATCH; ++q) {
          const int j = jb + 32 * q;
          if (j >= j1) break;
          float v[PER];
          Piece<T>::get(*reinterpret_cast<const uint4*>(y + j * PER), v);
#pragma unroll
          for (int g = 0; g < PER; g += 4) {
            u64 w[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) w[c] = weight(v[g + c]);
#pragma unroll
            for (int c = 0; c < 4; ++c) f(v[g + c], w[c], j * PER + g + c);
          }
        }
      } else {
        while (mask) {
          const int b0 = __ffs(mask) - 1;
          mask &= mask - 1;
          const int b1 = mask ? __ffs(mask) - 1 : b0;
          const bool two = mask != 0;
          mask &= mask - 1;
          const int at0 = (jb + b0 / PER * 32) * PER + b0 % PER, at1 = (jb + b1 / PER * 32) * PER + b1 % PER;
          const float x0 = value(at0), x1 = value(at1);
          const u64 w0 = weight(x0), w1 = weight(x1);
          f(x0, w0, at0);
          if (two) f(x1, w1, at1);
        }
      }
    }
  };
  // a logit that no token of a depth below `d` is under, and one that none of at least that depth exceeds
  auto bar_of = [&](float d) { return m - (d + 0.02f) / per_bin * 1.000001f; };
  auto roof_of = [&](float d) { return m - fmaxf(d - 0.02f, 0.f) / per_bin * 0.999999f; };
  // min-p in the same units; the largest always stays
  const u64 w_min = min_p > 0.0 ? static_cast<u64>(ceil(fmin(min_p, 1.0) * 35184372088832.0)) : 0ull;

  const bool by_k = top_k > 1 && top_k < p.V, by_p = top_p < 1.0;
  // The list in rank order, one token a thread (0 behind the last): a bitonic sort, in the warps where the distance allows it
  auto sorted = [&](uint32_t all) SP_INLINE -> u64 {
    u64 me = tid < all ? s.pair[tid] : 0ull;
    for (uint32_t k = 2; k < 2 * all; k *= 2) {
      for (uint32_t d = k / 2; d > 0; d /= 2) {
        u64 other;
        if (d >= 32) {
          __syncthreads();
          s.pair[tid] = me;
          __syncthreads();
          other = s.pair[tid ^ d];
        } else {
          other = __shfl_xor_sync(0xffffffffu, me, d);
        }
        const bool larger = ((tid & d) == 0) == ((tid & k) == 0);             // of the two, this thread keeps the larger
        me = (other > me) == larger ? other : me;
      }
    }
    __syncthreads();
    s.pair[tid] = me;
    __syncthreads();
    return me;
  };
  // The blocks' lists become one, in every block (`mine`: it is needed here); other blocks' tokens behind this block's own
  auto gather = [&](bool here) SP_INLINE -> uint32_t {
    sp_sync<C>();
    uint32_t all = s.list_n;
    if constexpr (C > 1) {
      if (here) {
        for (int d = 1; d < C; ++d) {
          const int r = (rank + d) % C;
          const uint32_t theirs = sp_peer32(&s.list_n, r);
          for (uint32_t i = tid; i < theirs && all + i < SP_LIST; i += SP_THREADS) s.pair[all + i] = sp_peer64(&s.pair[i], r);
          all += theirs;
        }
      }
    }
    return all;
  };
  auto note = [&](float v, int at) SP_INLINE {                            // one more token for the list, if there is room
    const uint32_t slot = atomicAdd(&s.list_n, 1u);
    if (slot < SP_LIST) s.pair[slot] = static_cast<u64>(sp_order(v)) << 32 | (0xffffffffu - static_cast<uint32_t>(first + at));
  };

  // ---- a small k: everything happens on a list
  if (by_k && top_k <= SP_LIST / 2) {
    // The k-th largest of `groups` largest: at least k tokens reach it. Of a block with fewer tokens than k, all are taken.
    const int lanes = top_k <= 64 ? 4 : 1, groups = SP_THREADS / lanes;
    float* tops = reinterpret_cast<float*>(s.count);
    float g = mine_top;
    if (lanes == 4) {
      g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 1));
      g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 2));
    }
    if (tid % lanes == 0) tops[tid / lanes] = g;
    if (tid == 0) s.found[0] = 0;
    __syncthreads();
    if (tid < groups) {
      const float v = tops[tid];
      int over = 0, same = 0;
#pragma unroll 8
      for (int j = 0; j < groups; j += 4) {
        const float4 o = *reinterpret_cast<const float4*>(tops + j);
        over += (o.x > v) + (o.y > v) + (o.z > v) + (o.w > v);
        same += (o.x == v) + (o.y == v) + (o.z == v) + (o.w == v);
      }
      if (over < top_k && top_k <= over + same) s.found[0] = static_cast<int>(sp_order(v));      // all that write it write the same
    }
    __syncthreads();
    const uint32_t bar = static_cast<uint32_t>(sp_all<C>(s, static_cast<uint32_t>(s.found[0]), 0, turn, sp_max));
    const float least = sp_value(bar);
    each([&](float v, int at) {
      if (v >= least && v > -CUDART_INF_F) note(v, at);
    });
    uint32_t all = gather(rank == 0);
    if constexpr (C > 1) {
      if (rank == 0 && tid == 0) s.found[1] = static_cast<int>(all);
      if (rank != 0) all = 0;
      cluster_sync_all();                                       // the others' lists have been read
      if (rank != 0) all = sp_peer32(&s.found[1], 0);
    }
    if (all <= SP_LIST) {
      if (rank == 0) {
        __syncthreads();
        const u64 pair = sorted(all);
        const bool in_k = tid < all && tid < top_k;
        const u64 w = in_k ? weight(sp_value(static_cast<uint32_t>(pair >> 32))) : 0ull;
        u64 total, ahead_w = sp_scan<u64>(s, w, total);
        const u64 most = by_p ? static_cast<u64>(top_p * static_cast<double>(total)) : ~0ull;
        const u64 kept = in_k && (tid == 0 || (ahead_w <= most && w >= w_min)) ? w : 0ull;
        s.weight[tid] = kept;
        u64 whole;
        sp_scan<u64>(s, kept, whole);
        const uint32_t kept_n = __syncthreads_count(kept != 0);               // they begin the list
        // a sum of 2^45 each of 512 tokens has no more than 54 bits: u times it may round up to it
        const u64 reach = sp_min(static_cast<u64>(u * static_cast<double>(whole)), whole - 1);
        if (kept) {
          const uint32_t index = 0xffffffffu - static_cast<uint32_t>(pair);
          u64 ahead = 0;
#pragma unroll 8
          for (uint32_t j = 0; j < kept_n; ++j) {
            const u64 weight_j = s.weight[j];
            ahead += static_cast<uint32_t>(s.pair[j]) > static_cast<uint32_t>(pair) ? weight_j : 0ull;       // a smaller index
          }
          if (ahead <= reach && reach < ahead + kept) p.out[row] = index;
        }
      }
      sp_sync<C>();
      return;
    }
    sp_sync<C>();                                               // too many equal ones: the general way
    if (tid == 0) s.list_n = 0;
    __syncthreads();
  }

  uint32_t tau_key = 0, tau_idx = 0xffffffffu;                  // kept: larger logits, and equal ones up to this index
  auto within = [&](float v, int at) {
    const uint32_t key = sp_order(v);
    return key > tau_key || (key == tau_key && static_cast<uint32_t>(first + at) <= tau_idx);
  };
  // Among tokens with masses f(value, place), this thread's summing up to `sum`: the index of the first one, in index order, whose mass
  // and its predecessors' exceed goal(whole). -1: none.
  auto pick = [&](u64 sum, auto goal_of, auto f) SP_INLINE -> long long {
    u64 mine, ahead = sp_scan<u64>(s, sum, mine), all = mine;
    if constexpr (C > 1) {
      if (tid == 0) s.xch[turn][1] = mine;
      cluster_sync_all();
      all = 0;
      for (int r = 0; r < C; ++r) {
        if (r == rank) ahead += all;
        all += sp_peer64(&s.xch[turn][1], r);
      }
    }
    const u64 goal = goal_of(all);
    // the warp whose tokens reach it: lanes' shares are interleaved, so a whole warp's are looked at
    const u64 w0 = __shfl_sync(0xffffffffu, ahead, 0), w1 = __shfl_sync(0xffffffffu, ahead + sum, 31);
    if (lane == 0 && w0 <= goal && goal < w1) {
      s.found[0] = warp;
      s.before = goal - w0;
    }
    const bool here = __syncthreads_or(lane == 0 && w0 <= goal && goal < w1);
    u64 at = ~0ull;
    if (here) {
      const int a0 = s.found[0] * per_warp * PER, a1 = min(pieces, (s.found[0] + 1) * per_warp) * PER;
      u64 left = s.before;
      for (int base = a0; base < a1; base += 8 * SP_THREADS) {      // eight tokens a thread at a time, one behind another
        u64 w[8], part = 0, whole;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const int i = base + tid * 8 + c;
          w[c] = f(i < a1 ? value(i) : -CUDART_INF_F, i);
          part += w[c];
        }
        u64 sofar = sp_scan<u64>(s, part, whole);
        if (sofar <= left && left < sofar + part) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            sofar += w[c];
            if (sofar > left) at = sp_min(at, static_cast<u64>(first + base + tid * 8 + c));
          }
        }
        if (left < whole) break;                                    // the same for all threads
        left -= whole;
      }
    }
    return static_cast<long long>(sp_all<C>(s, at, ~0ull, turn, sp_min));
  };

  // Moves tau to the last token of bin `b` (whose `size` tokens within tau begin a rank order) whose predecessors in the bin number
  // fewer than `room`, or have a mass of at most `room`. All threads of the cluster call it with the same arguments.
  auto resolve = [&](int b, uint32_t size, u64 room, bool by_mass) SP_INLINE {
    uint32_t key_lo = 0, key_hi = 0xffffffffu;
    const float d0 = b, d1 = b + 1;
    auto member = [&](float v, int at) SP_INLINE {
      const float d = depth(v);
      if (!(d >= d0 && d < d1)) return false;
      const uint32_t key = sp_order(v);
      return key >= key_lo && key <= key_hi && within(v, at);
    };
    while (size > SP_LIST) {
      u64 lo = ~0ull, hi = 0;
      each([&](float v, int at) {
        if (member(v, at)) {
          lo = sp_min(lo, sp_order(v));
          hi = sp_max(hi, sp_order(v));
        }
      });
      lo = sp_all<C>(s, lo, ~0ull, turn, sp_min);
      hi = sp_all<C>(s, hi, 0, turn, sp_max);
      key_lo = static_cast<uint32_t>(lo);
      key_hi = static_cast<uint32_t>(hi);
      if (key_lo == key_hi) {                                   // equal logits: the first `q` of them in index order
        u64 q = by_mass ? room / sp_max(1, weight(sp_value(key_lo))) + 1 : room;
        if (q >= size) q = size;
        auto one = [&](float v, int at) -> u64 { return member(v, at); };
        u64 mine = 0;
        each([&](float v, int at) { mine += one(v, at); });
        tau_idx = static_cast<uint32_t>(pick(mine, [&](u64) { return q - 1; }, one));
        tau_key = key_lo;
        return;
      }
      // finer bins over the logits that are there
      const int shift = max(0, 32 - __clz(key_hi - key_lo) - 10);             // 1024 of them
      sp_sync<C>();
      for (int i = tid; i < SP_BINS; i += SP_THREADS) {
        s.count[i] = 0;
        s.mass[i] = 0;
      }
      __syncthreads();
      each([&](float v, int at) {
        if (!member(v, at)) return;
        const uint32_t fine = (key_hi - sp_order(v)) >> shift;
        atomicAdd(&s.count[fine], 1u);
        if (by_mass) atomicAdd(&s.mass[fine], weight(v));
      });
      sp_sync<C>();
      uint32_t cnt[2] = {0, 0};
      u64 add[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        for (int r = 0; r < C; ++r) {
          cnt[j] += C == 1 ? s.count[2 * tid + j] : sp_peer32(&s.count[2 * tid + j], r);
          if (by_mass) add[j] += C == 1 ? s.mass[2 * tid + j] : sp_peer64(&s.mass[2 * tid + j], r);
        }
        if (!by_mass) add[j] = cnt[j];
      }
      u64 all, ahead = sp_scan<u64>(s, add[0] + add[1], all);
      if (tid == 0) s.found[0] = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 2; ++j) {                             // the last bin that has a kept token
        const u64 before = ahead + (j ? add[0] : 0);
        if (cnt[j] && (by_mass ? before <= room : before < room)) atomicMax(&s.found[0], 2 * tid + j);
      }
      __syncthreads();
      const int at = s.found[0];
      if (at >> 1 == tid) {
        s.before = ahead + (at & 1 ? add[0] : 0);
        s.found[1] = static_cast<int>(at & 1 ? cnt[1] : cnt[0]);
      }
      __syncthreads();
      room -= s.before;
      size = static_cast<uint32_t>(s.found[1]);
      const uint32_t near = static_cast<uint32_t>(at) << shift, far = near + ((1u << shift) - 1u);
      if (far < key_hi - key_lo) key_lo = key_hi - far;
      key_hi -= near;
      __syncthreads();
    }
    // ---- few enough to be ranked against each other
    sp_sync<C>();                                               // the bins' masses have been read
    if (tid == 0) s.list_n = 0;
    __syncthreads();
    each([&](float v, int at) {
      if (member(v, at)) note(v, at);
    });
    const uint32_t all = gather(true);
    sp_sync<C>();                                               // and the others have read this block's part
    const u64 pair = sorted(all);
    u64 whole, ahead = sp_scan<u64>(s, tid >= all ? 0ull : by_mass ? weight(sp_value(static_cast<uint32_t>(pair >> 32))) : 1ull, whole);
    u64 last = tid < all && (by_mass ? ahead <= room : ahead < room) ? pair : ~0ull;          // the last kept one is the smallest pair
    last = sp_all<1>(s, last, ~0ull, turn, sp_min);
    tau_key = static_cast<uint32_t>(last >> 32);
    tau_idx = 0xffffffffu - static_cast<uint32_t>(last);
  };

  // what is kept of a thread's tokens ahead of depth `from`, already summed; the last bin's weights are 0
  u64 kept = 0, mass = 0;
  float from = 0.f, to = SP_BINS - 1;
  if (by_k || by_p) {
    for (int i = tid; i < SP_BINS; i += SP_THREADS) s.count[i] = 0;
    __syncthreads();
    // top-p's whole in the same pass: its 64-bit exponentials run while the histogram's atomics wait (512 rows of 50400, top-p 0.9: 107 us.
    // 32-bit ones take 88, but are off by 2^-21, which moves the last token kept in some rows of a hundred; a bound on that error, and the rest
    // of the row weighed only where the border is nearer, 102 to 106, and 250 instead of 220 at a temperature of 2)
    const bool weighed = by_p && !by_k;
    for (int j = j0 + lane; j < j1; j += 32) {
      float v[PER];
      Piece<T>::get(*reinterpret_cast<const uint4*>(y + j * PER), v);
#pragma unroll
      for (int c = 0; c < PER; ++c) {
        const float d = depth(v[c]);
        if (d < SP_BINS - 1) atomicAdd(&s.count[static_cast<int>(d)], 1u);
      }
      if (weighed) {
#pragma unroll
        for (int c = 0; c < PER; ++c) mass += weight(v[c]);
      }
    }
    sp_sync<C>();
    uint32_t cnt[2] = {0, 0};                                   // of bins 2 tid and 2 tid + 1
#pragma unroll
    for (int j = 0; j < 2; ++j)
      for (int r = 0; r < C; ++r) cnt[j] += C == 1 ? s.count[2 * tid + j] : sp_peer32(&s.count[2 * tid + j], r);
    if (by_k) {
      uint32_t all, ahead = sp_scan<uint32_t>(s, cnt[0] + cnt[1], all);
      if (all > static_cast<uint32_t>(top_k)) {                 // else it keeps every token that has a weight
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t before = ahead + (j ? cnt[0] : 0);
          if (before < static_cast<uint32_t>(top_k) && static_cast<uint32_t>(top_k) <= before + cnt[j]) {
            s.found[0] = 2 * tid + j;
            s.found[1] = static_cast<int>(cnt[j]);
            s.found[2] = static_cast<int>(top_k - before);
          }
        }
        __syncthreads();
        const int b = s.found[0], size = s.found[1], room = s.found[2];
        __syncthreads();
        resolve(b, size, room, false);
#pragma unroll
        for (int j = 0; j < 2; ++j) cnt[j] = 2 * tid + j < b ? cnt[j] : (2 * tid + j == b ? room : 0);
        to = b + 1;
      }
    }
    if (by_p) {
      const float last = to - 1.f;
      auto in_k = [&](float v, float d, int at) { return d < to && !(d >= last && !within(v, at)); };
      if (by_k) {                                               // the mass of what top-k keeps
        mass = 0;
        weigh(bar_of(to), m, [&](float v, u64 w, int at) { mass += in_k(v, depth(v), at) ? w : 0ull; });
      }
      mass = sp_all<C>(s, mass, 0, turn, sp_add);
      const u64 most = static_cast<u64>(top_p * static_cast<double>(mass));
      // Which bins may hold the last kept token: first by counts times the weight in the middle of a bin, give or take 0.2% of the mass
      // if that is few enough tokens for a list, else 1%; should that not hold, by certain bounds: exp(-(b + 1) / 32) to exp(-b / 32) a
      // token, a little wider than rounding makes them
      for (int attempt = 0;; ++attempt) {
        float lo[2], hi[2], lo_all, hi_all;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float e = cnt[j] * sp_exp2(-(2 * tid + j) * (SP_STEP * 1.44269504f));
          lo[j] = e * (attempt == 2 ? 0.9690f : 0.98450f);      // exp(-1 / 32) = 0.96923, exp(-1 / 64) = 0.98450
          hi[j] = e * (attempt == 2 ? 1.0002f : 0.98450f);
        }
        const float lo_ahead = sp_scan<float>(s, lo[0] + lo[1], lo_all), hi_ahead = sp_scan<float>(s, hi[0] + hi[1], hi_all);
        const float give = attempt ? 0.01f : 0.002f;
        const float under = attempt == 2 ? share * lo_all * 0.9998f : (share - give) * lo_all;
        const float above = attempt == 2 ? share * hi_all * 1.0002f : (share + give) * hi_all;
        if (tid == 0) { s.found[0] = 0; s.found[1] = 0; }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (!cnt[j]) continue;
          if (hi_ahead + (j ? hi[0] : 0.f) <= under) atomicMax(&s.found[0], 2 * tid + j);       // kept
          if (lo_ahead + (j ? lo[0] : 0.f) <= above) atomicMax(&s.found[1], 2 * tid + j);       // perhaps
        }
        sp_sync<C>();                                           // `mass` may have been a list that others read
        const int b_lo = s.found[0], b_hi = s.found[1];
        for (int i = tid; i < SP_BINS; i += SP_THREADS) s.mass[i] = 0;
        __syncthreads();
        // ---- exact masses: ahead of the bracket, and bin by bin inside it
        from = b_lo;
        const float border = b_hi + 1;
        u64 head = 0;
        kept = 0;
        if (attempt == 0) {
          uint32_t some = 0;
#pragma unroll
          for (int j = 0; j < 2; ++j) some += 2 * tid + j >= b_lo && 2 * tid + j <= b_hi ? cnt[j] : 0u;
          uint32_t listed;
          sp_scan<uint32_t>(s, some, listed);
          if (by_k || listed > SP_LIST) continue;
          if (tid == 0) s.list_n = 0;
          __syncthreads();
          weigh(bar_of(border), m, [&](float v, u64 w, int at) {
            const float d = depth(v);
            if (d < from) {
              head += w;
              kept += w >= w_min ? w : 0ull;
            } else if (d < border) {
              note(v, at);
            }
          });
          head = sp_all<C>(s, head, 0, turn, sp_add);
          const uint32_t all = gather(true);
          sp_sync<C>();                                         // the others have read this block's part
          const u64 pair = sorted(all), w = tid < all ? weight(sp_value(static_cast<uint32_t>(pair >> 32))) : 0ull;
          u64 inside, ahead = head + sp_scan<u64>(s, w, inside);
          if (!(head <= most && (head + inside > most || b_hi >= to - 1.f || head + inside >= mass))) continue;
          s.weight[tid] = w;
          const u64 end = sp_all<1>(s, tid < all && ahead <= most ? pair : ~0ull, ~0ull, turn, sp_min);
          tau_key = static_cast<uint32_t>(end >> 32);
          tau_idx = 0xffffffffu - static_cast<uint32_t>(end);
          // each warp's share of what the list keeps of this block's tokens; places ahead of the first token and behind the last one
          // are the neighbours' tokens, which count there
          const int a0 = max(j0 * PER, pad), a1 = min(j1 * PER, pad + n);
          for (uint32_t i = lane; i < all; i += 32) {
            const int at = static_cast<int>(0xffffffffu - static_cast<uint32_t>(s.pair[i])) - first;
            if (at >= a0 && at < a1 && s.pair[i] >= end && s.weight[i] >= w_min) kept += s.weight[i];
          }
          to = floorf(depth(sp_value(tau_key))) + 1.f;
          from = SP_BINS;                                       // all summed
          break;
        }
        if (by_k) {
          weigh(bar_of(fminf(border, to)), m, [&](float v, u64 w, int at) {
            const float d = depth(v);
            if (!in_k(v, d, at)) return;
            if (d < from) {
              head += w;
              kept += w >= w_min ? w : 0ull;
            } else if (d < border) {
              atomicAdd(&s.mass[static_cast<int>(d)], w);
            }
          });
        } else {
          weigh(bar_of(border), m, [&](float v, u64 w, int) {
            const float d = depth(v);
            if (d < from) {
              head += w;
              kept += w >= w_min ? w : 0ull;
            } else if (d < border) {
              atomicAdd(&s.mass[static_cast<int>(d)], w);
            }
          });
        }
        head = sp_all<C>(s, head, 0, turn, sp_add);
        u64 add[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (2 * tid + j >= b_lo && 2 * tid + j <= b_hi)
            for (int r = 0; r < C; ++r) add[j] += C == 1 ? s.mass[2 * tid + j] : sp_peer64(&s.mass[2 * tid + j], r);
        u64 inside, ahead = sp_scan<u64>(s, add[0] + add[1], inside);
        ahead += head;
        // its first token is kept, and what follows its last one is not (or nothing of any weight does)
        if (attempt == 1 && !(head <= most && (head + inside > most || b_hi >= to - 1.f || head + inside >= mass))) continue;
        if (tid == 0) s.found[2] = b_lo;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int b = 2 * tid + j;
          if (cnt[j] && b >= b_lo && b <= b_hi && ahead + (j ? add[0] : 0) <= most) atomicMax(&s.found[2], b);
        }
        __syncthreads();
        const int b = s.found[2];
        if (b >> 1 == tid) {
          s.before = ahead + (b & 1 ? add[0] : 0);
          s.found[3] = static_cast<int>(b & 1 ? cnt[1] : cnt[0]);
        }
        __syncthreads();
        const u64 before = s.before;
        const int size = s.found[3];
        __syncthreads();
        resolve(b, size, most >= before ? most - before : 0ull, true);
        to = b + 1;
        break;
      }
    }
  }

  // ---- the kept mass in index order, and where the given share of it is reached
  auto keeps = [&](float v, int at) SP_INLINE -> u64 {
    const float d = depth(v);
    if (!(d < to) || (d >= to - 1.f && !within(v, at))) return 0;
    const u64 w = weight(v);
    return w >= w_min ? w : 0ull;
  };
  if (!by_k && !by_p) {
    // what min-p cuts off (a little less): exp(-d / 32) < min-p
    const float low = min_p > 0.0 ? fminf(static_cast<float>(-32.0 * log(fmin(min_p, 1.0))) + 1.f, SP_BINS - 1) : SP_BINS - 1;
    weigh(bar_of(low), m, [&](float, u64 w, int) { kept += w >= w_min ? w : 0ull; });
  } else if (from < SP_BINS) {
    weigh(bar_of(to), roof_of(from), [&](float v, u64 w, int at) {
      const float d = depth(v);
      if (d >= from && d < to && !(d >= to - 1.f && !within(v, at)) && w >= w_min) kept += w;
    });
  }
  // u < 1, but u times a mass of more than 53 bits may round up to the mass
  const long long token = pick(kept, [&](u64 all) { return sp_min(static_cast<u64>(u * static_cast<double>(all)), all - 1); }, keeps);
  if (rank == 0 && tid == 0) p.out[row] = token;
  sp_sync<C>();                                                 // nobody leaves while another reads its shared memory
}

template <typename T, int C>
static int sample_launch(const SampleParams& p, int rows, cudaStream_t stream) {
  auto kernel = sample_kernel<T, C>;
  const size_t smem = (sizeof(SampleShared) + 15) / 16 * 16 + static_cast<size_t>(p.slice) * sizeof(T) + 32;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  static unsigned long long ready = 0;                          // one bit per device
  if (dev > 63 || !((__atomic_load_n(&ready, __ATOMIC_ACQUIRE) >> dev) & 1)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev <= 63) __atomic_fetch_or(&ready, 1ull << dev, __ATOMIC_RELEASE);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * C);
  cfg.blockDim = dim3(SP_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kernel, p);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}
template <typename T>
static int sample_any(SampleParams& p, int rows, int num_sms, cudaStream_t stream) {
  // A block takes up to 100 KB of a row, so that an SM holds two; with fewer rows than SMs, several blocks share a row
  // (parts of 8192 tokens at least: every meeting of a cluster costs what 10000 tokens' pass does)
  const long long bytes = static_cast<long long>(p.V) * sizeof(T);
  int c = 1;
  while (c < 8 && (bytes / c > 101000 || (static_cast<long long>(rows) * c <= num_sms && p.V / c > 16384))) c *= 2;
  p.slice = ((p.V + c - 1) / c + 15) / 16 * 16;
  switch (c) {
    case 1: return sample_launch<T, 1>(p, rows, stream);
    case 2: return sample_launch<T, 2>(p, rows, stream);
    case 4: return sample_launch<T, 4>(p, rows, stream);
    default: return sample_launch<T, 8>(p, rows, stream);
  }
}

}  // namespace oslo

// The widest row: eight blocks' shared memory
extern "C" int oslo_sample_max_vocab(int dtype) { return 8 * 200000 / (dtype == OSLO_DT_FP32 ? 4 : 2); }

extern "C" int oslo_sample_tokens(const void* logits, long long ld, const void* uniform, int uniform64, const float* temperature,
                                  const int* top_k, const float* top_p, const float* min_p, double temperature1, int top_k1, double top_p1,
                                  double min_p1, long long* out, int rows, int V, int dtype, int num_sms, cudaStream_t stream) {
  if (rows < 0 || V <= 0 || V > oslo_sample_max_vocab(dtype)) return -1;
  if (rows == 0) return 0;
  if (rows > (1 << 24)) return -1;
  oslo::SampleParams p{};
  p.logits = logits; p.ld = ld; p.uniform = uniform; p.uniform64 = uniform64; p.temperature = temperature; p.top_k = top_k; p.top_p = top_p;
  p.min_p = min_p; p.temperature1 = temperature1; p.top_k1 = top_k1; p.top_p1 = top_p1; p.min_p1 = min_p1; p.out = out; p.V = V;
  OSLO_DISPATCH_T(dtype, return oslo::sample_any<T>(p, rows, num_sms, stream));
  return -2;
}
