// A cache whose sequences share a pool of pages: writing new keys and values (as they are, or in 8 bits), reading them back, and
// attention of one new token per sequence. Pools are [pages, heads, page, D]; row b of `table` [B, columns] names a sequence's pages in
// order, so position t of sequence b is row t % page of page table[b, t / page]. 8-bit pools hold e4m3 values and one fp32 scale per
// (page, head, row): a vector is scale * values, scale = largest magnitude / 448.
//
// A page number outside the pool, a position outside the table and a length outside [0, columns * page] are skipped or clamped (and
// reported by the bounds build), never followed.
//
// Not in the reference, whose cache grows by torch.cat (oslo/models/gptj/modeling_gptj.py:239-248).
#include <cuda_fp8.h>
#include <math_constants.h>

#include "num.cuh"
#include "oslo_kernels.h"
#include "ptx.cuh"

namespace oslo {

// ---------------------------------------------------------------------------------------------------------------- append and read
// Vectors in the order (row, k or v, head); a group of LPV lanes (8 values each) moves one. Both kernels are bound by memory: a block
// looks its rows' places up once (a search in `offsets`), then every group has U vectors on their way.
struct PagedMove {
  const void* k; const void* v;             // append: [T, heads, D] by strides (row, head)
  void* ko; void* vo;                       // read: [T, heads, D], contiguous
  void* kp; void* vp;                       // pools
  float* ks; float* vs;                     // scales of 8-bit pools
  const int* table; const int* lengths; const int* offsets;
  int* err;
  long long k_sr, k_sh, v_sr, v_sh, rows, pages;
  int B, heads, D, page, columns;
};

// The sequence of packed row r: the last b with offsets[b] <= r, provided that r < offsets[b + 1]; -1 where there is none
__device__ __forceinline__ int paged_sequence(const int* offsets, int B, long long r) {
  int lo = 0, hi = B;                       // offsets[lo] <= r < offsets[hi], if any
  if (r < offsets[0] || r >= offsets[B]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= r) lo = mid; else hi = mid;
  }
  return lo;
}
// The row of the pool (pages * page rows per head) at which position t of sequence b lies, as page * page_size + place; -1: nowhere
__device__ __forceinline__ long long paged_place(const PagedMove& p, int b, int t) {
  if (t < 0 || t / p.page >= p.columns) {
    OSLO_REPORT_BOUNDS(p.err);
    return -1;
  }
  const int id = p.table[static_cast<long long>(b) * p.columns + t / p.page];
  if (id < 0 || id >= p.pages) {
    OSLO_REPORT_BOUNDS(p.err);
    return -1;
  }
  return static_cast<long long>(id) * p.page + t % p.page;
}

template <int LPV> __device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int off = LPV / 2; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

constexpr int PM_THREADS = 256;

template <typename T, bool Q8, int LPV, int U, bool READ>
__global__ void __launch_bounds__(PM_THREADS) paged_move_kernel(const PagedMove p) {
  constexpr int GROUPS = PM_THREADS / LPV, SPAN = GROUPS * U;    // vectors a block moves
  __shared__ long long place[SPAN + 1];
  const int per = 2 * p.heads;
  const long long total = p.rows * per, v0 = static_cast<long long>(blockIdx.x) * SPAN;
  const long long r0 = v0 / per, r1 = min(p.rows - 1, (v0 + SPAN - 1) / per);
  for (int i = threadIdx.x; r0 + i <= r1; i += PM_THREADS) {
    const long long r = r0 + i;
    int b, t;
    if (p.offsets == nullptr) {
      b = static_cast<int>(r);
      t = p.lengths[b] - 1;
    } else {
      b = paged_sequence(p.offsets, p.B, r);
      if (b >= 0) t = READ ? static_cast<int>(r - p.offsets[b]) : p.lengths[b] - (p.offsets[b + 1] - static_cast<int>(r));
    }
    // a row of no sequence, and a new token of a sequence without a length for it, have no place
    place[i] = b < 0 || t < 0 ? -1 : paged_place(p, b, t);
  }
  __syncthreads();
  const int group = threadIdx.x / LPV, d0 = (threadIdx.x % LPV) * 8;
  const bool act = d0 < p.D;
  uint4 raw[U];
  float scale[U];
  long long at[U];                          // the vector's number in its pool, (page * heads + head) * page + place; -1: none
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long i = v0 + u * GROUPS + group;
    raw[u] = make_uint4(0, 0, 0, 0);
    scale[u] = 0.f;
    at[u] = -1;
    if (i >= total) continue;
    const long long r = i / per;
    const int w = static_cast<int>(i % per), h = w < p.heads ? w : w - p.heads;
    const bool val = w >= p.heads;
    const long long pl = place[r - r0];
    if (pl >= 0) at[u] = (pl / p.page * p.heads + h) * p.page + pl % p.page;
    if constexpr (READ) {
      if (at[u] < 0 || !act) continue;
      const void* pool = val ? p.vp : p.kp;
      if constexpr (Q8) {
        const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(pool) + at[u] * p.D + d0);
        raw[u].x = x.x; raw[u].y = x.y;
        scale[u] = (val ? p.vs : p.ks)[at[u]];
      } else {
        raw[u] = *reinterpret_cast<const uint4*>(static_cast<const T*>(pool) + at[u] * p.D + d0);
      }
    } else if (at[u] >= 0 && act) {
      const T* src = static_cast<const T*>(val ? p.v : p.k) + r * (val ? p.v_sr : p.k_sr) + h * (val ? p.v_sh : p.k_sh);
      raw[u] = *reinterpret_cast<const uint4*>(src + d0);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long i = v0 + u * GROUPS + group;
    const int w = static_cast<int>(i % per), h = w < p.heads ? w : w - p.heads;
    const bool val = w >= p.heads;
    const T* e = reinterpret_cast<const T*>(&raw[u]);
    if constexpr (READ) {
      if (i >= total || !act) continue;
      T* dst = static_cast<T*>(val ? p.vo : p.ko) + (i / per * p.heads + h) * p.D + d0;
      if constexpr (Q8) {
        float f[8];
        const uint32_t b2[2] = {raw[u].x, raw[u].y};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(b2[j >> 1] >> (16 * (j & 1))), __NV_E4M3);
          const float2 t2 = __half22float2(*reinterpret_cast<const __half2*>(&hr));
          f[2 * j] = t2.x * scale[u]; f[2 * j + 1] = t2.y * scale[u];
        }
        store_vec<T, 8>(dst, f);
      } else {
        *reinterpret_cast<uint4*>(dst) = raw[u];
      }
    } else if constexpr (Q8) {
      // the scale is the fp32 product with 1 / 448 and the values are e4m3 roundings (half a step: 2^-4) of fp32 quotients; a vector
      // that holds an infinity or no number reads back as no numbers: its scale is one of them
      float f[8], top = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = Num<T>::to(e[j]);
        top = fmaxf(top, fabsf(f[j]) <= CUDART_MAX_NORMAL_F ? fabsf(f[j]) : CUDART_INF_F);
      }
      top = group_max<LPV>(top);
      const float s = top * (1.f / 448.f), by = s > 0.f ? s : 1.f;
      if (at[u] < 0 || !act) continue;
      uint32_t out[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t b4 = 0;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float2 t2 = make_float2(__fdiv_rn(f[4 * j + 2 * c], by), __fdiv_rn(f[4 * j + 2 * c + 1], by));
          b4 |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(t2, __NV_SATFINITE, __NV_E4M3)) << (16 * c);
        }
        out[j] = b4;
      }
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(val ? p.vp : p.kp) + at[u] * p.D + d0) = make_uint2(out[0], out[1]);
      if (d0 == 0) (val ? p.vs : p.ks)[at[u]] = top == CUDART_INF_F ? CUDART_NAN_F : s;
    } else if (at[u] >= 0 && act) {
      *reinterpret_cast<uint4*>(static_cast<T*>(val ? p.vp : p.kp) + at[u] * p.D + d0) = raw[u];
    }
  }
}

template <typename T, bool Q8, int LPV, bool READ>
static int paged_move_launch(const PagedMove& p, int sms, cudaStream_t stream) {
  constexpr int GROUPS = PM_THREADS / LPV;
  const long long total = p.rows * 2 * p.heads;
  // four vectors a group once that still leaves every SM two blocks; a short call spreads over all SMs
  const bool deep = total >= 8ll * GROUPS * sms;
  const long long blocks = (total + GROUPS * (deep ? 4 : 1) - 1) / (GROUPS * (deep ? 4 : 1));
  if (blocks > 0x7fffffffll) return -1;
  if (deep) paged_move_kernel<T, Q8, LPV, 4, READ><<<static_cast<unsigned>(blocks), PM_THREADS, 0, stream>>>(p);
  else paged_move_kernel<T, Q8, LPV, 1, READ><<<static_cast<unsigned>(blocks), PM_THREADS, 0, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}
template <typename T, bool Q8, bool READ>
static int paged_move_dim(const PagedMove& p, int sms, cudaStream_t stream) {
  if (p.D <= 64) return paged_move_launch<T, Q8, 8, READ>(p, sms, stream);
  if (p.D <= 128) return paged_move_launch<T, Q8, 16, READ>(p, sms, stream);
  return paged_move_launch<T, Q8, 32, READ>(p, sms, stream);
}
template <bool READ>
static int paged_move(const PagedMove& p, int dtype, bool q8, int sms, cudaStream_t stream) {
  if (p.rows < 0 || p.heads <= 0 || p.D <= 0 || p.D > 256 || p.D % 8 || p.page <= 0 || p.columns <= 0 || p.pages <= 0 || p.B <= 0) return -1;
  if (p.rows == 0) return 0;
  if (dtype == OSLO_DT_BF16) return q8 ? paged_move_dim<__nv_bfloat16, true, READ>(p, sms, stream) : paged_move_dim<__nv_bfloat16, false, READ>(p, sms, stream);
  if (dtype == OSLO_DT_FP16) return q8 ? paged_move_dim<__half, true, READ>(p, sms, stream) : paged_move_dim<__half, false, READ>(p, sms, stream);
  return -2;
}

// ---------------------------------------------------------------------------------------------------------------- one new token
// o = softmax(scale q K^T) V of one query per sequence, `group` query heads to a key head. A cluster's CTAs share out the keys of one
// (sequence, key head) and join their (maximum, sum, output) through distributed shared memory: one launch, no workspace. Bound by
// how fast the pages arrive: every warp has a private queue of PA_STAGES x KPS keys in shared memory (cp.async, no barriers in the
// loop). The products of up to 16 query heads with 16 keys run on mma.sync - m16n8k16 is as small as one token's work gets; tcgen05's
// 128 rows would be 8 to 128 times more than there is - and stay far below the memory's pace.
//   16-bit pools: S = Q K^T with K straight from the queue (ldmatrix), P rounded to the pool's type for P V.
//   8-bit pools: four e4m3 bytes of ldmatrix's 32 bits become two f16 pairs. The key index inside a product and the output's columns
//   are permuted so that no byte moves between lanes; Q (divided by a power of two per row: f16 then holds it) is permuted alike, and
//   the value scales go into P, relative to the largest seen so far.
struct PagedAttn {
  const void* q;                            // [B, H, D] by strides (b, h)
  const void* kp; const void* vp;
  const float* ks; const float* vs;
  void* o;                                  // [B, H, D]
  const int* table; const int* lengths;
  int* err;
  long long q_sb, q_sh, pages;
  float scale;
  int H, heads, group, D, page, columns, window;
};
constexpr int PA_WARPS = 4;
constexpr float PA_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ void pa_cp16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void pa_cp4(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void pa_ldm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void pa_ldm4t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename M> __device__ __forceinline__ void pa_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<M, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename M> __device__ __forceinline__ uint32_t pa_pack(float a, float b) {
  if constexpr (std::is_same<M, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
__device__ __forceinline__ uint32_t pa_halves(uint32_t two) {     // two e4m3 bytes (the low 16 bits) as two f16
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// DP: head size rounded up to 64, 128 or 256. KPS keys per stage.
template <typename T, bool Q8, int DP> struct PagedShape {
  static constexpr int SIZE = Q8 ? 1 : 2;
  static constexpr int ROW = DP * SIZE;                           // bytes of a key in the queue
  static constexpr int KPS = Q8 && DP <= 128 ? 32 : 16;
  static constexpr int STAGES = DP == 64 ? 4 : (DP == 128 ? 3 : (Q8 ? 3 : 2));
  static constexpr int SCALES = Q8 ? 2 * KPS * 4 : 0;
  static constexpr int STAGE = 2 * KPS * ROW + SCALES + 16;      // keys, values, their scales, one bit per key that is there
  static constexpr int RING = STAGES * STAGE;
  // after the loop the queues hold the warps' outputs [PA_WARPS][16][DP] and the CTA's [16][DP] in 32 bits
  static constexpr int JOIN = (PA_WARPS + 1) * 16 * DP * 4;
  static constexpr int SMEM = PA_WARPS * RING > JOIN ? PA_WARPS * RING : JOIN;
};

template <typename T, bool Q8, int DP>
__global__ void __launch_bounds__(PA_WARPS * 32) paged_attn_kernel(const PagedAttn p) {
  using S = PagedShape<T, Q8, DP>;
  using M = typename std::conditional<Q8, __half, T>::type;      // the products' type
  constexpr int KPS = S::KPS, NT = KPS / 8, CH = S::ROW / 16;    // 16-byte pieces per key
  constexpr int CM = CH < 8 ? CH - 1 : 7;                        // swizzle: piece c of key r sits at c ^ (r & CM)
  extern __shared__ __align__(128) unsigned char pa_smem[];
  __shared__ float stat[PA_WARPS][16][3];                        // maximum, sum, value scale's reference
  __shared__ float fin[16][2];
  const int split = blockIdx.x, splits = gridDim.x;
  const int tiles = (p.group + 15) / 16, hk = blockIdx.y / tiles, h0 = blockIdx.y % tiles * 16, b = blockIdx.z;
  const int nh = min(16, p.group - h0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const T* qb = static_cast<const T*>(p.q) + b * p.q_sb + (static_cast<long long>(hk) * p.group + h0) * p.q_sh;

  int len = p.lengths[b];
  const long long room = static_cast<long long>(p.columns) * p.page;
  if (len < 0 || len > room) {
    OSLO_REPORT_BOUNDS(p.err);
    len = len < 0 ? 0 : static_cast<int>(room);
  }
  const int lo = p.window > 0 ? max(0, len - p.window) : 0;
  const int per = ((len - lo + splits - 1) / splits + 15) / 16 * 16;
  const int t0 = min(len, lo + split * per), t1 = min(len, t0 + per);

  // ---- the queue
  const uint32_t ring = smem_u32(pa_smem) + warp * S::RING;
  const int* row_table = p.table + static_cast<long long>(b) * p.columns;
  int ft = t0 + warp * KPS, slot_in = 0;
  int next_page = -1;                                             // page of this lane's key in the batch at ft
  auto look = [&](int t) {
    const int key = t + lane;
    return lane < KPS && key < t1 ? row_table[key / p.page] : -1;
  };
  next_page = look(ft);
  auto fetch = [&]() {
    if (ft < t1) {
      const int key = ft + lane;
      int id = next_page;
      if (lane < KPS && key < t1 && (id < 0 || id >= p.pages)) {
        OSLO_REPORT_BOUNDS(p.err);
        id = -1;
      }
      const bool have = lane < KPS && key < t1 && id >= 0;
      const long long vec = have ? (static_cast<long long>(id) * p.heads + hk) * p.page + key % p.page : -1;
      next_page = look(ft + PA_WARPS * KPS);
      const uint32_t at = ring + slot_in * S::STAGE;
      const uint32_t there = __ballot_sync(0xffffffffu, have);
      if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + S::STAGE - 16), "r"(there) : "memory");
      constexpr int LANES = CH < 32 ? CH : 32, ROWS = 32 / LANES;  // lanes on a key, keys at a time
      const int c = lane % LANES;
#pragma unroll
      for (int r0 = 0; r0 < KPS; r0 += ROWS) {
        const int r = r0 + lane / LANES;
        const long long mine = __shfl_sync(0xffffffffu, vec, r);
        const bool live = mine >= 0 && c * 16 < p.D * S::SIZE;
        const long long off = live ? mine * p.D * S::SIZE + c * 16 : 0;
        const uint32_t dst = at + r * S::ROW + ((c ^ (r & CM)) << 4);
        pa_cp16(dst, static_cast<const unsigned char*>(p.kp) + off, live);
        pa_cp16(dst + KPS * S::ROW, static_cast<const unsigned char*>(p.vp) + off, live);
      }
      if constexpr (Q8) {
        if (lane < KPS) {
          const uint32_t dst = at + 2 * KPS * S::ROW + lane * 4;
          pa_cp4(dst, p.ks + (have ? vec : 0), have);
          pa_cp4(dst + KPS * 4, p.vs + (have ? vec : 0), have);
        }
      }
    }
    ft += PA_WARPS * KPS;
    if (++slot_in == S::STAGES) slot_in = 0;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < S::STAGES - 1; ++i) fetch();

  // ---- queries as the left operand: rows g and g + 8 of the tile
  uint32_t qa[DP / 16][4];
  float unit[2] = {1.f, 1.f};                                     // Q8: the power of two that a row was divided by
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = g + 8 * half;
    const T* qr = qb + row * p.q_sh;
    float top = 0.f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int d = kk * 16 + (Q8 ? 4 * t4 + 2 * j : 2 * t4 + 8 * j);
        const bool in = row < nh && d < p.D;
        const float x = in ? Num<T>::to(qr[d]) : 0.f, y = in ? Num<T>::to(qr[d + 1]) : 0.f;
        if constexpr (Q8) {
          top = fmaxf(top, fmaxf(fabsf(x), fabsf(y)));
          const __nv_bfloat162 two = __floats2bfloat162_rn(x, y); // parked until the row's largest is known
          const __half2 twoh = __floats2half2_rn(x, y);
          qa[kk][half + 2 * j] = std::is_same<T, __half>::value ? *reinterpret_cast<const uint32_t*>(&twoh) : *reinterpret_cast<const uint32_t*>(&two);
        } else {
          qa[kk][half + 2 * j] = pa_pack<M>(x, y);
        }
      }
    }
    if constexpr (Q8 && !std::is_same<T, __half>::value) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^e with top / 2^e in [1, 2); rows of zeros, infinities and no numbers as they are
      const int e = top > 0.f && top <= CUDART_MAX_NORMAL_F ? min(126, max(-126, ilogbf(top))) : 0;
      unit[half] = ldexpf(1.f, e);
      const float inv = ldexpf(1.f, -e);
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t raw = qa[kk][half + 2 * j];
          const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw));
          qa[kk][half + 2 * j] = pa_pack<__half>(x.x * inv, x.y * inv);
        }
      }
    }
  }
  const float mult[2] = {p.scale * PA_LOG2E * unit[0], p.scale * PA_LOG2E * unit[1]};

  float o[DP / 8][4];
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) { o[i][0] = 0.f; o[i][1] = 0.f; o[i][2] = 0.f; o[i][3] = 0.f; }
  float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};
  float vref = 0.f;                                               // Q8: largest value scale so far (0: none)
  int slot = 0;
  for (int tb = t0 + warp * KPS; tb < t1; tb += PA_WARPS * KPS) {
    fetch();                                                      // into the slot of the batch before this one
    asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 1) : "memory");
    __syncwarp();                                                 // the other lanes' pieces too
    const uint32_t at = ring + slot * S::STAGE, atv = at + KPS * S::ROW;
    if (++slot == S::STAGES) slot = 0;
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) { s[n][0] = 0.f; s[n][1] = 0.f; s[n][2] = 0.f; s[n][3] = 0.f; }
    if constexpr (!Q8) {
      // matrices of one ldmatrix: keys n..n+7 / n+8..n+15, pieces c / c + 1
      const int r = (lane & 7) + ((lane >> 4) << 3), c = (lane >> 3) & 1;
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          uint32_t kf[4];
          const int row = n * 8 + r;
          pa_ldm4(kf, at + row * S::ROW + (((2 * kk + c) ^ (row & CM)) << 4));
          pa_mma<M>(s[n], qa[kk], kf[0], kf[1]);
          pa_mma<M>(s[n + 1], qa[kk], kf[2], kf[3]);
        }
      }
    } else {
      // matrices: 8 keys, pieces c .. c + 3, 16 values each
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int row = n * 8 + (lane & 7);
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk += 4) {
          uint32_t kf[4];
          pa_ldm4(kf, at + row * S::ROW + (((kk + (lane >> 3)) ^ (row & CM)) << 4));
#pragma unroll
          for (int i = 0; i < 4; ++i) pa_mma<M>(s[n], qa[kk + i], pa_halves(kf[i] & 0xffffu), pa_halves(kf[i] >> 16));
        }
      }
    }
    // ---- scores in log2 units; keys behind the last one, or without a page, have none
    uint32_t there;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(there) : "r"(at + S::STAGE - 16) : "memory");
    float mx[2] = {-CUDART_INF_F, -CUDART_INF_F};
    float vscale[NT][2], vtop = vref;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int key = n * 8 + 2 * t4 + j;
        float kscale = 1.f;
        if constexpr (Q8) {
          const float* sc = reinterpret_cast<const float*>(pa_smem + (at - smem_u32(pa_smem)) + 2 * KPS * S::ROW);
          kscale = sc[key];
          vscale[n][j] = sc[KPS + key];
          vtop = fmaxf(vtop, vscale[n][j]);
        }
        const bool in = (there >> key) & 1u;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float& x = s[n][2 * half + j];
          x = in ? x * (Q8 ? mult[half] * kscale : mult[half]) : -CUDART_INF_F;
          mx[half] = fmaxf(mx[half], x);
        }
      }
    }
    float keep[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 1));
      mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 2));
      const float mn = fmaxf(m[half], mx[half]);
      keep[half] = mn == -CUDART_INF_F ? 1.f : exp2f(m[half] - mn);
      m[half] = mn;
      l[half] *= keep[half];
    }
    float vinv = 1.f;
    if constexpr (Q8) {
      vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, 1));
      vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, 2));
      const float shrink = vtop > 0.f ? vref / vtop : 1.f;
      keep[0] *= shrink;
      keep[1] *= shrink;
      vref = vtop;
      vinv = vtop > 0.f ? 1.f / vtop : 0.f;
    }
    uint32_t pf[NT / 2][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float base = m[half] == -CUDART_INF_F ? 0.f : m[half];
        const float e0 = exp2f(s[n][2 * half] - base), e1 = exp2f(s[n][2 * half + 1] - base);
        l[half] += e0 + e1;
        if constexpr (Q8) pf[n >> 1][half + 2 * (n & 1)] = pa_pack<M>(e0 * (vscale[n][0] * vinv), e1 * (vscale[n][1] * vinv));
        else pf[n >> 1][half + 2 * (n & 1)] = pa_pack<M>(e0, e1);
      }
    }
    if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) { o[i][0] *= keep[0]; o[i][1] *= keep[0]; o[i][2] *= keep[1]; o[i][3] *= keep[1]; }
    }
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      const int row = n * 8 + (lane & 15);                        // matrices: keys 0-7 and 8-15 of piece c, then of piece c + 1
#pragma unroll
      for (int c = 0; c < CH; c += 2) {
        uint32_t vf[4];
        pa_ldm4t(vf, atv + row * S::ROW + (((c + (lane >> 4)) ^ (row & CM)) << 4));
        if constexpr (!Q8) {
          pa_mma<M>(o[c], pf[n >> 1], vf[0], vf[1]);
          pa_mma<M>(o[c + 1], pf[n >> 1], vf[2], vf[3]);
        } else {
          // 32 bits: columns 2g and 2g + 1 of two keys; even columns to one product, odd ones to the next
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t a = vf[2 * i], z = vf[2 * i + 1];
            pa_mma<M>(o[2 * (c + i)], pf[n >> 1], pa_halves(__byte_perm(a, 0, 0x4420)), pa_halves(__byte_perm(z, 0, 0x4420)));
            pa_mma<M>(o[2 * (c + i) + 1], pf[n >> 1], pa_halves(__byte_perm(a, 0, 0x4431)), pa_halves(__byte_perm(z, 0, 0x4431)));
          }
        }
      }
    }
    __syncwarp();                                                 // all lanes have read the slot before it is filled again
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
    l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
  }
  __syncthreads();                                                // the queues are empty: their space takes the outputs

  // ---- the block's warps
  float* part = reinterpret_cast<float*>(pa_smem);                // [PA_WARPS][16][DP]
  float* mine = part + PA_WARPS * 16 * DP;                        // [16][DP]
  const float vback = Q8 ? vref : 1.f;
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = 2 * t4 + j;
        const int d = Q8 ? (i >> 1) * 16 + 2 * n + (i & 1) : i * 8 + n;
        part[(warp * 16 + g + 8 * half) * DP + d] = o[i][2 * half + j] * vback;
      }
    }
  }
  if (t4 == 0) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      stat[warp][g + 8 * half][0] = m[half];
      stat[warp][g + 8 * half][1] = l[half];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nh * DP; i += PA_WARPS * 32) {
    const int row = i / DP;
    float mm = -CUDART_INF_F, sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) mm = fmaxf(mm, stat[w][row][0]);
    const float base = mm == -CUDART_INF_F ? 0.f : mm;
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) {
      const float f = exp2f(stat[w][row][0] - base);
      sum += f * stat[w][row][1];
      acc += f * part[(w * 16 + row) * DP + i % DP];
    }
    mine[i] = acc;
    if (i % DP == 0) {
      fin[row][0] = mm;
      fin[row][1] = sum;
    }
  }
  // ---- the cluster's blocks, in their order; each writes its share of the result
  T* out = static_cast<T*>(p.o) + (static_cast<long long>(b) * p.H + static_cast<long long>(hk) * p.group + h0) * p.D;
  if (splits > 1) cluster_sync_all();
  else __syncthreads();
  const uint32_t mine_s = smem_u32(mine), fin_s = smem_u32(&fin[0][0]);
  auto peer = [&](uint32_t addr, int r) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(addr, r)) : "memory");
    return v;
  };
  for (int i = split * PA_WARPS * 32 + threadIdx.x; i < nh * DP; i += splits * PA_WARPS * 32) {
    const int row = i / DP, d = i % DP;
    if (d >= p.D) continue;
    float val, sum;
    if (splits == 1) {
      sum = fin[row][1];
      val = mine[i];
    } else {
      float mm = -CUDART_INF_F;
      for (int r = 0; r < splits; ++r) mm = fmaxf(mm, peer(fin_s + row * 8, r));
      const float base = mm == -CUDART_INF_F ? 0.f : mm;
      sum = 0.f;
      val = 0.f;
      for (int r = 0; r < splits; ++r) {
        const float f = exp2f(peer(fin_s + row * 8, r) - base);
        sum += f * peer(fin_s + row * 8 + 4, r);
        val += f * peer(mine_s + i * 4, r);
      }
    }
    out[row * p.D + d] = Num<T>::from(sum == 0.f ? 0.f : val / sum);
  }
  if (splits > 1) cluster_sync_all();                             // nobody leaves while another reads its shared memory
}

template <typename T, bool Q8, int DP>
static int paged_attn_launch(const PagedAttn& p, int B, int splits, cudaStream_t stream) {
  using S = PagedShape<T, Q8, DP>;
  static_assert(S::SMEM <= 231000, "shared memory budget of one CTA");
  auto kernel = paged_attn_kernel<T, Q8, DP>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  static unsigned long long ready = 0;                            // one bit per device
  if (dev > 63 || !((__atomic_load_n(&ready, __ATOMIC_ACQUIRE) >> dev) & 1)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev <= 63) __atomic_fetch_or(&ready, 1ull << dev, __ATOMIC_RELEASE);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits, p.heads * ((p.group + 15) / 16), B);
  cfg.blockDim = dim3(PA_WARPS * 32);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kernel, p);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}
template <typename T, bool Q8>
static int paged_attn_dim(const PagedAttn& p, int B, int splits, cudaStream_t stream) {
  if (p.D <= 64) return paged_attn_launch<T, Q8, 64>(p, B, splits, stream);
  if (p.D <= 128) return paged_attn_launch<T, Q8, 128>(p, B, splits, stream);
  return paged_attn_launch<T, Q8, 256>(p, B, splits, stream);
}

}  // namespace oslo

extern "C" int oslo_paged_append(const void* k, const void* v, long long k_sr, long long k_sh, long long v_sr, long long v_sh, void* k_pages,
                                 void* v_pages, float* k_scale, float* v_scale, const int* table, const int* lengths, const int* offsets,
                                 long long rows, int B, int heads, int D, long long pages, int page, int columns, int dtype, int q8,
                                 int* err_word, int num_sms, cudaStream_t stream) {
  oslo::PagedMove p{};
  p.k = k; p.v = v; p.k_sr = k_sr; p.k_sh = k_sh; p.v_sr = v_sr; p.v_sh = v_sh;
  p.kp = k_pages; p.vp = v_pages; p.ks = k_scale; p.vs = v_scale; p.table = table; p.lengths = lengths; p.offsets = offsets;
  p.err = err_word; p.rows = rows; p.pages = pages; p.B = B; p.heads = heads; p.D = D; p.page = page; p.columns = columns;
  return oslo::paged_move<false>(p, dtype, q8 != 0, num_sms, stream);
}

extern "C" int oslo_paged_read(const void* k_pages, const void* v_pages, const float* k_scale, const float* v_scale, void* k, void* v,
                               const int* table, const int* offsets, long long rows, int B, int heads, int D, long long pages, int page,
                               int columns, int dtype, int q8, int* err_word, int num_sms, cudaStream_t stream) {
  oslo::PagedMove p{};
  p.ko = k; p.vo = v; p.kp = const_cast<void*>(k_pages); p.vp = const_cast<void*>(v_pages);
  p.ks = const_cast<float*>(k_scale); p.vs = const_cast<float*>(v_scale); p.table = table; p.offsets = offsets;
  p.err = err_word; p.rows = rows; p.pages = pages; p.B = B; p.heads = heads; p.D = D; p.page = page; p.columns = columns;
  return oslo::paged_move<true>(p, dtype, q8 != 0, num_sms, stream);
}

extern "C" int oslo_paged_attn(const void* q, long long q_sb, long long q_sh, const void* k_pages, const void* v_pages, const float* k_scale,
                               const float* v_scale, void* o, const int* table, const int* lengths, int B, int H, int heads, int D,
                               long long pages, int page, int columns, float scale, int window, int dtype, int q8, int* err_word,
                               int num_sms, cudaStream_t stream) {
  if (B <= 0 || H <= 0 || heads <= 0 || H % heads || D <= 0 || D > 256 || D % 8 || page <= 0 || columns <= 0 || pages <= 0) return -1;
  if (B > 65535 || heads * ((H / heads + 15) / 16) > 65535) return -1;
  if (static_cast<long long>(columns) * page > 0x7fffffffll) return -1;
  oslo::PagedAttn p{};
  p.q = q; p.q_sb = q_sb; p.q_sh = q_sh; p.kp = k_pages; p.vp = v_pages; p.ks = k_scale; p.vs = v_scale; p.o = o; p.table = table;
  p.lengths = lengths; p.err = err_word; p.pages = pages; p.scale = scale; p.H = H; p.heads = heads; p.group = H / heads; p.D = D;
  p.page = page; p.columns = columns; p.window = window;
  // splits of a sequence's keys: enough for a few blocks per SM, none shorter than 64 keys of the longest possible sequence
  const long long units = static_cast<long long>(B) * heads * ((p.group + 15) / 16), most = static_cast<long long>(columns) * page;
  const long long span = window > 0 && window < most ? window : most;
  int splits = 1;
  while (splits < 8 && units * splits < 4ll * num_sms && span > 64ll * splits) splits *= 2;
  if (dtype == OSLO_DT_BF16) return q8 ? oslo::paged_attn_dim<__nv_bfloat16, true>(p, B, splits, stream) : oslo::paged_attn_dim<__nv_bfloat16, false>(p, B, splits, stream);
  if (dtype == OSLO_DT_FP16) return q8 ? oslo::paged_attn_dim<__half, true>(p, B, splits, stream) : oslo::paged_attn_dim<__half, false>(p, B, splits, stream);
  return -2;
}
