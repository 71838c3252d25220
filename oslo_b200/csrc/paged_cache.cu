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
// Vectors in the order (row, head), keys and values by different blocks (gridDim.y); a group of LPV lanes (8 values each) moves one. Both
// kernels are bound by memory, as long as a vector's way is found in a few instructions: a block looks its rows' places up once (a search
// in `offsets`), and a group walks from vector to vector without dividing. U vectors are on their way at a time. 8104 rows of 8 heads of 128
// into 8 bits: 15 us (3.3 TB/s; 39 with a division per vector); 65000 rows from 8 bits: 73 us (5.5 TB/s; 153), from 16 bits 85 us (6.2 TB/s).
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
// The vector of the pool at which position t of sequence b lies for head 0 (head h: h * page further); -1: nowhere
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
  return static_cast<long long>(id) * p.heads * p.page + t % p.page;
}

// The largest magnitude of a group's 16-bit values, as an fp32 number; infinity for infinities and what is no number. Magnitudes of either
// type order like their bits, and those two kinds have the largest.
template <typename T, int LPV> __device__ __forceinline__ float group_top(const uint4& raw) {
  uint32_t x = __vmaxu2(__vmaxu2(raw.x & 0x7fff7fffu, raw.y & 0x7fff7fffu), __vmaxu2(raw.z & 0x7fff7fffu, raw.w & 0x7fff7fffu));
#pragma unroll
  for (int off = LPV / 2; off > 0; off >>= 1) x = __vmaxu2(x, __shfl_xor_sync(0xffffffffu, x, off));
  const uint16_t top = static_cast<uint16_t>(max(x & 0xffffu, x >> 16));
  if constexpr (std::is_same<T, __half>::value) return top >= 0x7c00 ? CUDART_INF_F : __half2float(__ushort_as_half(top));
  else return top >= 0x7f80 ? CUDART_INF_F : __bfloat162float(__ushort_as_bfloat16(top));
}

constexpr int PM_THREADS = 256, PM_OFFSETS = 1024;

template <typename T, bool Q8, int LPV, int U, int R, bool READ>
__global__ void __launch_bounds__(PM_THREADS) paged_move_kernel(const PagedMove p) {
  constexpr int GROUPS = PM_THREADS / LPV, SPAN = GROUPS * U * R;            // vectors a block moves, U a group at a time
  __shared__ long long place[SPAN + 1];
  __shared__ int starts[PM_OFFSETS + 1];
  const int per = p.heads;
  const long long total = p.rows * per, v0 = static_cast<long long>(blockIdx.x) * SPAN;
  const long long r0 = v0 / per;
  const int skip = static_cast<int>(v0 - r0 * per), span = static_cast<int>(min(static_cast<long long>(SPAN), total - v0));
  const int last = (skip + span - 1) / per;
  const int* offsets = p.offsets;
  if (p.offsets != nullptr && p.B <= PM_OFFSETS) {              // one load instead of a chain of them
    for (int i = threadIdx.x; i <= p.B; i += PM_THREADS) starts[i] = p.offsets[i];
    offsets = starts;
    __syncthreads();
  }
  for (int i = threadIdx.x; i <= last; i += PM_THREADS) {
    const long long r = r0 + i;
    int b, t;
    if (p.offsets == nullptr) {
      b = static_cast<int>(r);
      t = p.lengths[b] - 1;
    } else {
      b = paged_sequence(offsets, p.B, r);
      if (b >= 0) t = READ ? static_cast<int>(r - offsets[b]) : p.lengths[b] - (offsets[b + 1] - static_cast<int>(r));
    }
    // a row of no sequence, and a new token of a sequence without a length for it, have no place
    place[i] = b < 0 || t < 0 ? -1 : paged_place(p, b, t);
  }
  __syncthreads();
  const bool val = blockIdx.y != 0;
  const T* src = static_cast<const T*>(val ? p.v : p.k);
  T* dst = static_cast<T*>(val ? p.vo : p.ko);
  void* pool = val ? p.vp : p.kp;
  float* scales = val ? p.vs : p.ks;
  const long long sr = val ? p.v_sr : p.k_sr, sh = val ? p.v_sh : p.k_sh;
  const int group = threadIdx.x / LPV, d0 = (threadIdx.x % LPV) * 8;
  const bool act = d0 < p.D;
  int left = span - group;                  // vectors from this group's next one to the block's last
  int row = (skip + group) / per, h = skip + group - row * per;
  const int rows_on = GROUPS / per, heads_on = GROUPS - rows_on * per;
  for (int it = 0; it < R; ++it) {
    uint4 raw[U];
    float scale[U];
    long long at[U], out[U];                // the vector's number in its pool, and in the packed rows; -1: none
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw[u] = make_uint4(0, 0, 0, 0);
      scale[u] = 0.f;
      at[u] = out[u] = -1;
      if (left > 0) {
        const long long pl = place[row];
        if (pl >= 0) at[u] = pl + h * p.page;
        out[u] = (r0 + row) * per + h;
        if constexpr (READ) {
          if (pl >= 0 && act) {
            if constexpr (Q8) {
              const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(pool) + at[u] * p.D + d0);
              raw[u].x = x.x; raw[u].y = x.y;
              scale[u] = scales[at[u]];
            } else {
              raw[u] = *reinterpret_cast<const uint4*>(static_cast<const T*>(pool) + at[u] * p.D + d0);
            }
          }
        } else if (pl >= 0 && act) {
          raw[u] = *reinterpret_cast<const uint4*>(src + (r0 + row) * sr + h * sh + d0);
        }
      }
      left -= GROUPS;
      row += rows_on;
      h += heads_on;
      if (h >= per) { h -= per; ++row; }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (READ) {
        if (out[u] < 0 || !act) continue;
        if constexpr (Q8) {
          float f[8];
          const uint32_t b2[2] = {raw[u].x, raw[u].y};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(b2[j >> 1] >> (16 * (j & 1))), __NV_E4M3);
            const float2 t2 = __half22float2(*reinterpret_cast<const __half2*>(&hr));
            f[2 * j] = t2.x * scale[u]; f[2 * j + 1] = t2.y * scale[u];
          }
          store_vec<T, 8>(dst + out[u] * p.D + d0, f);
        } else {
          *reinterpret_cast<uint4*>(dst + out[u] * p.D + d0) = raw[u];
        }
      } else if constexpr (Q8) {
        // the scale is the fp32 product with 1 / 448 and the values are e4m3 roundings (half a step: 2^-4) of fp32 products with its
        // reciprocal (eight divisions a lane cost as much as the memory takes); a vector that holds an infinity or no number, and
        // one whose largest is too small for a reciprocal, reads back as no numbers or as zeros
        const float top = group_top<T, LPV>(raw[u]);
        if (at[u] < 0 || !act) continue;
        const float s = top * (1.f / 448.f), r = __fdiv_rn(1.f, s), by = r <= CUDART_MAX_NORMAL_F ? r : 0.f;
        const T* e = reinterpret_cast<const T*>(&raw[u]);
        uint32_t bytes[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          bytes[j] = 0;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float2 t2 = make_float2(Num<T>::to(e[4 * j + 2 * c]) * by, Num<T>::to(e[4 * j + 2 * c + 1]) * by);
            bytes[j] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(t2, __NV_SATFINITE, __NV_E4M3)) << (16 * c);
          }
        }
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(pool) + at[u] * p.D + d0) = make_uint2(bytes[0], bytes[1]);
        if (d0 == 0) scales[at[u]] = top == CUDART_INF_F ? CUDART_NAN_F : s;
      } else if (at[u] >= 0 && act) {
        *reinterpret_cast<uint4*>(static_cast<T*>(pool) + at[u] * p.D + d0) = raw[u];
      }
    }
  }
}

template <typename T, bool Q8, int LPV, bool READ>
static int paged_move_launch(const PagedMove& p, int sms, cudaStream_t stream) {
  constexpr int GROUPS = PM_THREADS / LPV;
  const long long total = p.rows * p.heads;
  // a block looks up its rows' places once: sixteen vectors a group where that leaves every SM two blocks (four on their way at a time),
  // one where a short call has to spread over all SMs
  const int deep = total >= 16ll * GROUPS * sms ? 16 : (total >= 4ll * GROUPS * sms ? 4 : 1);
  const long long blocks = (total + GROUPS * deep - 1) / (GROUPS * deep);
  if (blocks > 0x7fffffffll) return -1;
  const dim3 grid(static_cast<unsigned>(blocks), 2);
  if (deep == 16) paged_move_kernel<T, Q8, LPV, 4, 4, READ><<<grid, PM_THREADS, 0, stream>>>(p);
  else if (deep == 4) paged_move_kernel<T, Q8, LPV, 4, 1, READ><<<grid, PM_THREADS, 0, stream>>>(p);
  else paged_move_kernel<T, Q8, LPV, 1, 1, READ><<<grid, PM_THREADS, 0, stream>>>(p);
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
// how fast the pages arrive: every warp has a private queue of STAGES x 16 keys in shared memory (cp.async, no barriers in the loop).
// The products of 16 keys with 8 query heads (NB = 2: 16) run on mma.sync - m16n8k16 with the keys as its 16 rows is as small as one
// token's work gets; tcgen05's 128 rows would be 8 to 128 times more than there is - and stay far below the memory's pace.
//   S^T = K q^T: K straight from the queue (ldmatrix). A weight's reference follows the running maximum only when a score has outgrown
//   it by 2^8, so a step usually needs one vote and no exchange. P^T is rounded to the pool's type, since the products take two operands of
//   one 16-bit type (half a step: 2^-8 of a weight in bf16, 2^-11 in fp16, as for the result itself; e4m3 pools: f16, 2^-11), and turned by
//   movmatrix into the right operand of O^T = V^T P^T.
//   8-bit pools: four e4m3 bytes of ldmatrix's 32 bits become two f16 pairs. The column index inside the first product and the rows of
//   the second are permuted so that no byte moves between lanes; q (divided by a power of two per head: f16 then holds it) is permuted
//   alike, and the value scales go into P, relative to the largest seen so far or a sixteenth of it.
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
  int B, by_length;                         // by_length: blocks take the sequences in the order of their lengths, the longest first
};
constexpr int PA_WARPS = 4, PA_SORTED = 512;
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

__device__ __forceinline__ uint32_t pa_turn(uint32_t x) {            // an 8 x 8 matrix of 16-bit values, transposed
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// The sequence with `rank` longer ones (equal lengths: by number). Blocks that start late then have little to do: 128 sequences of 1 to
// 6000 tokens, 8 key heads, 8 bits: 228 us without
__device__ __forceinline__ int pa_by_length(const int* lengths, int B, int rank, int* space) {
  __shared__ int found;
  for (int i = threadIdx.x; i < B; i += PA_WARPS * 32) space[i] = lengths[i];
  __syncthreads();
  for (int i = threadIdx.x; i < B; i += PA_WARPS * 32) {
    const int mine = space[i];
    int ahead = 0;
#pragma unroll 8
    for (int j = 0; j < B; ++j) ahead += space[j] > mine || (space[j] == mine && j < i);
    if (ahead == rank) found = i;
  }
  __syncthreads();
  return found;
}

// DP: head size rounded up to 64, 128 or 256; NB: 8 NB query heads per CTA
template <typename T, bool Q8, int DP, int NB> struct PagedShape {
  static constexpr int SIZE = Q8 ? 1 : 2, KPS = 16;
  static constexpr int ROW = DP * SIZE;                           // bytes of a key in the queue
  static constexpr int STAGE = 2 * KPS * ROW + (Q8 ? 2 * KPS * 4 : 0) + 16;      // keys, values, their scales, one bit per key that is there
  static constexpr int STAGES = ROW <= 64 ? 6 : (ROW <= 128 ? 4 : 3);
  static constexpr int RING = STAGES * STAGE;
  // after the loop the queues hold the warps' outputs and the CTA's, [PA_WARPS + 1][8 NB][DP] in 32 bits
  static constexpr int JOIN = (PA_WARPS + 1) * 8 * NB * DP * 4;
  static constexpr int SMEM = PA_WARPS * RING > JOIN ? PA_WARPS * RING : JOIN;
};

template <typename T, bool Q8, int DP, int NB>
__global__ void __launch_bounds__(PA_WARPS * 32) paged_attn_kernel(const PagedAttn p) {
  using S = PagedShape<T, Q8, DP, NB>;
  using M = typename std::conditional<Q8, __half, T>::type;      // the products' type
  constexpr int KPS = S::KPS, CH = S::ROW / 16, HEADS = 8 * NB;  // CH: 16-byte pieces per key
  constexpr int CM = CH < 8 ? CH - 1 : 7;                        // swizzle: piece c of key r sits at c ^ (r & CM)
  extern __shared__ __align__(128) unsigned char pa_smem[];
  __shared__ float stat[PA_WARPS][HEADS][2];                     // maximum, sum
  __shared__ float fin[HEADS][2];
  const int split = blockIdx.x, splits = gridDim.x;
  const int tiles = (p.group + HEADS - 1) / HEADS, hk = blockIdx.y / tiles, h0 = blockIdx.y % tiles * HEADS;
  const int b = p.by_length ? pa_by_length(p.lengths, p.B, blockIdx.z, reinterpret_cast<int*>(pa_smem)) : blockIdx.z;
  const int nh = min(HEADS, p.group - h0);
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
  auto look = [&](int t) {                                        // page of this lane's key in the batch at t
    const int key = t + lane;
    return lane < KPS && key < t1 ? row_table[key / p.page] : -1;
  };
  int next_page = look(ft);
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

  // ---- queries as the right operand: this lane's head of every 8 is g. 8-bit pools: columns in the order of the keys' bytes
  uint32_t qf[NB][DP / 16][2];
  float mult[NB][2];                                              // of the heads 2 t4 and 2 t4 + 1 (S^T's columns)
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int head = nb * 8 + g;
    const T* qr = qb + head * p.q_sh;
    float top = 0.f, unit = 1.f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int d = kk * 16 + (Q8 ? 4 * t4 + 2 * j : 2 * t4 + 8 * j);
        qf[nb][kk][j] = head < nh && d < p.D ? *reinterpret_cast<const uint32_t*>(qr + d) : 0u;
      }
    }
    if constexpr (Q8 && !std::is_same<T, __half>::value) {
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qf[nb][kk][j]));
          top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^e with top / 2^e in [1, 2); heads of zeros, infinities and no numbers as they are
      const int e = top > 0.f && top <= CUDART_MAX_NORMAL_F ? min(126, max(-126, ilogbf(top))) : 0;
      unit = ldexpf(1.f, e);
      const float inv = ldexpf(1.f, -e);
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qf[nb][kk][j]));
          qf[nb][kk][j] = pa_pack<__half>(x.x * inv, x.y * inv);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) mult[nb][j] = p.scale * PA_LOG2E * __shfl_sync(0xffffffffu, unit, (2 * t4 + j) * 4);
  }

  float o[NB][DP / 16][4];
  float m[NB][2], l[NB][2];                                       // reference and this lane's sum, heads 2 t4 + j
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[nb][i][j] = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) { m[nb][j] = -CUDART_INF_F; l[nb][j] = 0.f; }
  }
  float vref = 0.f, vinv = 0.f;                                   // Q8: the value scales' reference (0: none yet)
  uint32_t met = 0;                                               // whether this warp has met a key
  int slot = 0;
  for (int tb = t0 + warp * KPS; tb < t1; tb += PA_WARPS * KPS) {
    fetch();                                                      // into the slot of the batch before this one
    asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 1) : "memory");
    __syncwarp();                                                 // the other lanes' pieces too
    const uint32_t at = ring + slot * S::STAGE, atv = at + KPS * S::ROW;
    if (++slot == S::STAGES) slot = 0;
    float s[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) { s[nb][0] = 0.f; s[nb][1] = 0.f; s[nb][2] = 0.f; s[nb][3] = 0.f; }
    {
      const int r = lane & 15, c = lane >> 4;                     // matrices: keys 0-7 and 8-15 of one piece, then of the next
      if constexpr (!Q8) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          uint32_t kf[4];
          pa_ldm4(kf, at + r * S::ROW + (((2 * kk + c) ^ (r & CM)) << 4));
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) pa_mma<M>(s[nb], kf, qf[nb][kk][0], qf[nb][kk][1]);
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk += 2) {                 // a piece is 16 values of a key
          uint32_t x[4];
          pa_ldm4(x, at + r * S::ROW + (((kk + c) ^ (r & CM)) << 4));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t kf[4] = {pa_halves(x[2 * i] & 0xffffu), pa_halves(x[2 * i + 1] & 0xffffu), pa_halves(x[2 * i] >> 16), pa_halves(x[2 * i + 1] >> 16)};
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) pa_mma<M>(s[nb], kf, qf[nb][kk + i][0], qf[nb][kk + i][1]);
          }
        }
      }
    }
    // ---- scores in log2 units; keys behind the last one, or without a page, have none. This lane's keys: g and g + 8
    uint32_t there;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(there) : "r"(at + S::STAGE - 16) : "memory");
    met |= there;
    const bool in[2] = {((there >> g) & 1u) != 0, ((there >> (g + 8)) & 1u) != 0};
    float kscale[2] = {1.f, 1.f}, vscale[2] = {1.f, 1.f};
    if constexpr (Q8) {
      const float* sc = reinterpret_cast<const float*>(pa_smem + (at - smem_u32(pa_smem)) + 2 * KPS * S::ROW);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        kscale[half] = sc[g + 8 * half];
        vscale[half] = sc[KPS + g + 8 * half];
      }
    }
    bool grow = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float& x = s[nb][2 * half + j];
          x = in[half] ? x * (Q8 ? mult[nb][j] * kscale[half] : mult[nb][j]) : -CUDART_INF_F;
          grow |= x > m[nb][j] + 8.f;
        }
      }
    }
    if constexpr (Q8) grow |= fmaxf(in[0] ? vscale[0] : 0.f, in[1] ? vscale[1] : 0.f) > 16.f * vref;
    if (__any_sync(0xffffffffu, grow)) {                          // the references follow; what has been summed is brought to them
      float shrink = 1.f;
      if constexpr (Q8) {
        float v = fmaxf(vref, fmaxf(in[0] ? vscale[0] : 0.f, in[1] ? vscale[1] : 0.f));
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
        shrink = v > 0.f ? vref / v : 1.f;
        vref = v;
        vinv = v > 0.f ? 1.f / v : 0.f;
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x = fmaxf(m[nb][j], fmaxf(s[nb][j], s[nb][2 + j]));
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
          const float keep = x == -CUDART_INF_F ? 1.f : exp2f(m[nb][j] - x);
          m[nb][j] = x;
          l[nb][j] *= keep;
#pragma unroll
          for (int i = 0; i < DP / 16; ++i) {                     // O^T's columns are S^T's
            o[nb][i][j] *= keep * shrink;
            o[nb][i][2 + j] *= keep * shrink;
          }
        }
      }
    }
    uint32_t pf[NB][2];                                           // P^T, keys 0-7 and 8-15
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float e[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          e[j] = exp2f(s[nb][2 * half + j] - (m[nb][j] == -CUDART_INF_F ? 0.f : m[nb][j]));
          l[nb][j] += e[j];
        }
        const float f = Q8 ? (in[half] ? vscale[half] * vinv : 0.f) : 1.f;
        pf[nb][half] = pa_turn(Q8 ? pa_pack<M>(e[0] * f, e[1] * f) : pa_pack<M>(e[0], e[1]));
      }
    }
    {
      const int r = (lane & 7) + ((lane >> 4) << 3), c = (lane >> 3) & 1;      // matrices: keys 0-7 of a piece and of the next, then keys 8-15
#pragma unroll
      for (int i = 0; i < CH; i += 2) {
        uint32_t x[4];
        pa_ldm4t(x, atv + r * S::ROW + (((i + c) ^ (r & CM)) << 4));
        if constexpr (!Q8) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) pa_mma<M>(o[nb][i / 2], x, pf[nb][0], pf[nb][1]);
        } else {
          // 32 bits: columns 2g and 2g + 1 of two keys; even columns are the product's rows 0-7, odd ones its rows 8-15
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t a = x[u], z = x[2 + u];
            const uint32_t vf[4] = {pa_halves(__byte_perm(a, 0, 0x4420)), pa_halves(__byte_perm(a, 0, 0x4431)),
                                    pa_halves(__byte_perm(z, 0, 0x4420)), pa_halves(__byte_perm(z, 0, 0x4431))};
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) pa_mma<M>(o[nb][i + u], vf, pf[nb][0], pf[nb][1]);
          }
        }
      }
    }
    __syncwarp();                                                 // all lanes have read the slot before it is filled again
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l[nb][j] += __shfl_xor_sync(0xffffffffu, l[nb][j], off);
  __syncthreads();                                                // the queues are empty: their space takes the outputs

  // ---- the block's warps
  float* part = reinterpret_cast<float*>(pa_smem);                // [PA_WARPS][HEADS][DP]
  float* mine = part + PA_WARPS * HEADS * DP;                     // [HEADS][DP]
  const float vback = Q8 ? vref : 1.f;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int d = i * 16 + (Q8 ? 2 * g + half : g + 8 * half);
          part[(warp * HEADS + nb * 8 + 2 * t4 + j) * DP + d] = o[nb][i][2 * half + j] * vback;
        }
      }
    }
    if (g == 0) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // no finite score among keys that are there is not the same as no key: it ends in 0 / 0
        stat[warp][nb * 8 + 2 * t4 + j][0] = met && m[nb][j] == -CUDART_INF_F ? -CUDART_MAX_NORMAL_F : m[nb][j];
        stat[warp][nb * 8 + 2 * t4 + j][1] = l[nb][j];
      }
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
      acc += f * part[(w * HEADS + row) * DP + i % DP];
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
    float val, sum, mm = -CUDART_INF_F;
    if (splits == 1) {
      mm = fin[row][0];
      sum = fin[row][1];
      val = mine[i];
    } else {
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
    out[row * p.D + d] = Num<T>::from(mm == -CUDART_INF_F ? 0.f : val / sum);      // no key: zeros
  }
  if (splits > 1) cluster_sync_all();                             // nobody leaves while another reads its shared memory
}

template <typename T, bool Q8, int DP, int NB>
static int paged_attn_launch(const PagedAttn& p, int B, int splits, cudaStream_t stream) {
  using S = PagedShape<T, Q8, DP, NB>;
  static_assert(S::SMEM <= 231000, "shared memory budget of one CTA");
  auto kernel = paged_attn_kernel<T, Q8, DP, NB>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  static unsigned long long ready = 0;                            // one bit per device
  if (dev > 63 || !((__atomic_load_n(&ready, __ATOMIC_ACQUIRE) >> dev) & 1)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);      // sixteen
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev <= 63) __atomic_fetch_or(&ready, 1ull << dev, __ATOMIC_RELEASE);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits, p.heads * ((p.group + 8 * NB - 1) / (8 * NB)), B);
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
  if (p.group <= 8) {
    if (p.D <= 64) return paged_attn_launch<T, Q8, 64, 1>(p, B, splits, stream);
    if (p.D <= 128) return paged_attn_launch<T, Q8, 128, 1>(p, B, splits, stream);
    return paged_attn_launch<T, Q8, 256, 1>(p, B, splits, stream);
  }
  if (p.D <= 64) return paged_attn_launch<T, Q8, 64, 2>(p, B, splits, stream);
  if (p.D <= 128) return paged_attn_launch<T, Q8, 128, 2>(p, B, splits, stream);
  return paged_attn_launch<T, Q8, 256, 2>(p, B, splits, stream);
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
  if (static_cast<long long>(columns) * page > 0x7fff0000ll) return -1;      // a warp looks a batch of keys past the last one
  oslo::PagedAttn p{};
  p.q = q; p.q_sb = q_sb; p.q_sh = q_sh; p.kp = k_pages; p.vp = v_pages; p.ks = k_scale; p.vs = v_scale; p.o = o; p.table = table;
  p.lengths = lengths; p.err = err_word; p.pages = pages; p.scale = scale; p.H = H; p.heads = heads; p.group = H / heads; p.D = D;
  p.page = page; p.columns = columns; p.window = window;
  // splits of a sequence's keys (the blocks of a cluster): enough for two blocks per SM, none shorter than 64 keys of the longest possible
  // sequence; a block costs about 4 us besides its keys (512 units, 16-bit: 112 us in one part each, 122 in two, 173 in eight)
  const long long units = static_cast<long long>(B) * heads * ((p.group + 15) / 16), most = static_cast<long long>(columns) * page;
  const long long span = window > 0 && window < most ? window : most;
  int splits = 1;
  while (splits < 16 && units * splits < 2ll * num_sms && span > 64ll * splits) splits *= 2;
  p.B = B;
  p.by_length = B > 1 && B <= oslo::PA_SORTED && units * splits > 2ll * num_sms;
  if (dtype == OSLO_DT_BF16) return q8 ? oslo::paged_attn_dim<__nv_bfloat16, true>(p, B, splits, stream) : oslo::paged_attn_dim<__nv_bfloat16, false>(p, B, splits, stream);
  if (dtype == OSLO_DT_FP16) return q8 ? oslo::paged_attn_dim<__half, true>(p, B, splits, stream) : oslo::paged_attn_dim<__half, false>(p, B, splits, stream);
  return -2;
}
