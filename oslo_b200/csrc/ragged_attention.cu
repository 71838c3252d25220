// Causal attention with grouped heads over sequences of different lengths that lie one behind another, forward and backward, on the
// tcgen05 tensor cores with TMEM accumulators.
//
// Sequence b has queries offsets[b] .. offsets[b + 1] - 1 and keys key_offsets[b] .. key_offsets[b + 1] - 1; its last query stands at its
// last key: query i sees key j where j <= i + nk - nq (and j > i + nk - nq - window). Rows of no sequence, and queries that see nothing,
// get zeros. Offsets are read on the device only: a grid of the largest possible number of tiles looks its tiles up.
//
// A tile's rows are (token, head) pairs, `pack` heads of a key head's group per token (the largest power of two up to 64 that divides the
// group): one TMA box {64 columns, pack heads, rows / pack tokens} fetches them, short sequences fill tiles, and the sum over the
// group's heads in dK and dV happens in one accumulator, always in the same order.
//
//   forward  rows = queries   S = Q K^T                    P = exp2(S - m)              O += P V
//   dK, dV   rows = keys      S^T = K Q^T, dP^T = V dO^T   P^T, dS^T = P^T o (dP - delta)   dV += P^T dO, dK += dS^T Q
//   dQ       rows = queries   S = Q K^T, dP = dO V^T       dS = P o (dP - delta)        dQ += dS K
//
// P is rounded to the inputs' type for its products, since the tensor core multiplies numbers of one 16-bit type: half a step is 2^-8 of a
// weight in bf16 and 2^-11 in fp16, as for the results themselves, and two numbers a weight would double the products of P V. With that
// outputs are 1.25 to 1.4 times as far from the formula as one rounding at the end puts them. dS, a difference, goes into its products as
// two numbers of that type: rounded to one, dQ and dK were 1.5 (bf16) to 1.9 (fp16) times as far off, now 1.1 to 1.4 times; it costs 5 % of
// the backward pass with heads of 128. Maxima, sums and all accumulators are 32-bit.
//
// Not in the reference, which pads batches (oslo/models/gptj/modeling_gptj.py:151-191 is the attention of one).
#include "attention_sm100.cuh"

namespace oslo {

struct RaggedParams {
  const int* q_off; const int* k_off;
  int B, Hq, Hk, pack, pack_log, subs;      // subs: packs of heads per key head
  long long Tq, Tk;
  int D, fp16, window;
  float scale;
  void* out; long long o_sr, o_sh;          // forward: O. backward: the gradient of this launch
  void* out2; long long o2_sr, o2_sh;       // dK beside dV
  float* lse;                               // [Tq, Hq], natural logarithm
  const float2* stats;                      // backward: [Tq, Hq] of -(log-sum-exp in log2 units) and -delta
  int* err;
};

// Where the x-th tile of `rows` packed rows is. Sequences in their order, each one's last tiles first (they are the longest); the rows
// ahead of the first sequence and behind the last one are sequences without counterpart.
struct RaggedTile {
  int seq, first;                           // first packed row (within the sequence) of the tile; seq -1: no such tile
  int q0, nq, k0, nk;                       // the sequence's tokens
};
__device__ __forceinline__ int ragged_clip(int v, long long hi) { return v < 0 ? 0 : (v > hi ? static_cast<int>(hi) : v); }
// all 32 lanes of a warp
__device__ __forceinline__ RaggedTile ragged_find(const RaggedParams& p, bool key_rows, int rows, int x) {
  const int lane = threadIdx.x & 31;
  const int* off = key_rows ? p.k_off : p.q_off;
  const long long total = key_rows ? p.Tk : p.Tq;
  const int log = key_rows ? 0 : p.pack_log;
  RaggedTile t;
  t.seq = -1; t.first = 0; t.q0 = t.nq = t.k0 = t.nk = 0;
  int done = 0;
  for (int base = 0; base < p.B + 2; base += 32) {
    const int s = base + lane;
    int lo = 0, hi = 0;
    if (s < p.B) { lo = ragged_clip(off[s], total); hi = ragged_clip(off[s + 1], total); }
    else if (s == p.B) { lo = ragged_clip(off[p.B], total); hi = static_cast<int>(total); }
    else if (s == p.B + 1) { lo = 0; hi = ragged_clip(off[0], total); }
    const int n = hi > lo ? (((hi - lo) << log) + rows - 1) / rows : 0;
    int sum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, x < done + sum);
    if (hit) {
      const int w = __ffs(hit) - 1;
      const int ahead = done + __shfl_sync(0xffffffffu, sum - n, w), count = __shfl_sync(0xffffffffu, n, w);
      const int mlo = __shfl_sync(0xffffffffu, lo, w), mhi = __shfl_sync(0xffffffffu, hi, w);
      t.seq = base + w;
      t.first = (key_rows ? x - ahead : count - 1 - (x - ahead)) * rows;        // first key tiles have the most queries
      if (key_rows) { t.k0 = mlo; t.nk = mhi - mlo; } else { t.q0 = mlo; t.nq = mhi - mlo; }
      if (t.seq < p.B) {
        const int* other = key_rows ? p.q_off : p.k_off;
        const long long ot = key_rows ? p.Tq : p.Tk;
        const int a = ragged_clip(other[t.seq], ot), z = ragged_clip(other[t.seq + 1], ot);
        if (key_rows) { t.q0 = a; t.nq = max(0, z - a); } else { t.k0 = a; t.nk = max(0, z - a); }
      }
      return t;
    }
    done += __shfl_sync(0xffffffffu, sum, 31);
  }
  return t;
}

__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// two at a time: a * k + b, and a sum
__device__ __forceinline__ float2 fma2(float2 a, float k, float b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%5, %5};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(k), "f"(b));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float k, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%6, %6};\n\tmov.b64 z, {%4, %5};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(k));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2v(float2 a, float2 b, float c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %6};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {      // no number stays no number
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 2^x of two numbers up to 100 on the FMA pipe, to 2.6e-6 of its value: x = n + f with |f| <= 1/2 (n by adding 1.5 * 2^23), 2^f by a
// polynomial of degree 4 with the least largest relative error (found by reweighted least squares), times 2^n. Below -126.5 it is 0 (n is
// -127 there, whose exponent bits are those of 0), so what a mask hides weighs nothing; what is no number stays so through the polynomial,
// whatever 2^n its bits make. 2.6e-6 is less than a hundredth of what rounding the weight to fp16 changes next (2^-11), and changes the sum
// of weights by no more than that share.
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  x.x = max_nan(x.x, -127.f);
  x.y = max_nan(x.y, -127.f);
  const float2 t = fma2(x, 1.f, 12582912.f), n = fma2(t, 1.f, -12582912.f), f = fma2v(n, make_float2(-1.f, -1.f), 0.f);
  const float2 g = make_float2(x.x + f.x, x.y + f.y);
  float2 e = fma2(g, 0.009570101698774808f, 0.05591786030272724f);
  e = fma2v(e, g, 0.24024744833108522f);
  e = fma2v(e, g, 0.6931218147397942f);
  e = fma2v(e, g, 0.999999261444132f);
  return mul2(e, make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u)));
}
// a and b as 16-bit values and what those lack, as 16-bit values too: together 16 (bf16) or 22 (fp16) bits of them
template <bool F16> __device__ __forceinline__ void split2(float2 a, uint32_t& hi, uint32_t& lo) {
  float2 h;
  if (F16) {
    hi = fa_pack2(a.x, a.y, true);
    h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  } else {                                          // cut off, not rounded: a byte permutation
    const uint32_t x = __float_as_uint(a.x), y = __float_as_uint(a.y);
    hi = __byte_perm(x, y, 0x7632);
    h = make_float2(__uint_as_float(x & 0xffff0000u), __uint_as_float(y & 0xffff0000u));
  }
  a = fma2(h, -1.f, a);
  lo = fa_pack2(a.x, a.y, F16);
}
__device__ __forceinline__ void ragged_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int col, int head, int row) {
  tma_load_3d(dst, map, bar, col, head, row);
}
// Rows [from, rows) of a tile of `subs` sub-tiles [rows x 128 bytes] become zeros: they belong to other sequences, and what they hold
// (no numbers, infinities) must not meet a weight of zero in a product. One warp; the tile has arrived.
__device__ __forceinline__ void ragged_wipe(uint32_t tile, int from, int rows, int subs) {
  const int lane = threadIdx.x & 31, pieces = (rows - from) * 8;
  for (int c = 0; c < subs; ++c)
    for (int i = lane; i < pieces; i += 32)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + c * rows * 128 + from * 128 + i * 16), "r"(0) : "memory");
  fence_proxy_async_smem();
  __syncwarp();
}
// Lanes 0-31 of the calling warp's TMEM quarter hold a row each: columns [from, to) of its accumulator (zeros where `empty`), times
// `mult`, into a row of the result (D columns; `live` rows only). 32 columns of 32 rows pass through `stage`, 2 KB of shared memory that
// nothing else uses any more, so that four lanes write 64 bytes of a row and eight rows are met at a time (a lane a row met 32, at 5000
// cycles a tile of 128 columns). Piece c of row r lies at c ^ (r / 2 % 4), which keeps both directions free of bank conflicts. CHECK: whether
// a value of this lane's row is infinite or no number.
template <bool CHECK = false>
__device__ __forceinline__ bool ragged_store(uint32_t acc, int from, int to, bool filled, bool empty, float mult, uint16_t* row, int D, bool live,
                                             bool fp16, uint32_t stage) {
  if (!filled) {                            // no products, perhaps with copies on their way to where the stage is
    if (live)
      for (int c = from; c < to && c < D; c += 8) *reinterpret_cast<uint4*>(row + c) = make_uint4(0, 0, 0, 0);
    return false;
  }
  bool odd = false;
  const int lane = threadIdx.x & 31;
  const uint32_t alive = __ballot_sync(0xffffffffu, live);
#pragma unroll 1
  for (int c0 = from; c0 < to; c0 += 32) {
    uint32_t r[32];
    tmem_ld_32x32(acc + c0, r);
    tmem_wait_ld();
    if (empty) {
#pragma unroll
      for (int i = 0; i < 32; ++i) r[i] = 0u;
    }
    if (CHECK) {
#pragma unroll
      for (int i = 0; i < 32; ++i) odd |= (r[i] & 0x7f800000u) == 0x7f800000u;
    }
    __syncwarp();                           // the columns before these have been read
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = fa_pack2(__uint_as_float(r[8 * c + 2 * i]) * mult, __uint_as_float(r[8 * c + 2 * i + 1]) * mult, fp16);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 64 + ((c ^ (lane >> 1 & 3)) << 4)), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                   "r"(v[3]) : "memory");
    }
    __syncwarp();
    const int c = lane & 3, col = c0 + 8 * c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 8 * i + (lane >> 2);   // the row this lane writes a piece of
      uint16_t* out = reinterpret_cast<uint16_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), at));
      uint4 v;
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(stage + at * 64 + ((c ^ (at >> 1 & 3)) << 4))
                   : "memory");
      if ((alive >> at & 1u) && col < D) *reinterpret_cast<uint4*>(out + col) = v;
    }
  }
  return odd;
}

// ---------------------------------------------------------------------------------------------------------------- forward
// MT tiles of 128 rows per CTA. D <= 128: two, with a softmax warpgroup each (thread = row), so that the tensor core works for one tile
// while the other's exponentials run. S of two blocks of 64 keys per tile: Q K^T of the next block runs under the softmax of this one (with
// blocks of 128 keys TMEM holds one S a tile; its Q K^T then waited for P V: 350 us instead of 298 for 2 x 4096 tokens, 32/8 heads of
// 128, which take 261 since the results pass through shared memory). P overwrites S. Warp 0: TMA; a warp a tile issues its products; then a warpgroup a tile for the softmax. A wait that is over at once
// still takes 100 to 200 cycles and a commit not much less, so an issuer has two of each a block: K of the next block and V of this one
// share a stage (with one warp for both tiles and five waits and commits a tile: 449 us).
template <int DP> struct RaggedFwd {
  static constexpr int MT = DP <= 128 ? 2 : 1, BN = 64;
  static constexpr int FIRST = 1 + MT, THREADS = 32 * (FIRST + 4 * MT), ROWS = 128 * MT;      // FIRST: the first softmax warp
  static constexpr int DC = DP / 64;
  // of 8 pairs of exponentials, those that the FMA pipe computes: 16 a clock come from the special function unit, half of a block's time.
  // 0, 1, 2, 3 of 8, 2 x 4096 tokens, 32/8 heads: 268, 285, 261, 271 us for heads of 128, 264, 263, 254, 253 for 64; 0 and 2 of 8: 498, 510
  // for 256 (one tile: its products wait for its softmax, and the polynomial's longer chain shows)
  static constexpr int FMA_EXP = DP <= 128 ? 2 : 0;
  static constexpr uint32_t Q_SUB = 128 * 128, Q_TILE = DC * Q_SUB, KV_SUB = BN * 128, KV_TILE = DC * KV_SUB;
  static constexpr int STAGES = DP == 256 ? 2 : (DP == 128 ? 4 : 6);       // of K of block j + 1 and V of block j
  static constexpr uint32_t S_COL = 0, O_COL = 256;                // S: tile i, buffer b at (2 i + b) BN
  static_assert(2 * MT * BN <= 256 && MT * DP <= 256, "TMEM budget");
  static constexpr uint32_t TILES = MT * Q_TILE + (1 + 2 * STAGES) * KV_TILE;
  static constexpr int B_Q = 0, B_F = 1, B_E = B_F + STAGES, B_S = B_E + STAGES, B_P = B_S + 4, B_O = B_P + 4, B_W = B_O + 2,
                       BARS = B_W + 1;                             // B_Q: Q and the first K; B_S, B_P: 2 tile + buffer; B_W: rows wiped
  static constexpr uint32_t SMEM = TILES + BARS * 8 + 64 + 1024;
};

// F16: the inputs are fp16 (a branch at every packed pair otherwise)
template <int DP, bool F16>
__global__ void __launch_bounds__(RaggedFwd<DP>::THREADS, 1)
ragged_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                  const RaggedParams p) {
  using F = RaggedFwd<DP>;
  constexpr int BN = F::BN, MT = F::MT, DC = F::DC, ST = F::STAGES;
  extern __shared__ uint8_t ragged_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ragged_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t q_s = smem_u32(smem), kv_s = q_s + MT * F::Q_TILE;       // K of block 0, then the stages
  auto k_at = [&](int j) { return j == 0 ? kv_s : kv_s + (1 + 2 * ((j - 1) % ST)) * F::KV_TILE; };
  auto v_at = [&](int j) { return kv_s + (2 + 2 * (j % ST)) * F::KV_TILE; };
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + F::TILES);
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * i; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + F::BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  RaggedTile* found = reinterpret_cast<RaggedTile*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = blockIdx.y / p.subs, h0 = hk * (p.Hq / p.Hk) + blockIdx.y % p.subs * p.pack;
  if (warp == 0) {
    const RaggedTile t = ragged_find(p, false, F::ROWS, blockIdx.x);
    if (lane == 0) *found = t;
  }
  if (threadIdx.x == 32) {
    // four softmax warps hand over a P; every tile's issuer gives a stage back
    for (int i = 0; i < F::BARS; ++i)
      mbar_init(bar(i), i >= F::B_P && i < F::B_P + 4 ? 4 : (i >= F::B_E && i < F::B_S ? MT : 1));
    *abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  const RaggedTile t = *found;
  if (t.seq < 0) return;                                            // the whole block
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // ---- which blocks of keys: from `lo` (both tiles), n[i] of them for tile i
  const int offset = t.nk - t.nq, rows = t.nq << p.pack_log;
  const int tok0 = t.first >> p.pack_log;
  const int lo = p.window > 0 ? max(0, tok0 + offset - p.window + 1) / BN * BN : 0;
  int n[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int first = t.first + i * 128;
    if (first < rows) {
      const int last_tok = (min(rows, first + 128) - 1) >> p.pack_log;
      const int hi = min(t.nk, last_tok + offset + 1);
      n[i] = hi > lo ? (hi - lo + BN - 1) / BN : 0;
    }
  }
  const int blocks = max(n[0], n[1]), tail = t.nk - (lo + (blocks - 1) * BN);      // tail: keys of the sequence in the last block

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    int ok = blocks > 0;
    if (lane == 0 && blocks > 0) {
      tma_prefetch_desc(&tq); tma_prefetch_desc(&tk); tma_prefetch_desc(&tv);
      mbar_expect_tx(bar(F::B_Q), MT * F::Q_TILE + F::KV_TILE);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int c = 0; c < DC; ++c)
          ragged_load(q_s + i * F::Q_TILE + c * F::Q_SUB, &tq, bar(F::B_Q), c * 64, h0, t.q0 + ((t.first + i * 128) >> p.pack_log));
#pragma unroll
      for (int c = 0; c < DC; ++c) ragged_load(kv_s + c * F::KV_SUB, &tk, bar(F::B_Q), c * 64, hk, t.k0 + lo);
      for (int j = 0; j < blocks && ok; ++j) {
        const int st = j % ST, row = t.k0 + lo + j * BN;
        ok = mbar_wait(bar(F::B_E + st), ((j / ST) & 1) ^ 1, abort_flag, p.err, ERR_WAIT_EMPTY);
        if (!ok) break;
        mbar_expect_tx(bar(F::B_F + st), j + 1 < blocks ? 2 * F::KV_TILE : F::KV_TILE);
        if (j + 1 < blocks) {
#pragma unroll
          for (int c = 0; c < DC; ++c) ragged_load(k_at(j + 1) + c * F::KV_SUB, &tk, bar(F::B_F + st), c * 64, hk, row + BN);
        }
#pragma unroll
        for (int c = 0; c < DC; ++c) ragged_load(v_at(j) + c * F::KV_SUB, &tv, bar(F::B_F + st), c * 64, hk, row);
      }
    }
    ok = __shfl_sync(0xffffffffu, ok, 0);
    if (ok && tail < BN) {                  // the last block's values of other sequences
      const int j = blocks - 1;
      if (mbar_wait_warp(bar(F::B_F + j % ST), (j / ST) & 1, abort_flag, p.err, ERR_WAIT_FULL)) {
        ragged_wipe(v_at(j), tail, BN, DC);
        if (lane == 0) mbar_arrive(bar(F::B_W));
      }
    }
  } else if (warp <= MT) {
    // ------------------------------------------------------------------ MMA issuer of a tile: the whole warp runs the loop, so that
    // addresses and descriptors are uniform; one lane issues
    const int i = warp - 1;
    if (blocks > 0) {
      constexpr int fmt = F16 ? 0 : 1;
      const uint32_t idesc_qk = make_idesc_f16(128, BN, fmt, 0, 0), idesc_pv = make_idesc_f16(128, DP, fmt, 0, 1);
      const uint64_t desc_k = make_smem_desc(0, 16, 1024), desc_v = make_smem_desc(0, F::KV_SUB, 1024);      // plus (address >> 4)
      const bool issuer = elect_one();
      auto wait = [&](int b, uint32_t parity) { return mbar_wait_warp(bar(b), parity, abort_flag, p.err, ERR_WAIT_FULL); };
      auto qk = [&](int j) {
        const uint64_t da = desc_k + ((q_s + i * F::Q_TILE) >> 4), db = desc_k + (k_at(j) >> 4);
        const uint32_t dst = tmem + F::S_COL + (2 * i + (j & 1)) * BN;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
          umma_f16(dst, da + (((kk >> 2) * F::Q_SUB + (kk & 3) * 32) >> 4), db + (((kk >> 2) * F::KV_SUB + (kk & 3) * 32) >> 4), idesc_qk, kk != 0);
      };
      bool ok = wait(F::B_Q, 0);
      tc_fence_after();
      if (ok && n[i] > 0 && issuer) {
        qk(0);
        umma_commit(bar(F::B_S + 2 * i));
      }
      __syncwarp();
      for (int j = 0; j < n[i]; ++j) {
        const int st = j % ST, buf = 2 * i + (j & 1);
        ok = wait(F::B_F + st, (j / ST) & 1);
        if (!ok) break;
        tc_fence_after();
        if (issuer) {
          // S of block j + 1 takes the place of P of block j - 1, whose product was issued before: those of one thread run in order.
          // The commit, also without a block j + 1, says that O holds block j - 1.
          if (j + 1 < n[i]) qk(j + 1);
          umma_commit(bar(F::B_S + (buf ^ 1)));
        }
        __syncwarp();
        ok = (j + 1 < blocks || tail >= BN || wait(F::B_W, 0)) && wait(F::B_P + buf, (j >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        if (issuer) {
          const uint64_t db = desc_v + (v_at(j) >> 4);
          const uint32_t src = tmem + F::S_COL + buf * BN;
#pragma unroll
          for (int ks = 0; ks < BN / 16; ++ks) umma_f16_ts(tmem + F::O_COL + i * DP, src + ks * 8, db + ks * 128, idesc_pv, (j | ks) != 0);
          umma_commit(bar(F::B_E + st));
          if (j + 1 == n[i]) umma_commit(bar(F::B_O + i));
        }
        __syncwarp();
      }
      // blocks that only the other tile needs: given back as they come (not before: an arrival belongs to its own round)
      for (int j = n[i]; j < blocks && ok; ++j) {
        ok = wait(F::B_F + j % ST, (j / ST) & 1);
        if (ok && issuer) mbar_arrive(bar(F::B_E + j % ST));
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax: thread = row
    const int i = (warp - F::FIRST) >> 2, quad = warp & 3;
    const int r = t.first + i * 128 + quad * 32 + lane, tok = r >> p.pack_log, head = h0 + (r & (p.pack - 1));
    const bool live = r < rows;
    const uint32_t lane_at = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t o_at = lane_at + F::O_COL + i * DP;
    const float sc = p.scale * FA_LOG2E;
    constexpr bool fp16 = F16;
    const int last = min(t.nk - 1, tok + offset), first = p.window > 0 ? tok + offset - p.window + 1 : 0;
    const int first_tok = (t.first + i * 128) >> p.pack_log, last_tok = (t.first + i * 128 + 127) >> p.pack_log;
    float m = -CUDART_INF_F, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n[i]; ++j) {
      const int buf = 2 * i + (j & 1), n0 = lo + j * BN;
      ok = mbar_wait_warp(bar(F::B_S + buf), (j >> 1) & 1, abort_flag, p.err, ERR_WAIT_TMEM_FULL);
      if (!ok) break;
      tc_fence_after();
      const uint32_t s_at = lane_at + F::S_COL + buf * BN;
      uint32_t x[BN / 32][32];
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) tmem_ld_32x32(s_at + c * 32, x[c]);
      tmem_wait_ld();
      auto s = [&](int c) -> float { return __uint_as_float(x[c >> 5][c & 31]); };
      // only blocks that reach past the diagonal, the window's edge or the keys' end of some row
      if (n0 + BN > min(t.nk, first_tok + offset + 1) || (p.window > 0 && n0 <= last_tok + offset - p.window)) {
        auto below = [](int k) { return k <= 0 ? 0u : (k >= 32 ? 0xffffffffu : (1u << k) - 1u); };
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) {
          const uint32_t vis = below(last - (n0 + c * 32) + 1) & ~below(first - (n0 + c * 32));
#pragma unroll
          for (int u = 0; u < 32; ++u)
            if (!((vis >> u) & 1u)) x[c][u] = 0xff800000u;
        }
      }
      float mx4[4] = {s(0), s(1), s(2), s(3)};
#pragma unroll
      for (int c = 4; c + 8 <= BN; c += 8) {
#pragma unroll
        for (int u = 0; u < 4; ++u) mx4[u] = max3(mx4[u], s(c + u), s(c + 4 + u));
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) mx4[u] = fmaxf(mx4[u], s(BN - 4 + u));
      const float mx = fmaxf(max3(mx4[0], mx4[1], mx4[2]), mx4[3]) * sc, m_new = fmaxf(m, mx);
      // O is multiplied only when a row of this warp has outgrown its reference by 2^8
      if (__any_sync(0xffffffffu, j == 0 || m_new - m > 8.f)) {
        const float factor = m == -CUDART_INF_F ? 0.f : exp2f(m - m_new);
        m = m_new;
        l *= factor;
        if (j > 0) {
          // O holds block j - 1 as soon as S of block j + 1 is there
          ok = mbar_wait_warp(bar(F::B_S + (buf ^ 1)), ((j + 1) >> 1) & 1, abort_flag, p.err, ERR_WAIT_TMEM_FULL);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c0 = 0; c0 < DP; c0 += 32) {
            uint32_t y[32];
            tmem_ld_32x32(o_at + c0, y);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c) y[c] = __float_as_uint(__uint_as_float(y[c]) * factor);
            tmem_st_32x32(o_at + c0, y);
          }
          tmem_wait_st();
        }
      }
      const float base = m == -CUDART_INF_F ? 0.f : -m;
      float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          float2 e = fma2(make_float2(__uint_as_float(x[c][2 * u]), __uint_as_float(x[c][2 * u + 1])), sc, base);
          if (u % 8 < F::FMA_EXP) {
            e = exp2_fma(e);
          } else {
            e.x = exp2f(e.x);
            e.y = exp2f(e.y);
          }
          sum2[u & 1] = add2(sum2[u & 1], e);
          w[u] = fa_pack2(e.x, e.y, fp16);
        }
        tmem_st_32x16(s_at + c * 16, w);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(F::B_P + buf));
      l += (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
    }
    if (ok && n[i] > 0) {
      ok = mbar_wait_warp(bar(F::B_O + i), 0, abort_flag, p.err, ERR_WAIT_TMEM_FULL);
      tc_fence_after();
    }
    const long long at = t.q0 + tok;
    const bool seen = ok && n[i] > 0 && live && last >= first && last >= 0;      // a query that sees no key: zeros
    uint16_t* orow = reinterpret_cast<uint16_t*>(p.out) + at * p.o_sr + head * p.o_sh;
    ragged_store(o_at, 0, DP, ok && n[i] > 0, !seen, seen ? 1.f / l : 0.f, orow, p.D, live, fp16, q_s + i * F::Q_TILE + quad * 2048);
    if (live && p.lse) p.lse[at * p.Hq + head] = seen ? (m + log2f(l)) * FA_LN2 : 0.f;
  }

  if (*abort_flag) {                        // copies in flight land before the shared memory is given back
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------------------------- backward
// What the other kernels need of a query row: its log-sum-exp in log2 units and delta[t, h] = sum_d dO O in 32 bits, negative, side by side; DP / 8
// lanes a row. Bound by reading both. O is the rounded output: that moves delta by up to half a step of each term (2^-8 in bf16, 2^-11 in fp16),
// as it moves everything else that is made of the output; an output in 32 bits kept for this would double what the forward pass writes.
template <typename T, int LPR>
__global__ void __launch_bounds__(256) ragged_delta_kernel(const T* __restrict__ o, const T* __restrict__ g, const float* __restrict__ lse,
                                                           float2* __restrict__ stats, long long rows, int H, int D, long long o_sr, long long o_sh, long long g_sr,
                                                           long long g_sh) {
  const long long row = static_cast<long long>(blockIdx.x) * (256 / LPR) + threadIdx.x / LPR;
  const int d = threadIdx.x % LPR * 8;
  float acc = 0.f;
  if (row < rows && d < D) {
    const long long t = row / H, h = row % H;
    const uint4 a = *reinterpret_cast<const uint4*>(o + t * o_sr + h * o_sh + d), b = *reinterpret_cast<const uint4*>(g + t * g_sr + h * g_sh + d);
    const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 u, v;
      if constexpr (std::is_same<T, __half>::value) {
        u = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
        v = __half22float2(*reinterpret_cast<const __half2*>(&y[i]));
      } else {
        u = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x[i]));
        v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&y[i]));
      }
      acc += u.x * v.x + u.y * v.y;
    }
  }
#pragma unroll
  for (int s = LPR / 2; s > 0; s >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, s);
  if (row < rows && d == 0) stats[row] = make_float2(-lse[row] * FA_LOG2E, -acc);
}

enum : int { RB_DKV = 0, RB_DV = 1, RB_DK = 2, RB_DQ = 3 };

// 128 resident rows (TMEM lane = row), blocks of 64 streamed columns. S and dP of two blocks in TMEM; two warpgroups transform one half
// of the columns each: P and dS go back, packed, into the half they came from. Head sizes of 256 take dV and dK in two launches: both
// accumulators fill TMEM alone. r1, s1: what S is made of; r2, s2: what dP (and dV) is made of.
//
// 2 x 4096 tokens, 32/8 heads: 1338 us with heads of 128, 993 with 64, 3290 with 256 (a block of dK and dV takes 2240 cycles with 128, of
// which its products need 1540: S and dP have 64 columns, which the tensor core takes at three quarters of its rate, since both
// operands come from shared memory). Per block one wait and one commit fewer (JOINT), the statistics brought by a warp of their own and a
// uniform test for blocks without a mask: 1278 instead of 1450, before dS became two numbers. Exponentials on the FMA pipe do not pay here (1408 instead of 1363): the
// transform is bound by its instructions, which is why two values at a time are multiplied and added.
template <int DP, int MODE> struct RaggedBwd {
  static constexpr bool KEY_ROWS = MODE != RB_DQ, DPROD = MODE != RB_DV;        // DPROD: dP is needed
  static constexpr int BN = 64, DC = DP / 64, THREADS = 64 + 256 + (KEY_ROWS ? 32 : 0), NST = DP == 256 ? 2 : 4;    // NST: blocks of statistics
  static constexpr uint32_t R_SUB = 128 * 128, R_TILE = DC * R_SUB, C_SUB = BN * 128, C_TILE = DC * C_SUB;
  static constexpr int NRES = DPROD ? 2 : 1;
  // a copy takes longer than a block's products: as many blocks ahead as there is room for. JOINT: both operands of a block share a stage,
  // which saves the issuer waits and commits (100 to 200 cycles each)
  static constexpr bool JOINT = DP < 256;
  static constexpr int S1 = DP == 256 ? 2 : (DP == 128 ? 4 : 6), S2 = DP == 256 ? (MODE == RB_DV ? 2 : 1) : S1;
  static constexpr uint32_t STATS = KEY_ROWS ? NST * BN * 8 : 0;
  static constexpr uint32_t TILES = NRES * R_TILE + (S1 + S2) * C_TILE;
  static constexpr uint32_t S_COL = 0, DP_COL = 2 * BN, ACC = 4 * BN, ACC2 = ACC + DP;      // ACC2: dK beside dV
  static_assert((MODE == RB_DKV ? ACC2 : ACC) + DP <= 512, "TMEM budget");
  static constexpr int B_R = 0, B_1F = 1, B_1E = B_1F + S1, B_2F = B_1E + S1, B_2E = B_2F + S2, B_SP = B_2E + S2, B_TR = B_SP + 2,
                       B_ST = B_TR + 2, B_SE = B_ST + NST, B_ACC = B_SE + NST, BARS = B_ACC + 1;
  static constexpr uint32_t SMEM = TILES + STATS + BARS * 8 + 64 + 1024;
};

// fp16: dS may be beyond the type (65504) where dQ and dK are not. A tile whose accumulator has rows that are infinite or no number runs a
// second time, with dS times 2^-26 (|dP| and |delta| are at most 256 * 65504^2 < 2^40), and writes those rows only. A weight is then off by up
// to 2, against a largest one of more than 65504. Loss-scaled training gets there; others pay a look at each row's results.
__device__ __forceinline__ void mbar_inval(uint32_t bar) { asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }

template <int DP, int MODE, bool F16>
__global__ void __launch_bounds__(RaggedBwd<DP, MODE>::THREADS, 1)
ragged_bwd_kernel(const __grid_constant__ CUtensorMap tr1, const __grid_constant__ CUtensorMap tr2, const __grid_constant__ CUtensorMap ts1,
                  const __grid_constant__ CUtensorMap ts2, const RaggedParams p) {
  using F = RaggedBwd<DP, MODE>;
  constexpr int BN = F::BN, DC = F::DC;
  constexpr bool KEY_ROWS = F::KEY_ROWS;
  extern __shared__ uint8_t ragged_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ragged_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t r1_s = smem_u32(smem), r2_s = r1_s + F::R_TILE, s1_s = r1_s + F::NRES * F::R_TILE, s2_s = s1_s + F::S1 * F::C_TILE;
  float2* stats = reinterpret_cast<float2*>(smem + F::TILES);      // [NST blocks][BN]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + F::TILES + F::STATS);
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * i; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + F::BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  RaggedTile* found = reinterpret_cast<RaggedTile*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = p.Hq / p.Hk;
  const int hk = KEY_ROWS ? blockIdx.y : blockIdx.y / p.subs, sub0 = KEY_ROWS ? 0 : blockIdx.y % p.subs;
  if (warp == 0) {
    const RaggedTile t = ragged_find(p, KEY_ROWS, 128, blockIdx.x);
    if (lane == 0) *found = t;
  }
  auto init_barriers = [&]() {
    for (int i = 0; i < F::BARS; ++i) mbar_init(bar(i), (i >= F::B_TR && i < F::B_TR + 2) || (i >= F::B_SE && i < F::B_SE + F::NST) ? 8 : 1);
    fence_barrier_init();
  };
  if (threadIdx.x == 32) {
    *abort_flag = 0;
    init_barriers();
  }
  __syncthreads();
  const RaggedTile t = *found;
  if (t.seq < 0) return;                                            // the whole block
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // ---- the streamed columns: packed queries (for each pack of the group's heads in turn), or keys
  const int offset = t.nk - t.nq, rows = t.nq << p.pack_log;
  int c_lo = 0, c_hi;
  if (KEY_ROWS) {
    c_hi = rows;
    c_lo = (max(0, t.first - offset) << p.pack_log) / BN * BN;
    // as long long: a window may be as wide as it likes
    if (p.window > 0) c_hi = static_cast<int>(min(static_cast<long long>(rows), max(0ll, static_cast<long long>(t.first) + 127 - offset + p.window) << p.pack_log));
  } else {
    const int last_tok = (min(rows, t.first + 128) - 1) >> p.pack_log;
    c_hi = min(t.nk, last_tok + offset + 1);
    if (p.window > 0) c_lo = max(0, (t.first >> p.pack_log) + offset - p.window + 1) / BN * BN;
  }
  const int per = c_hi > c_lo && t.nq > 0 && t.nk > 0 ? (c_hi - c_lo + BN - 1) / BN : 0, blocks = KEY_ROWS ? per * p.subs : per;
  const int end = KEY_ROWS ? rows : t.nk;                           // columns from here on are of other sequences
  auto column = [&](int j) { return c_lo + (KEY_ROWS ? j % per : j) * BN; };
  auto heads_of = [&](int j) { return hk * group + (KEY_ROWS ? j / per : sub0) * p.pack; };

  constexpr bool AGAIN = F16 && F::DPROD;                           // the tile may run a second time
  float lift = 1.f;                                                 // what dS is multiplied by
  bool odd = false;                                                 // a row whose result was no number the first time
#pragma unroll 1
  for (int turn = 0;; ++turn) {
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0 && blocks > 0) {
      const int row = KEY_ROWS ? t.k0 + t.first : t.q0 + (t.first >> p.pack_log), rh = KEY_ROWS ? hk : heads_of(0);
      tma_prefetch_desc(&tr1); tma_prefetch_desc(&tr2); tma_prefetch_desc(&ts1); tma_prefetch_desc(&ts2);
      mbar_expect_tx(bar(F::B_R), F::NRES * F::R_TILE);
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        ragged_load(r1_s + c * F::R_SUB, &tr1, bar(F::B_R), c * 64, rh, row);
        if (F::DPROD) ragged_load(r2_s + c * F::R_SUB, &tr2, bar(F::B_R), c * 64, rh, row);
      }
      bool ok = true;
      for (int j = 0; j < blocks && ok; ++j) {
        const int c0 = column(j), ch = KEY_ROWS ? heads_of(j) : hk, cr = KEY_ROWS ? t.q0 + (c0 >> p.pack_log) : t.k0 + c0;
        const int st1 = j % F::S1, st2 = j % F::S2;
        auto load = [&](const CUtensorMap* map, uint32_t dst, int full, int empty, uint32_t ph) -> bool {
          if (!mbar_wait(bar(empty), ph ^ 1, abort_flag, p.err, ERR_WAIT_EMPTY)) return false;
          mbar_expect_tx(bar(full), F::C_TILE);
#pragma unroll
          for (int c = 0; c < DC; ++c) ragged_load(dst + c * F::C_SUB, map, bar(full), c * 64, ch, cr);
          return true;
        };
        if (F::JOINT) {
          ok = mbar_wait(bar(F::B_1E + st1), ((j / F::S1) & 1) ^ 1, abort_flag, p.err, ERR_WAIT_EMPTY);
          if (!ok) break;
          mbar_expect_tx(bar(F::B_1F + st1), 2 * F::C_TILE);
#pragma unroll
          for (int c = 0; c < DC; ++c) {
            ragged_load(s2_s + st1 * F::C_TILE + c * F::C_SUB, &ts2, bar(F::B_1F + st1), c * 64, ch, cr);
            ragged_load(s1_s + st1 * F::C_TILE + c * F::C_SUB, &ts1, bar(F::B_1F + st1), c * 64, ch, cr);
          }
        } else {
          ok = load(&ts2, s2_s + st2 * F::C_TILE, F::B_2F + st2, F::B_2E + st2, (j / F::S2) & 1) &&
               load(&ts1, s1_s + st1 * F::C_TILE, F::B_1F + st1, F::B_1E + st1, (j / F::S1) & 1);
        }
      }
    }
  } else if (KEY_ROWS && warp == 10) {
    // ------------------------------------------------------------------ statistics of the columns, two a lane
    auto fetch = [&](int j, float2 (&v)[2]) {
      const int c0 = column(j), ch = heads_of(j);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int c = c0 + lane * 2 + u;
        v[u] = c < rows ? p.stats[static_cast<long long>(t.q0 + (c >> p.pack_log)) * p.Hq + ch + (c & (p.pack - 1))] : make_float2(0.f, 0.f);
      }
    };
    float2 now[2], next[2];
    if (blocks > 0) fetch(0, now);
    for (int j = 0; j < blocks; ++j) {
      if (j + 1 < blocks) fetch(j + 1, next);
      const int st = j % F::NST;
      if (!mbar_wait_warp(bar(F::B_SE + st), ((j / F::NST) & 1) ^ 1, abort_flag, p.err, ERR_WAIT_EMPTY)) break;
      *reinterpret_cast<float4*>(stats + st * BN + lane * 2) = make_float4(now[0].x, now[1].x, AGAIN ? now[0].y * lift : now[0].y, AGAIN ? now[1].y * lift : now[1].y);
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(F::B_ST + st));
      now[0] = next[0];
      now[1] = next[1];
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer: the whole warp runs the loops, one lane issues
    if (blocks > 0) {
      constexpr int fmt = F16 ? 0 : 1;
      const uint32_t idesc_1 = make_idesc_f16(128, BN, fmt, 0, 0), idesc_2 = make_idesc_f16(128, DP, fmt, 0, 1);
      const uint64_t desc_1 = make_smem_desc(0, 16, 1024), desc_2 = make_smem_desc(0, F::C_SUB, 1024);        // plus (address >> 4)
      const bool issuer = elect_one();
      auto wait = [&](int b, uint32_t parity) { return mbar_wait_warp(bar(b), parity, abort_flag, p.err, ERR_WAIT_FULL); };
      auto product = [&](uint32_t dst, uint32_t res, uint32_t tile) {
        const uint64_t da = desc_1 + (res >> 4), db = desc_1 + (tile >> 4);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
          umma_f16(dst, da + (((kk >> 2) * F::R_SUB + (kk & 3) * 32) >> 4), db + (((kk >> 2) * F::C_SUB + (kk & 3) * 32) >> 4), idesc_1, kk != 0);
      };
      // 16 columns a step; each half of the 64 columns has its packed values at its own first columns
      auto second = [&](uint32_t acc, uint32_t src, uint32_t tile, bool more) {
        const uint64_t db = desc_2 + (tile >> 4);
#pragma unroll
        for (int ks = 0; ks < BN / 16; ++ks) umma_f16_ts(acc, src + (ks >> 1) * 32 + (ks & 1) * 8, db + ks * 128, idesc_2, more || ks != 0);
      };
      bool ok = wait(F::B_R, 0);
      auto first_stage = [&](int j) -> bool {
        const int buf = j & 1, st1 = j % F::S1, st2 = j % F::S2, left = end - column(j);
        const uint32_t t1 = s1_s + st1 * F::C_TILE, t2 = s2_s + st2 * F::C_TILE;
        if (!wait((F::JOINT ? F::B_1F + st1 : F::B_2F + st2), F::JOINT ? (j / F::S1) & 1 : (j / F::S2) & 1)) return false;
        if (left < BN && KEY_ROWS) ragged_wipe(t2, left, BN, DC);
        if (F::JOINT && left < BN) ragged_wipe(t1, left, BN, DC);
        tc_fence_after();
        if (F::DPROD && issuer) {
          product(tmem + F::DP_COL + buf * BN, r2_s, t2);
          if (!F::JOINT) umma_commit(bar(F::B_2E + st2));
        }
        if (!F::JOINT) {
          if (!wait(F::B_1F + st1, (j / F::S1) & 1)) return false;
          if (left < BN) ragged_wipe(t1, left, BN, DC);
          tc_fence_after();
        }
        if (issuer) {
          product(tmem + F::S_COL + buf * BN, r1_s, t1);
          if (MODE == RB_DV) umma_commit(bar(F::B_1E + st1));
          umma_commit(bar(F::B_SP + buf));
        }
        __syncwarp();
        return true;
      };
      if (ok) ok = first_stage(0);
      for (int j = 0; j < blocks && ok; ++j) {
        if (j + 1 < blocks) {
          ok = first_stage(j + 1);
          if (!ok) break;
        }
        const int buf = j & 1, st1 = j % F::S1, st2 = j % F::S2;
        ok = wait(F::B_TR + buf, (j >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        if (issuer) {
          if (MODE == RB_DKV || MODE == RB_DV) {
            second(tmem + F::ACC, tmem + F::S_COL + buf * BN, s2_s + st2 * F::C_TILE, j != 0);
            if (!F::JOINT) umma_commit(bar(F::B_2E + st2));
          }
          if (F::DPROD) {
            second(tmem + (MODE == RB_DKV ? F::ACC2 : F::ACC), tmem + F::DP_COL + buf * BN, s1_s + st1 * F::C_TILE, j != 0);
            second(tmem + (MODE == RB_DKV ? F::ACC2 : F::ACC), tmem + F::DP_COL + buf * BN + 16, s1_s + st1 * F::C_TILE, true);
            umma_commit(bar(F::B_1E + st1));
          }
          if (j + 1 == blocks) umma_commit(bar(F::B_ACC));
        }
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------------ transform: thread = resident row, one half of the columns
    const int half = (warp - 2) >> 2, quad = warp & 3, r = t.first + quad * 32 + lane;
    const uint32_t lane_at = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const float sc = p.scale * FA_LOG2E;
    constexpr bool fp16 = F16;
    const bool live = KEY_ROWS ? r < t.nk : r < rows;
    const int tok = KEY_ROWS ? 0 : r >> p.pack_log, head = KEY_ROWS ? hk : heads_of(0) + (r & (p.pack - 1));
    // columns that every row of the tile meets: from plain_lo up to plain_hi
    int plain_lo, plain_hi;
    if (KEY_ROWS) {
      plain_lo = max(0, t.first + 127 - offset) << p.pack_log;
      plain_hi = p.window > 0 ? static_cast<int>(min(static_cast<long long>(rows), max(0ll, static_cast<long long>(t.first) - offset + p.window) << p.pack_log)) : rows;
    } else {
      plain_hi = min(t.nk, (t.first >> p.pack_log) + offset + 1);
      plain_lo = p.window > 0 ? max(0, ((t.first + 127) >> p.pack_log) + offset - p.window + 1) : 0;
    }
    float2 own = make_float2(0.f, 0.f);
    if (!KEY_ROWS && live) own = p.stats[static_cast<long long>(t.q0 + tok) * p.Hq + head];
    if (AGAIN) own.y *= lift;
    bool ok = true;
    for (int j = 0; j < blocks && ok; ++j) {
      const int buf = j & 1, b0 = column(j), c0 = b0 + half * 32, st = j % F::NST;
      float4 col[KEY_ROWS ? 16 : 1];                // statistics of this half's columns, two columns a piece, while the products run
      if (KEY_ROWS) {
        ok = mbar_wait_warp(bar(F::B_ST + st), (j / F::NST) & 1, abort_flag, p.err, ERR_WAIT_FULL);
        if (!ok) break;
        const float4* sb = reinterpret_cast<const float4*>(stats + st * BN + half * 32);
#pragma unroll
        for (int i = 0; i < 16; ++i) col[i] = sb[i];
      }
      ok = mbar_wait_warp(bar(F::B_SP + buf), (j >> 1) & 1, abort_flag, p.err, ERR_WAIT_TMEM_FULL);
      if (!ok) break;
      tc_fence_after();
      const uint32_t s_at = lane_at + F::S_COL + buf * BN + half * 32, d_at = lane_at + F::DP_COL + buf * BN + half * 32;
      uint32_t x[32], y[32];
      tmem_ld_32x32(s_at, x);
      if (F::DPROD) tmem_ld_32x32(d_at, y);
      tmem_wait_ld();
      // ---- which of the 32 columns this row meets: bits, where a row of the tile does not meet the whole block
      uint32_t vis = 0xffffffffu;
      const bool all = b0 >= plain_lo && b0 + BN <= plain_hi;
      if (!all) {
        auto below = [](int k) { return k <= 0 ? 0u : (k >= 32 ? 0xffffffffu : (1u << k) - 1u); };
        if (KEY_ROWS) {
          // queries (packed) from the one that stands at this key on; with a window up to the last that reaches back to it
          const int from = max(0, r - offset) << p.pack_log;
          long long to = rows;
          if (p.window > 0) to = min(to, max(0ll, static_cast<long long>(r) - offset + p.window) << p.pack_log);
          vis = live ? below(static_cast<int>(to) - c0) & ~below(from - c0) : 0u;
        } else {
          const int last = min(t.nk - 1, tok + offset), from = p.window > 0 ? tok + offset - p.window + 1 : 0;
          vis = live ? below(last - c0 + 1) & ~below(from - c0) : 0u;
        }
      }
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float4 two = KEY_ROWS ? col[i] : make_float4(own.x, own.x, own.y, own.y);
        float2 e = fma2(make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), sc, make_float2(two.x, two.y));
        e.x = exp2f(e.x);
        e.y = exp2f(e.y);
        if (MODE == RB_DKV || MODE == RB_DV) w[i] = fa_pack2(e.x, e.y, fp16);
        if (F::DPROD) {
          const float2 dp = make_float2(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1])), delta = make_float2(two.z, two.w);
          split2<F16>(mul2(e, AGAIN ? fma2(dp, lift, delta) : add2(dp, delta)), y[2 * i], y[2 * i + 1]);
        }
      }
      if (!all) {                                   // what is not met counts as zero, whatever came out
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint32_t keep = ((vis >> (2 * i)) & 1u ? 0xffffu : 0u) | ((vis >> (2 * i + 1)) & 1u ? 0xffff0000u : 0u);
          if (MODE == RB_DKV || MODE == RB_DV) w[i] &= keep;
          if (F::DPROD) {
            y[2 * i] &= keep;
            y[2 * i + 1] &= keep;
          }
        }
      }
      if (MODE == RB_DKV || MODE == RB_DV) tmem_st_32x16(s_at, w);
      if (F::DPROD) {
        uint32_t z[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) { z[i] = y[2 * i]; w[i] = y[2 * i + 1]; }
        tmem_st_32x16(d_at, z);
        tmem_st_32x16(d_at + 16, w);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(F::B_TR + buf));
        if (KEY_ROWS) mbar_arrive(bar(F::B_SE + st));
      }
    }
    if (ok && blocks > 0) {
      ok = mbar_wait_warp(bar(F::B_ACC), 0, abort_flag, p.err, ERR_WAIT_TMEM_FULL);
      tc_fence_after();
    }
    // ---- each warpgroup stores one half of the accumulator's columns
    const bool filled = ok && blocks > 0;
    const uint32_t stage = r1_s + (half * 4 + quad) * 2048;           // the products have read the resident rows
    const long long at = KEY_ROWS ? t.k0 + r : t.q0 + tok;
    uint16_t* row = reinterpret_cast<uint16_t*>(p.out) + at * p.o_sr + head * p.o_sh;
    const bool write = live && (turn == 0 || odd);
    if (MODE == RB_DKV || MODE == RB_DV) {
      if (turn == 0) ragged_store(lane_at + F::ACC, half * DP / 2, (half + 1) * DP / 2, filled, false, 1.f, row, p.D, live, fp16, stage);
    }
    if (F::DPROD) {
      if (MODE == RB_DKV) row = reinterpret_cast<uint16_t*>(p.out2) + at * p.o2_sr + head * p.o2_sh;
      odd = ragged_store<AGAIN>(lane_at + (MODE == RB_DKV ? F::ACC2 : F::ACC), half * DP / 2, (half + 1) * DP / 2, filled, false,
                                AGAIN ? p.scale / lift : p.scale, row, p.D, write, fp16, stage) && live;
    }
  }
  if (!AGAIN) break;
  fence_proxy_async_smem();                 // copies may overwrite the stages
  tc_fence_before();
  const bool some = __syncthreads_or(odd);
  tc_fence_after();
  if (!some || turn == 1 || *abort_flag) break;
  // the barriers start anew, once the last arrivals at those of emptied stages are there
  if (warp == 1) {
    auto last_phase = [&](int first, int stages) {
      for (int st = 0; st < stages && st < blocks; ++st)
        mbar_wait_warp(bar(first + st), ((blocks - 1 - st) / stages) & 1, abort_flag, p.err, ERR_WAIT_EMPTY);
    };
    last_phase(F::B_1E, F::S1);
    if (!F::JOINT) last_phase(F::B_2E, F::S2);
  }
  __syncthreads();
  if (*abort_flag) break;
  if (threadIdx.x == 32) {
    for (int i = 0; i < F::BARS; ++i) mbar_inval(bar(i));
    init_barriers();
  }
  __syncthreads();
  lift = 1.f / 67108864.f;
  }

  if (*abort_flag) {                        // copies in flight land before the shared memory is given back
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------------------------- host side
// {D, heads, rows} over [rows, heads, D] by strides; box {64, `heads_box`, `rows_box`}
static int ragged_map(CUtensorMap* map, const void* ptr, int D, int heads, long long rows, long long sh, long long sr, int heads_box,
                      int rows_box, bool fp16) {
  const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(heads), static_cast<uint64_t>(rows)};
  const uint64_t strides[2] = {static_cast<uint64_t>(heads == 1 ? D : sh), static_cast<uint64_t>(rows == 1 ? (heads == 1 ? D : sh * heads) : sr)};
  const uint32_t box[3] = {64, static_cast<uint32_t>(heads_box), static_cast<uint32_t>(rows_box)};
  return make_tma_nd_16bit(map, ptr, 3, dims, strides, box, fp16);
}
template <typename K> static int ragged_ready(K kernel, uint32_t smem, unsigned long long* ready) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev > 63 || !((__atomic_load_n(ready, __ATOMIC_ACQUIRE) >> dev) & 1)) {   // one bit per device
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev <= 63) __atomic_fetch_or(ready, 1ull << dev, __ATOMIC_RELEASE);
  }
  return 0;
}
static int ragged_check(RaggedParams& p) {
  if (p.B <= 0 || p.Hq <= 0 || p.Hk <= 0 || p.Hq % p.Hk || p.Tq <= 0 || p.Tk <= 0 || p.Tq + p.Tk > 0x7fffffff) return -1;      // places of queries among keys are ints
  if (p.D <= 0 || p.D > 256 || p.D % 8) return -2;
  if (p.window >= p.Tk) p.window = 0;                // it reaches every key
  const int group = p.Hq / p.Hk;
  p.pack = 1;
  p.pack_log = 0;
  while (p.pack < 64 && group % (2 * p.pack) == 0) { p.pack *= 2; ++p.pack_log; }
  p.subs = group / p.pack;
  if (p.Tq * p.pack > 0x7fffffffll - 16384 || p.Hk * p.subs > 65535) return -1;
  return 0;
}
static void ragged_bind() {
  static thread_local bool bound = false;   // the driver's encoder needs a current context
  if (!bound) { cudaFree(nullptr); bound = true; }
}

template <int DP, bool F16>
static int ragged_fwd_launch(const CUtensorMap* m, const RaggedParams& p, cudaStream_t stream) {
  using F = RaggedFwd<DP>;
  static_assert(F::SMEM <= 232448, "shared memory budget of one CTA");
  static unsigned long long ready = 0;
  if (const int rc = ragged_ready(ragged_fwd_kernel<DP, F16>, F::SMEM, &ready)) return rc;
  const long long tiles = ((p.Tq << p.pack_log) + F::ROWS - 1) / F::ROWS + p.B + 2;
  ragged_fwd_kernel<DP, F16><<<dim3(static_cast<unsigned>(tiles), p.Hk * p.subs), F::THREADS, F::SMEM, stream>>>(m[0], m[1], m[2], p);
  return static_cast<int>(cudaGetLastError());
}
template <int DP, int MODE, bool F16>
static int ragged_bwd_any(const CUtensorMap& r1, const CUtensorMap& r2, const CUtensorMap& s1, const CUtensorMap& s2, const RaggedParams& p,
                             cudaStream_t stream) {
  using F = RaggedBwd<DP, MODE>;
  static_assert(F::SMEM <= 232448, "shared memory budget of one CTA");
  static unsigned long long ready = 0;
  if (const int rc = ragged_ready(ragged_bwd_kernel<DP, MODE, F16>, F::SMEM, &ready)) return rc;
  const long long rows = F::KEY_ROWS ? p.Tk : p.Tq << p.pack_log, tiles = (rows + 127) / 128 + p.B + 2;
  ragged_bwd_kernel<DP, MODE, F16><<<dim3(static_cast<unsigned>(tiles), F::KEY_ROWS ? p.Hk : p.Hk * p.subs), F::THREADS, F::SMEM, stream>>>(r1, r2, s1, s2, p);
  return static_cast<int>(cudaGetLastError());
}

template <int DP, int MODE>
static int ragged_bwd_launch(const CUtensorMap& r1, const CUtensorMap& r2, const CUtensorMap& s1, const CUtensorMap& s2, const RaggedParams& p,
                             cudaStream_t stream) {
  return p.fp16 ? ragged_bwd_any<DP, MODE, true>(r1, r2, s1, s2, p, stream) : ragged_bwd_any<DP, MODE, false>(r1, r2, s1, s2, p, stream);
}

}  // namespace oslo

extern "C" int oslo_ragged_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const int* q_off, const int* k_off, int B,
                               int Hq, int Hk, long long Tq, long long Tk, int D, long long q_sr, long long q_sh, long long k_sr,
                               long long k_sh, long long v_sr, long long v_sh, long long o_sr, long long o_sh, float scale, int window,
                               int dtype, int* err_word, cudaStream_t stream) {
  using namespace oslo;
  RaggedParams p{};
  p.q_off = q_off; p.k_off = k_off; p.B = B; p.Hq = Hq; p.Hk = Hk; p.Tq = Tq; p.Tk = Tk; p.D = D; p.window = window; p.scale = scale;
  p.out = o; p.o_sr = o_sr; p.o_sh = o_sh; p.lse = lse; p.err = err_word;
  if (dtype != OSLO_DT_BF16 && dtype != OSLO_DT_FP16) return -3;
  p.fp16 = dtype == OSLO_DT_FP16;
  if (const int rc = ragged_check(p)) return rc;
  if ((reinterpret_cast<uintptr_t>(o) & 15) || o_sr % 8 || o_sh % 8) return -4;
  ragged_bind();
  const int bn = 64;
  CUtensorMap m[3];
  int rc;
  if ((rc = ragged_map(&m[0], q, D, Hq, Tq, q_sh, q_sr, p.pack, 128 / p.pack, p.fp16))) return rc;
  if ((rc = ragged_map(&m[1], k, D, Hk, Tk, k_sh, k_sr, 1, bn, p.fp16))) return rc;
  if ((rc = ragged_map(&m[2], v, D, Hk, Tk, v_sh, v_sr, 1, bn, p.fp16))) return rc;
  if (D <= 64) return p.fp16 ? ragged_fwd_launch<64, true>(m, p, stream) : ragged_fwd_launch<64, false>(m, p, stream);
  if (D <= 128) return p.fp16 ? ragged_fwd_launch<128, true>(m, p, stream) : ragged_fwd_launch<128, false>(m, p, stream);
  return p.fp16 ? ragged_fwd_launch<256, true>(m, p, stream) : ragged_fwd_launch<256, false>(m, p, stream);
}

// stats: workspace [Tq, Hq, 2]
extern "C" int oslo_ragged_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, const float* lse, float* stats,
                               void* dq, void* dk, void* dv, const int* q_off, const int* k_off, int B, int Hq, int Hk, long long Tq,
                               long long Tk, int D, long long q_sr, long long q_sh, long long k_sr, long long k_sh, long long v_sr,
                               long long v_sh, long long o_sr, long long o_sh, long long g_sr, long long g_sh, long long dq_sr,
                               long long dq_sh, long long dk_sr, long long dk_sh, long long dv_sr, long long dv_sh, float scale, int window,
                               int dtype, int* err_word, cudaStream_t stream) {
  using namespace oslo;
  RaggedParams p{};
  p.q_off = q_off; p.k_off = k_off; p.B = B; p.Hq = Hq; p.Hk = Hk; p.Tq = Tq; p.Tk = Tk; p.D = D; p.window = window; p.scale = scale;
  p.stats = reinterpret_cast<const float2*>(stats); p.err = err_word;
  if (dtype != OSLO_DT_BF16 && dtype != OSLO_DT_FP16) return -3;
  p.fp16 = dtype == OSLO_DT_FP16;
  if (const int rc = ragged_check(p)) return rc;
  const void* ptrs[5] = {o, dout, dq, dk, dv};
  for (const void* x : ptrs)
    if (reinterpret_cast<uintptr_t>(x) & 15) return -4;
  for (long long s : {o_sr, o_sh, g_sr, g_sh, dq_sr, dq_sh, dk_sr, dk_sh, dv_sr, dv_sh})
    if (s % 8) return -4;
  ragged_bind();
  {
    const long long rows = Tq * Hq;
    const int lpr = D <= 64 ? 8 : (D <= 128 ? 16 : 32);
    const long long blocks = (rows + 256 / lpr - 1) / (256 / lpr);
    if (blocks > 0x7fffffffll) return -1;
#define RAGGED_DELTA(T, L) ragged_delta_kernel<T, L><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(static_cast<const T*>(o), static_cast<const T*>(dout), lse, \
                                                                                                     reinterpret_cast<float2*>(stats), rows, Hq, D, o_sr, o_sh, g_sr, g_sh)
    if (p.fp16) {
      if (lpr == 8) RAGGED_DELTA(__half, 8);
      else if (lpr == 16) RAGGED_DELTA(__half, 16);
      else RAGGED_DELTA(__half, 32);
    } else {
      if (lpr == 8) RAGGED_DELTA(__nv_bfloat16, 8);
      else if (lpr == 16) RAGGED_DELTA(__nv_bfloat16, 16);
      else RAGGED_DELTA(__nv_bfloat16, 32);
    }
#undef RAGGED_DELTA
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  CUtensorMap kr, vr, qs, gs, qr, gr, ks, vs;      // r: 128 resident rows, s: 64 streamed ones
  int rc;
  if ((rc = ragged_map(&kr, k, D, Hk, Tk, k_sh, k_sr, 1, 128, p.fp16)) || (rc = ragged_map(&ks, k, D, Hk, Tk, k_sh, k_sr, 1, 64, p.fp16)) ||
      (rc = ragged_map(&vr, v, D, Hk, Tk, v_sh, v_sr, 1, 128, p.fp16)) || (rc = ragged_map(&vs, v, D, Hk, Tk, v_sh, v_sr, 1, 64, p.fp16)) ||
      (rc = ragged_map(&qr, q, D, Hq, Tq, q_sh, q_sr, p.pack, 128 / p.pack, p.fp16)) ||
      (rc = ragged_map(&qs, q, D, Hq, Tq, q_sh, q_sr, p.pack, 64 / p.pack, p.fp16)) ||
      (rc = ragged_map(&gr, dout, D, Hq, Tq, g_sh, g_sr, p.pack, 128 / p.pack, p.fp16)) ||
      (rc = ragged_map(&gs, dout, D, Hq, Tq, g_sh, g_sr, p.pack, 64 / p.pack, p.fp16)))
    return rc;
  RaggedParams a = p;
  a.out = dq; a.o_sr = dq_sr; a.o_sh = dq_sh;
  RaggedParams b = p;
  b.out = dv; b.o_sr = dv_sr; b.o_sh = dv_sh; b.out2 = dk; b.o2_sr = dk_sr; b.o2_sh = dk_sh;
  if (D <= 64) {
    if ((rc = ragged_bwd_launch<64, RB_DKV>(kr, vr, qs, gs, b, stream))) return rc;
    return ragged_bwd_launch<64, RB_DQ>(qr, gr, ks, vs, a, stream);
  }
  if (D <= 128) {
    if ((rc = ragged_bwd_launch<128, RB_DKV>(kr, vr, qs, gs, b, stream))) return rc;
    return ragged_bwd_launch<128, RB_DQ>(qr, gr, ks, vs, a, stream);
  }
  RaggedParams c = p;
  c.out = dk; c.o_sr = dk_sr; c.o_sh = dk_sh;
  if ((rc = ragged_bwd_launch<256, RB_DV>(kr, vr, qs, gs, b, stream))) return rc;
  if ((rc = ragged_bwd_launch<256, RB_DK>(kr, vr, qs, gs, c, stream))) return rc;
  return ragged_bwd_launch<256, RB_DQ>(qr, gr, ks, vs, a, stream);
}
