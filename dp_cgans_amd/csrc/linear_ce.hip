// Softmax cross entropy of a Linear layer over a large vocabulary, with its gradients, a piece of rows at a time.  What a piece keeps
// of its logits: half precision for the loss alone, 8 bytes for every 64 or 128 of them; with gradients, 2 bytes each; fp32, 4
// bytes each.  (A piece is all rows up to 1 GiB of that or twice the fp32 size of dW: 8192 x 131072 in half precision, 2.1 GB.  The
// caller may ask for smaller ones.)
//
//   l = h W^T,  lse_r = log sum_v e^(l_rv),  loss_r = lse_r - l_(r, t_r),
//   d_rv = e^(l_rv - lse_r) - [v = t_r],  dh = alpha d W,  dW = alpha d^T h,  alpha = gscale / rows that count.
//
// Half-precision operands (bf16, fp16), per piece of rows:
//   1. logits tiles on the matrix cores, fp32 accumulators.  A wave reduces its 128 (or 64) vocabulary entries of a row, its
//      slab, to a pair: ref = max l and the sum of x = e^(l - ref) in fp32; for training it leaves
//      2^15 x in fp16 in P: 11 bits down to 2^-29 of the slab's largest, where a later bf16 holds 8, and 2^-40 of it in all.  (x
//      itself would have 11 bits to 2^-14 and nothing below 2^-25: beside a sure target, all the rest of the row.)
//   2. per row: the slabs' pairs become one, lse = ref + log sum, loss = (ref - l_t) + log sum, p_t - 1 = expm1(-loss): a
//      sure row's small loss keeps its digits.
//   3. P becomes d in the operands' type, which the matrix instruction asks for: e^(slab's ref - row's ref) / row's sum times
//      what is there, p_t - 1 in the target's place, exactly 0 in rows that are ignored.  (Up to 16 rows: to the sum of two such
//      numbers.)  With the result's own rounding this leaves dh and dW 0.0019 off in bf16, 0.00072 in fp16, where the
//      result's rounding alone makes 0.0017 and 0.00071.
//   4. dh and dW as products over d.  dW of several pieces adds up in fp32.
// That is 6 T V D flops.  They bound it for widths in the thousands (6 D flops against the 10 bytes per logit that writing
// P, turning it into d and reading it twice move: 8192 x 2048 x 131072 spends 3.6 + 0.8 + 3.0 + 3.1 ms on steps 1, 3 and
// 4); below a width of about 500 the traffic does.
//
// P's layout [vocabulary / 8][row][8 entries] serves all three products: 16-byte chunks of 8 vocabulary entries are k-runs
// of the dh product's operand and, transposed on the way out of LDS, m-runs of dW's; step 1 and 3 touch it in runs of
// consecutive rows.
//
// fp32 operands: the products are dpc_gemm_f32_ex's (fp32 matrix cores), the logits of a piece in fp32.  Pieces of up to 16 rows
// have kernels of their own for what reads or writes all of W once.
#include "dpc_common.h"
#include "../../include/dpcgan_hip.h"
#include <math.h>
#include <string.h>
#include <type_traits>

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

#define LCE_BK 32               // k of one tile of an operand
#define LCE_LOG2E 1.4426950408889634f
#define LCE_LN2 0.6931471805599453f

// e^(l - ref), l <= ref.  The difference first: it is exact near ref and never above 0, whatever the size of the logits.  (With
// l log2 e - ref log2 e as one multiply-add the rounding of the product with ref stays in the exponent: up to 1 for logits of
// 2^24, and 2^8, which no fp32 sum holds, for those of 2^32.)
__device__ __forceinline__ float lce_exp(float l, float ref) { return __builtin_amdgcn_exp2f((l - ref) * LCE_LOG2E); }

#define LCE_HELD 32768.f        // e^(l - max) in [0, 1] in fp16, whose largest number is 65504
#define LCE_FEW 16              // rows of a piece that the few-rows kernels take: one 16 x 16 block of a matrix instruction

enum { LCE_LOGITS = 0, LCE_DH = 1, LCE_DW = 2 };

// 16-bit element types and their matrix instruction.  16 x 16 x 32 and not 32 x 32 x 16: the chip lowers its clock under
// these products, and with half the accumulator traffic per multiplication the smaller block keeps a higher one (nothing
// but matrix instructions on random bf16: 1946 against 1707 TFLOP/s; on zeros both reach 2450).
template <typename E> struct Half;
template <> struct Half<__bf16> {
  typedef bf16x8 v8;
  static __device__ __forceinline__ f32x4 mfma(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static constexpr float kUp = 1.f;         // d as it is: bf16 has fp32's range
};
template <> struct Half<_Float16> {
  typedef f16x8 v8;
  static __device__ __forceinline__ f32x4 mfma(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static constexpr float kUp = 16384.f;     // |d| <= 1 lifted by 2^14: normal numbers down to 2^-28, steps of 2^-38 below
};

// What a product reads and writes.  The result is C[n][m]: m is the contiguous axis of the output.
struct LceArgs {
  const char* A; int64_t lda;     // LOGITS: W [V][D]; DH: W [V][D] (k = row); DW: masked h [rows][D] (k = row); bytes per row
  const char* B; int64_t ldb;     // LOGITS: h [rows][D]
  char* P; int64_t prow;          // P, rows of one chunk column
  int M, N, K;
  int tiles_m, tiles_n;
  // LOGITS
  f32x2* stat;                    // [slab][prow] (reference, sum of e^(l - reference)); a slab is a wave's vocabulary entries
  float* lt;                      // [row] logit of the target
  const int64_t* target;
  int grads;
  // DH / DW
  const float* alpha;
  void* C; int64_t ldc;           // elements
  int c_f32;                      // C is fp32
  const float* add;               // fp32 [n][ldadd] added to the result (accumulation over pieces, or into dW)
  int64_t ldadd;
  // tiles from `whole` on - the last, incomplete round of the chip - are cut into `splits` ranges of K, each of which leaves
  // its fp32 sums in a slab of its own: part [split][tile][BN][BM]
  int whole, splits, kchunk;
  float* part;
};

// Tile `tl` of a product: groups of 8 m-tiles run through all n-tiles, so that the tiles an XCD works on at a time share
// rows of both operands.
__device__ __forceinline__ void lce_tile_at(int tl, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int per = 8 * tiles_n, grp = tl / per, gm = min(8, tiles_m - grp * 8);
  tm = grp * 8 + (tl - grp * per) % gm;
  tn = (tl - grp * per) / gm;
}

// Runs of neighbouring tiles per XCD: blocks go to the 8 XCDs in turn; each XCD takes a contiguous run of tile numbers
// (the tail that does not divide by 8 stays in place).
__device__ __forceinline__ int lce_xcd(int b, int total) {
  const int per = total >> 3, even = per << 3;
  return b < even ? (b & 7) * per + (b >> 3) : b;
}

// 16 bytes per lane from base + off[lane] to lds + 16 * lane.  LCE_NONE as an offset is out of range: zeros.  (Buffer
// loads: the per-lane offset stays in its register for the whole loop and the base moves in scalar registers; and the
// compiler keeps counting LDS reads beside them, where a global load to LDS makes it wait for every one.)
#define LCE_NONE 0x80000000u
__device__ __forceinline__ void lce_dma(const char* base, uint32_t off, char* lds) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)LCE_NONE, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, (int)off, 0, 0, 0);
}
// (__restrict: a read that carries no alias information is held back by the compiler until every load to LDS has landed)
__device__ __forceinline__ u32x2 lce_tr(const char* __restrict lds) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)lds));
}

// Two 16 x 16 blocks' results, 4 consecutive m per lane, as 8 consecutive m per lane: lanes of group G (of 16) come to hold
// chunk G / 2 of block G & 1.
__device__ __forceinline__ u32x4 lce_pair(u32x2 x, u32x2 y) {
  const auto lo = __builtin_amdgcn_permlane16_swap(x.x, y.x, false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(x.y, y.y, false, false);
  return u32x4{lo[0], hi[0], lo[1], hi[1]};
}

typedef std::integral_constant<bool, true> Yes;
typedef std::integral_constant<bool, false> No;

// Waits until at most N of this wave's memory operations are in flight.
template <int N>
__device__ __forceinline__ void lce_wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// A wave's 16 SM x 16 SN logits: (reference, sum) of its slab for each row, the target's logit, and what is left of them in P.
// C layout of a 16 x 16 block: n = lane & 15 (nw has it), m = 4 (lane >> 4) + e.
template <int SM, int SN>
__device__ __forceinline__ void lce_logits_end(const LceArgs& g, f32x4 (&acc)[SM][SN], int mw, int nw, int G) {
  if (mw + SM * 16 > g.M) {
#pragma unroll
    for (int i = 0; i < SM; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (mw + i * 16 + 4 * G + e >= g.M)
#pragma unroll
          for (int j = 0; j < SN; ++j) acc[i][j][e] = -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < SN; ++j) {
    const int n = nw + j * 16;
    const int64_t t = n < g.N ? g.target[n] : -1;
    if (__any(t >= mw && t < mw + SM * 16)) {
      const int at = t >= mw && t < mw + SM * 16 ? (int)(t - mw) : -1;
#pragma unroll
      for (int i = 0; i < SM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (at == i * 16 + 4 * G + e) g.lt[n] = acc[i][j][e];
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < SM; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, acc[i][j][e]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    // the reference: the largest logit.  (All -inf: e^(l - 0) = 0, not NaN.)
    const float ref = top == -INFINITY ? 0.f : top;
    f32x4 run = {0.f, 0.f, 0.f, 0.f};                                // (four short sums: a sure row's is 1 and what little there is beside it)
#pragma unroll
    for (int i = 0; i < SM; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = lce_exp(acc[i][j][e], ref);
      run += acc[i][j];
    }
    float sum = (run.x + run.y) + (run.z + run.w);
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (G == 0 && mw < g.M) g.stat[(int64_t)(mw / (SM * 16)) * g.prow + n] = f32x2{ref, sum};
    if (g.grads) {
#pragma unroll
      for (int i = 0; i < SM; i += 2) {
        u32x2 x[2];
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const f16x2 v = {(_Float16)(acc[i + w][j][2 * c] * LCE_HELD), (_Float16)(acc[i + w][j][2 * c + 1] * LCE_HELD)};
            x[w][c] = __builtin_bit_cast(uint32_t, v);
          }
        // (past the caches: nothing reads P before all of it is there - 8192 x 131072: 3.84 -> 3.57 ms)
        __builtin_nontemporal_store(lce_pair(x[0], x[1]),
                                    reinterpret_cast<u32x4*>(g.P + ((int64_t)((mw + (i + (G & 1)) * 16) / 8 + (G >> 1)) * g.prow + n) * 16));
      }
    }
  }
}

// One BM x BN tile of a product, WM x WN waves.  A tile of an operand is 32 k; it goes from memory straight into LDS, 16
// bytes per lane, in one of three images:
//   k-runs  (W and h of LOGITS, P of DH): [row][4 chunks of 8 k], chunk c of row r at c ^ (r / 2 & 3) - read 16 bytes a lane
//   m-runs  (W of DH, h of DW): [k][chunks of 8 m], chunk c of row k at c ^ (2 (k & 3) + (k & 8))      - read transposed
//           (P of DW): [chunk of 8 m][k], k at k ^ 4 (chunk & 1)                                       - read transposed
// The transposing read gives lane i of 16 the column i of a 4 x 16 block whose row r comes from lanes 4r .. 4r+3; the
// swizzles put what the 32 lanes of one LDS cycle read on different banks.
//
// NS = 3 tiles are in use or on their way.  Iteration kt: while the products of the wave's upper rows run, its lower rows'
// fragments are read; then, once tile kt + 1 has landed for every wave and tile kt has been read by all (one barrier),
// tile kt + NS goes on its way into the freed slot and the next tile's first fragments are read while the lower rows'
// products run.
//
// 256 x 256 with 8 waves of 128 x 64 for the logits (a wave's 128 entries are a slab) and of 64 x 128 for the gradients, whose
// transposed reads of A take two instructions each (dh 2 % faster); 200 registers, 96 KB of LDS, one block per CU.  On 8192
// rows, width 2048, vocabulary 131072: 1227 (logits), 1475 (dh) and 1427 (dW) TFLOP/s where a library product of the same shape
// reaches 1374 to 1594 and nothing but matrix instructions 1946.  What limits it is power first: the clock falls to 1.8 GHz,
// and with all operands 0 the same instructions take 17 to 24 % less time at 2.4.  Then the steps between the products: the
// matrix units are busy 75 % of the cycles, 80 % without the reads of LDS, 97 % without loads and reads.  Measured and
// dropped: 4 waves of 128 x 128 (spills, or the same), two 4-wave blocks per CU (dh 1.3 times as long), four and five tiles in
// LDS (the same), one barrier per 64 k (dW 4 % faster, the others 6 to 9 % slower), blocks started at different times, both
// halves of W's lines at once (half the requests to L2, logits 2 % slower), slots as constants in a loop over three tiles
// (spills), one block per CU that goes from output tile to output tile with the next one's first loads on their way while
// results leave (the logits 0.5 to 2 % faster for as much code again: power, not time, is short).
template <typename E, int MODE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void lce_product_kernel(LceArgs g) {
  using H = Half<E>;
  constexpr int NT = WM * WN * 64;
  constexpr int SM = BM / WM / 16, SN = BN / WN / 16, SH = SM / 2;
  constexpr int NA = BM * 4 / NT, NB = BN * 4 / NT;
  constexpr int SLOT = (BM + BN) * 64, NS = 3;
  constexpr bool A_K = MODE == LCE_LOGITS, B_K = MODE != LCE_DW;
  __shared__ __attribute__((aligned(1024))) char lds[NS * SLOT];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int rest = g.tiles_m * g.tiles_n - g.whole;
  int tl, split = 0, k_begin = 0, k_end = g.K;
  if ((int)blockIdx.x < g.whole) {
    tl = lce_xcd(blockIdx.x, g.whole);
  } else {
    const int u = lce_xcd(blockIdx.x - g.whole, rest * g.splits);
    split = u / rest;
    tl = g.whole + u - split * rest;
    k_begin = split * g.kchunk;
    k_end = min(g.K, k_begin + g.kchunk);
  }
  int m0, n0;
  lce_tile_at(tl, g.tiles_m, g.tiles_n, m0, n0);
  m0 *= BM;
  n0 *= BN;
  const int nk = (k_end - k_begin + LCE_BK - 1) / LCE_BK;

  // this thread's chunks of a K-tile, as offsets from the tile's first k; none where the operand ends
  uint32_t oa[NA], ob[NB];
  const char *pa, *pb0;
  int64_t step_a, step_b;
  const int ck = (tid & 3) ^ ((tid >> 3) & 3);                          // k-runs: chunk of this thread
  if (A_K) {
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int r = i * (NT / 4) + (tid >> 2);
      oa[i] = m0 + r < g.M ? (uint32_t)r * (uint32_t)g.lda + ck * 16 : LCE_NONE;
    }
    pa = g.A + (int64_t)m0 * g.lda;
    step_a = LCE_BK * 2;
  } else {
    constexpr int CR = BM / 8;
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int k = i * (NT / CR) + tid / CR, c = (tid % CR) ^ (2 * (k & 3) + (k & 8));
      oa[i] = m0 + c * 8 < g.M ? (uint32_t)k * (uint32_t)g.lda + c * 16 : LCE_NONE;
    }
    pa = g.A + (int64_t)k_begin * g.lda + (int64_t)m0 * 2;
    step_a = LCE_BK * g.lda;
  }
  if (MODE == LCE_LOGITS) {
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int r = i * (NT / 4) + (tid >> 2);
      ob[i] = n0 + r < g.N ? (uint32_t)r * (uint32_t)g.ldb + ck * 16 : LCE_NONE;
    }
    pb0 = g.B + (int64_t)n0 * g.ldb;
    step_b = LCE_BK * 2;
  } else if (MODE == LCE_DH) {
#pragma unroll
    for (int i = 0; i < NB; ++i) ob[i] = ((uint32_t)ck * (uint32_t)g.prow + i * (NT / 4) + (tid >> 2)) * 16;
    pb0 = g.P + ((int64_t)(k_begin / 8) * g.prow + n0) * 16;
    step_b = LCE_BK / 8 * g.prow * 16;
  } else {
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int n8 = i * (NT / 32) + (tid >> 5), k = (tid & 31) ^ (4 * (n8 & 1));
      ob[i] = ((uint32_t)n8 * (uint32_t)g.prow + k) * 16;
    }
    pb0 = g.P + ((int64_t)(n0 / 8) * g.prow + k_begin) * 16;
    step_b = LCE_BK * 16;
  }
  // Tiles are loaded in order; before the one that crosses the end of K, what lies past it becomes "none" (DW: K is whole tiles).
  const int kt_cut = MODE != LCE_DW && k_begin + nk * LCE_BK > g.K ? nk - 1 : -1;
  const auto cut = [&]() {
    const int k0 = k_begin + kt_cut * LCE_BK;
    const bool kend = k0 / 8 + ck >= g.K / 8;
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (A_K ? kend : k0 + i * (NT / (BM / 8)) + tid / (BM / 8) >= g.K) oa[i] = LCE_NONE;
    if (MODE == LCE_LOGITS && kend) {
#pragma unroll
      for (int i = 0; i < NB; ++i) ob[i] = LCE_NONE;
    }
  };
  const auto issue_one = [&](int kt, char* buf, int l) {                // load l (of NA + NB) of tile kt
    char* at = buf + wave * 1024;
    if (l < NA) lce_dma(pa + kt * step_a, oa[l < NA ? l : 0], at + l * NT * 16);
    else lce_dma(pb0 + kt * step_b, ob[l < NA ? 0 : l - NA], at + BM * 64 + (l - NA) * NT * 16);
  };
  const auto issue = [&](int kt, char* buf) {
    if (kt == kt_cut) cut();
#pragma unroll
    for (int l = 0; l < NA + NB; ++l) issue_one(kt, buf, l);
  };

  // lane addresses inside an image
  const int l16 = lane & 15, G = lane >> 4;
  const int kq = l16 * 64 + ((G ^ ((l16 >> 1) & 3)) * 16);                          // k-runs: row and chunk of this lane
  const int mk = (8 * G + (l16 >> 2)) * (BM * 2) + (l16 & 1) * 8;                   // m-runs [k][chunk]
  const int mc = (l16 & 3) >> 1, mx = 2 * (l16 >> 2) + 8 * (G & 1);
  int ma[SM];
#pragma unroll
  for (int i = 0; i < SM; ++i) ma[i] = mk + (((2 * (wm * SM + i) + mc) ^ mx) * 16);
  const int pb = ((l16 >> 1) & 1) * 64;
  const int pq = mc * 512 + (8 * G + (l16 >> 2)) * 16 + (l16 & 1) * 8;              // m-runs [chunk][k]
  static_assert(SM % 4 == 0 && SN % 2 == 0, "a wave's rows in whole 64s, its columns in whole 32s");
  const auto frag_a = [&](const char* buf, int i) -> typename H::v8 {
    if (A_K) return *reinterpret_cast<const typename H::v8*>(buf + (wm * SM + i) * 1024 + kq);
    const char* q = buf + ma[i];
    const u32x2 lo = lce_tr(q), hi = lce_tr(q + 4 * (BM * 2));
    return __builtin_bit_cast(typename H::v8, u32x4{lo.x, lo.y, hi.x, hi.y});
  };
  const auto frag_b = [&](const char* buf, int j) -> typename H::v8 {
    const char* q = buf + BM * 64 + (wn * SN + j) * 1024;
    if (B_K) return *reinterpret_cast<const typename H::v8*>(q + kq);
    const u32x2 lo = lce_tr(q + pq + pb), hi = lce_tr(q + pq + (64 - pb));
    return __builtin_bit_cast(typename H::v8, u32x4{lo.x, lo.y, hi.x, hi.y});
  };

  f32x4 acc[SM][SN];
#pragma unroll
  for (int i = 0; i < SM; ++i)
#pragma unroll
    for (int j = 0; j < SN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  typename H::v8 a0[SH], a1[SH], b[SN];
  // One half of a tile's products with the reads of the next half, and a tile's loads, evenly between them: a wave that waits
  // for the matrix unit has them behind it.  In this order, pinned, each product first: what stands before the first one
  // after a barrier holds up every wave at once.  Column by column, so that b[j] is free for the next tile's once its products
  // have been issued.
  const auto half_tile = [&](auto lower, auto more, auto load, const char* buf, int kt, char* into) {
    constexpr bool LOW = decltype(lower)::value, MORE = decltype(more)::value, LOAD = decltype(load)::value;
    constexpr int SLOTS = SH * SN, L = NA + NB;
#pragma unroll
    for (int j = 0; j < SN; ++j) {
#pragma unroll
      for (int i = 0; i < SH; ++i) {
        acc[(LOW ? SH : 0) + i][j] = H::mfma((LOW ? a1 : a0)[i], b[j], acc[(LOW ? SH : 0) + i][j]);
        __builtin_amdgcn_sched_barrier(0);
        const int p = j * SH + i;
#pragma unroll
        for (int q = 0; q < SH; ++q)
          if (p == q * SLOTS / SH) {
            if (!LOW) a1[q] = frag_a(buf, SH + q);
            else if (MORE) a0[q] = frag_a(buf, q);
          }
        if (LOW && MORE && i == SH - 1) b[j] = frag_b(buf, j);
        if (LOAD) {
#pragma unroll
          for (int l = 0; l < L; ++l)
            if (l * SLOTS / L + SLOTS / L / 2 == p) issue_one(kt, into, l);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  // The next tile has landed for every wave - `ahead`: NS - 2 others may be on their way behind it - and this one has been read.
  const auto meet = [&](bool ahead) {
    if (ahead) lce_wait_vm<(NS - 2) * (NA + NB)>();
    else lce_wait_vm<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };

  if (nk > 0) {
#pragma unroll
    for (int k = 0; k < NS - 1; ++k)
      if (k < nk) issue(k, lds + k * SLOT);
    meet(nk >= NS - 1);
    if (nk >= NS) issue(NS - 1, lds + (NS - 1) * SLOT);
#pragma unroll
    for (int j = 0; j < SN; ++j) b[j] = frag_b(lds, j);
#pragma unroll
    for (int i = 0; i < SH; ++i) a0[i] = frag_a(lds, i);
    int cur = 0, kt = 0;
    const auto tile = [&](auto more, auto load, bool ahead) {
      const int nxt = cur + 1 == NS ? 0 : cur + 1;
      half_tile(No(), No(), No(), lds + cur * SLOT, 0, nullptr);
      if (decltype(more)::value) meet(ahead);
      half_tile(Yes(), more, load, lds + nxt * SLOT, kt + NS, lds + cur * SLOT);
      cur = nxt;
    };
    // (where K ends inside a tile the offsets of its loads change before them - outside of the loop, in which the test cost 1 %)
    for (int pass = kt_cut < NS; pass < 2; ++pass) {
      if (pass && kt_cut >= NS) cut();
      for (const int end = (pass ? nk : kt_cut) - NS; kt < end; ++kt) tile(Yes(), Yes(), true);
    }
    for (; kt + 1 < nk; ++kt) tile(Yes(), No(), kt + NS - 1 < nk);           // nothing more to load
    tile(No(), No(), false);
  }

  // C layout of a 16 x 16 block: n = lane & 15, m = 4 (lane >> 4) + e
  const int mw = m0 + wm * SM * 16, nw = n0 + wn * SN * 16 + l16;
  if (MODE == LCE_LOGITS) {
    lce_logits_end<SM, SN>(g, acc, mw, nw, G);
  } else {
    if (tl >= g.whole) {
      float* q = g.part + ((int64_t)(split * rest + tl - g.whole) * BN + wn * SN * 16 + l16) * BM + wm * SM * 16 + 4 * G;
#pragma unroll
      for (int j = 0; j < SN; ++j)
#pragma unroll
        for (int i = 0; i < SM; ++i) *reinterpret_cast<f32x4*>(q + j * 16 * BM + i * 16) = acc[i][j];
      return;
    }
    const float alpha = g.alpha[0];
#pragma unroll
    for (int j = 0; j < SN; ++j) {
      const int n = nw + j * 16;
      const bool row = n < g.N;
      const int64_t o = (int64_t)n * g.ldc;
      if (g.add && row) {
        f32x4 x[SM];
#pragma unroll
        for (int i = 0; i < SM; ++i)
          if (mw + i * 16 + 4 * G < g.M) x[i] = *reinterpret_cast<const f32x4*>(g.add + (int64_t)n * g.ldadd + mw + i * 16 + 4 * G);
#pragma unroll
        for (int i = 0; i < SM; ++i) acc[i][j] = alpha * acc[i][j] + x[i];
      } else {
#pragma unroll
        for (int i = 0; i < SM; ++i) acc[i][j] *= alpha;
      }
      if (g.c_f32) {
#pragma unroll
        for (int i = 0; i < SM; ++i) {
          const int m = mw + i * 16 + 4 * G;
          if (row && m < g.M) *reinterpret_cast<f32x4*>((float*)g.C + o + m) = acc[i][j];
        }
      } else {
        typedef E e4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int i = 0; i < SM; i += 2) {
          const u32x4 v = lce_pair(__builtin_bit_cast(u32x2, __builtin_convertvector(acc[i][j], e4)),
                                   __builtin_bit_cast(u32x2, __builtin_convertvector(acc[i + 1][j], e4)));
          const int m = mw + (i + (G & 1)) * 16 + (G >> 1) * 8;
          if (row && m < g.M) *reinterpret_cast<u32x4*>((E*)g.C + o + m) = v;
        }
      }
    }
  }
}

// Logits of at most 16 rows: reading W once is all there is to it.  One wave per block takes 64 vocabulary entries and no LDS: a
// lane's 16 bytes of W are one operand of a matrix instruction, and 32 of them are on their way.  One row, vocabulary 131072,
// width 2048: 136 us for the call (4.0 TB/s), 144 with tiles through LDS; 4 x 256 x 18000 in a graph 8.9 against 10.0 us.
template <typename E>
__global__ __launch_bounds__(64) void lce_few_kernel(LceArgs g) {
  using H = Half<E>;
  constexpr int SM = 4, U = 8;
  const int l16 = threadIdx.x & 15, G = threadIdx.x >> 4, mw = blockIdx.x * 16 * SM;
  const char *pa[SM], *pb = g.B + (int64_t)min(l16, g.N - 1) * g.ldb + G * 16;        // (past the last row or entry: that one again, and not used)
#pragma unroll
  for (int i = 0; i < SM; ++i) pa[i] = g.A + (int64_t)min(mw + i * 16 + l16, g.M - 1) * g.lda + G * 16;
  f32x4 acc[SM][1];
#pragma unroll
  for (int i = 0; i < SM; ++i) acc[i][0] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < g.K; k += 32 * U) {
    u32x4 a[U][SM], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = k + 32 * u + 8 * G < g.K;
      b[u] = in ? *reinterpret_cast<const u32x4*>(pb + (k + 32 * u) * 2) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < SM; ++i) a[u][i] = in ? *reinterpret_cast<const u32x4*>(pa[i] + (k + 32 * u) * 2) : u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < SM; ++i)
        acc[i][0] = H::mfma(__builtin_bit_cast(typename H::v8, a[u][i]), __builtin_bit_cast(typename H::v8, b[u]), acc[i][0]);
  }
  lce_logits_end<SM, 1>(g, acc, mw, l16, G);
}

// ---- the passes between the products --------------------------------------------------------------------------------
// Two (reference, sum) pairs of a row as one.  (A sum of 0 - all logits -inf - leaves the other as it is.)
__device__ __forceinline__ f32x2 lce_join(f32x2 x, f32x2 y) {
  if (x.y == 0.f) return y;
  if (y.y == 0.f) return x;
  const float m = fmaxf(x.x, y.x);
  return f32x2{m, x.y * lce_exp(x.x, m) + y.y * lce_exp(y.x, m)};
}

// Per row: the slabs' pairs become one, lse, the loss and what the gradient needs.  16 rows x 64 runs of slabs per block (with
// 32 rows x 8 runs a thread's chain of 128 dependent loads and exponents took 65 us for 4096 x 1024 pairs, now 8); the runs
// meet within their waves first and through LDS once.
struct LceRowArgs {
  const f32x2* stat; int64_t prow; int slabs; int rows; int V;
  const float* lt; const int64_t* target; int64_t ignore;
  float* loss; float* lse;      // lse nullable
  f32x2* live;                  // (reference, 1 / sum) of a row, (0, 0) where it takes no part in the gradient; nullable
  float* pm1;                   // p_t - 1
  // one block more: *alpha = scale / (rows of the whole call that count, or 1)
  float* alpha; float scale; int mean; const int64_t* all; int64_t T;
  float* total;                 // of a call that is one block: the mean (or sum) of the losses; nullable
};
__global__ __launch_bounds__(1024) void lce_rows_kernel(LceRowArgs a) {
  __shared__ f32x2 red[16][16];
  if (a.alpha && blockIdx.x + 1 == gridDim.x) {
    int c = 0;
    if (a.mean)
      for (int64_t i = threadIdx.x; i < a.T; i += 1024) c += a.all[i] != a.ignore;
    c = dpc_block_sum(c, reinterpret_cast<int*>(red));
    if (threadIdx.x == 0) a.alpha[0] = a.scale / (a.mean ? (float)max(c, 1) : 1.f);
    return;
  }
  const int r = threadIdx.x & 15, w = threadIdx.x >> 4;
  const int n = blockIdx.x * 16 + r;
  f32x2 x = {0.f, 0.f};
  if (n < a.rows) {
#pragma unroll 4
    for (int s = w; s < a.slabs; s += 64) x = lce_join(x, a.stat[(int64_t)s * a.prow + n]);
  }
  x = lce_join(x, f32x2{__shfl_xor(x.x, 16, 64), __shfl_xor(x.y, 16, 64)});
  x = lce_join(x, f32x2{__shfl_xor(x.x, 32, 64), __shfl_xor(x.y, 32, 64)});
  if ((w & 3) == 0) red[w >> 2][r] = x;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  x = lce_join(lce_join(red[w][r], red[w + 4][r]), lce_join(red[w + 8][r], red[w + 12][r]));
  x = lce_join(x, f32x2{__shfl_xor(x.x, 16, 64), __shfl_xor(x.y, 16, 64)});
  x = lce_join(x, f32x2{__shfl_xor(x.x, 32, 64), __shfl_xor(x.y, 32, 64)});
  double sum = 0.0;
  int count = 0;
  if (w == 0 && n < a.rows) {
    const int64_t t = a.target[n];
    const bool off = t == a.ignore, bad = !off && (t < 0 || t >= a.V);
    // The loss from what is exact near it: where the target is the row's largest logit it is the logarithm of the sum - not
    // the difference of two numbers of the logits' size.
    const float l2 = log2f(x.y);
    const float loss = off ? 0.f : (bad ? NAN : fmaf(LCE_LN2, l2, x.x - a.lt[n]));
    a.loss[n] = loss;
    if (a.lse) a.lse[n] = fmaf(LCE_LN2, l2, x.x);
    if (a.live) {
      a.live[n] = off || bad ? f32x2{0.f, 0.f} : f32x2{x.x, 1.f / x.y};
      a.pm1[n] = off || bad ? 0.f : expm1f(-loss);
    }
    sum = (double)loss;
    count = !off;
  }
  if (a.total) {
    sum = dpc_wave_sum(sum);
    count = dpc_wave_sum(count);
    if (threadIdx.x == 0) a.total[0] = (float)(sum / (a.mean ? (double)max(count, 1) : 1.0));
  }
}

// The losses of all rows of the call as one: their sum, over the rows that count if `mean`.  One block, in a fixed order: a launch
// of its own for the loss alone, a block beside those that turn logits into d otherwise (a launch less: fp32 500 x 256 x
// 18000 175 -> 172 us).
struct LceTotal { const float* loss; const int64_t* target; int64_t T, ignore; int mean; float* total; };
template <int NT>
__device__ __forceinline__ void lce_total(const LceTotal& a) {
  __shared__ double red[16];
  __shared__ int redi[16];
  double s = 0.0;
  int c = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < a.T; i += NT) {
    s += (double)a.loss[i];
    c += a.target[i] != a.ignore;
  }
  s = dpc_block_sum(s, red);
  c = dpc_block_sum(c, redi);
  if (threadIdx.x == 0) a.total[0] = (float)(s / (a.mean ? (double)max(c, 1) : 1.0));
}

// P from 2^15 e^(l - slab max) in fp16 to d in the operands' type, in place.  One thread per row and slab.
// NT: P is much larger than the 256 MB of the last-level cache - read and written past it (2 GB: 846 -> 780 us; 0.3 GB: 96 -> 103 us).
// `copies` blocks from `slabs` * prow / 256 on copy h with its ignored rows, and the rows up to the end of the piece's last tile,
// set to 0: what such a row holds must not reach dW (0 x NaN).  One more of the last piece: the total.
template <typename E, bool NT>
__global__ __launch_bounds__(256) void lce_scale_kernel(char* P, int64_t prow, const f32x2* stat, int slabs, int rows, int slab_rows, const f32x2* live,
                                                        const float* pm1, const int64_t* target, const char* h, int64_t ldh, int row16, char* hm, int copies,
                                                        LceTotal all) {
  const int first = slabs * (int)(prow / 256);
  if ((int)blockIdx.x >= first + copies) {
    lce_total<256>(all);
    return;
  }
  if ((int)blockIdx.x >= first) {
    for (int64_t i = (int64_t)(blockIdx.x - first) * 256 + threadIdx.x; i < prow * row16; i += (int64_t)copies * 256) {
      const int n = (int)(i / row16), c = (int)(i - (int64_t)n * row16);
      u32x4 v = {0u, 0u, 0u, 0u};
      if (n < rows && live[n].y != 0.f) v = *reinterpret_cast<const u32x4*>(h + (int64_t)n * ldh + c * 16);
      *reinterpret_cast<u32x4*>(hm + i * 16) = v;
    }
    return;
  }
  const int nb = (int)(prow / 256), slab = blockIdx.x / nb, n = (blockIdx.x - slab * nb) * 256 + threadIdx.x;
  const f32x2 gl = n < rows ? live[n] : f32x2{0.f, 0.f};
  const bool on = gl.y != 0.f;                                         // (NaN is on: such a row keeps its NaN)
  const f32x2 st = on ? stat[(int64_t)slab * prow + n] : f32x2{0.f, 0.f};
  // (a slab of nothing but -inf has the sum 0 and a reference that may lie far above the row's)
  const float f = st.y == 0.f ? 0.f : lce_exp(st.x, gl.x) * gl.y * (Half<E>::kUp / LCE_HELD);
  int at = -1;
  float pt = 0.f;
  if (on) {
    const int64_t t = target[n] - (int64_t)slab * slab_rows;
    if (t >= 0 && t < slab_rows) { at = (int)t; pt = pm1[n] * Half<E>::kUp; }
  }
  char* p = P + ((int64_t)slab * (slab_rows / 8) * prow + n) * 16;
  for (int c0 = 0; c0 < slab_rows / 8; c0 += 8) {
    u32x4 q[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const u32x4* at = reinterpret_cast<const u32x4*>(p + (c0 + c) * prow * 16);
      q[c] = NT ? __builtin_nontemporal_load(at) : *at;
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const f16x8 x = __builtin_bit_cast(f16x8, q[c]);
      typename Half<E>::v8 y;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (E)(on ? ((c0 + c) * 8 + e == at ? pt : (float)x[e] * f) : 0.f);
      u32x4* to = reinterpret_cast<u32x4*>(p + (c0 + c) * prow * 16);
      if (NT) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, y), to);
      else *to = __builtin_bit_cast(u32x4, y);
    }
  }
}

// The same for at most LCE_FEW rows.  A gradient there may hang on two or three entries of d, whose roundings to 8 bits do not
// average out, so d is held as the sum of two numbers of the operands' type, in the rows n and n + LCE_FEW, and h twice
// beside them: dW comes out of one product over 2 LCE_FEW rows, dh of the sum of its rows - a product of 32 rows costs what one
// of 16 does, and the rest of P's 256 rows is not touched (1 x 2048 x 131072 467 -> 460 us, 16 x 256 x 18000 38 -> 36).  16
// chunks of 8 entries per block.
template <typename E>
__global__ __launch_bounds__(256) void lce_few_scale_kernel(char* P, int64_t prow, const f32x2* stat, int slabs, int rows, const f32x2* live, const float* pm1,
                                                            const int64_t* target, const char* h, int64_t ldh, int row16, char* hm, int copies, LceTotal all) {
  const int first = (slabs + 1) / 2;
  if ((int)blockIdx.x >= first + copies) {
    lce_total<256>(all);
    return;
  }
  if ((int)blockIdx.x >= first) {
    for (int i = (blockIdx.x - first) * 256 + threadIdx.x; i < LCE_FEW * row16; i += copies * 256) {
      const int n = i / row16, c = i - n * row16;
      u32x4 v = {0u, 0u, 0u, 0u};
      if (n < rows && live[n].y != 0.f) v = *reinterpret_cast<const u32x4*>(h + (int64_t)n * ldh + c * 16);
      *reinterpret_cast<u32x4*>(hm + (int64_t)i * 16) = v;
      *reinterpret_cast<u32x4*>(hm + ((int64_t)LCE_FEW * row16 + i) * 16) = v;
    }
    return;
  }
  const int n = threadIdx.x % LCE_FEW, chunk = blockIdx.x * 16 + threadIdx.x / LCE_FEW, slab = chunk / 8;
  if (slab >= slabs) return;
  const f32x2 gl = n < rows ? live[n] : f32x2{0.f, 0.f};
  const bool on = gl.y != 0.f;
  const f32x2 st = on ? stat[(int64_t)slab * prow + n] : f32x2{0.f, 0.f};
  const float f = st.y == 0.f ? 0.f : lce_exp(st.x, gl.x) * gl.y * (Half<E>::kUp / LCE_HELD);
  const int64_t t = on ? target[n] - (int64_t)chunk * 8 : -1;
  u32x4* at = reinterpret_cast<u32x4*>(P + ((int64_t)chunk * prow + n) * 16);
  const f16x8 x = __builtin_bit_cast(f16x8, *at);
  typename Half<E>::v8 y, z;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float d = on ? (t == e ? pm1[n] * Half<E>::kUp : (float)x[e] * f) : 0.f;
    const E hi = (E)d;
    y[e] = hi;
    z[e] = (E)(d - (float)hi);
  }
  at[0] = __builtin_bit_cast(u32x4, y);
  at[LCE_FEW] = __builtin_bit_cast(u32x4, z);
}
// dh[n] = x[n] + x[n + LCE_FEW]
template <typename E>
__global__ __launch_bounds__(256) void lce_few_join_kernel(const float* x, int rows, int D, E* dh, int64_t lddh) {
  for (int i = blockIdx.x * 256 + threadIdx.x; i < rows * D; i += gridDim.x * 256) {
    const int n = i / D, c = i - n * D;
    dh[(int64_t)n * lddh + c] = (E)(x[i] + x[i + LCE_FEW * D]);
  }
}

// Rows of `row16` 16-byte chunks to another pitch.
__global__ __launch_bounds__(256) void lce_pitch_kernel(const char* h, int64_t ldh, int rows, int row16, char* to, int64_t ldt) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)rows * row16; i += (int64_t)gridDim.x * 256) {
    const int64_t n = i / row16, c = i - n * row16;
    *reinterpret_cast<u32x4*>(to + n * ldt + c * 16) = *reinterpret_cast<const u32x4*>(h + n * ldh + c * 16);
  }
}

// C[n][m] = alpha * (sum of the K ranges' slabs, in their order) [+ add] for the tiles that were cut.  One block per 1024 entries.
template <typename E, int BM, int BN>
__global__ __launch_bounds__(256) void lce_fold_kernel(LceArgs g) {
  const int rest = g.tiles_m * g.tiles_n - g.whole;
  const int t = blockIdx.x / (BM * BN / 1024), at = (blockIdx.x % (BM * BN / 1024)) * 1024 + threadIdx.x * 4;
  int tm, tn;
  lce_tile_at(g.whole + t, g.tiles_m, g.tiles_n, tm, tn);
  const int n = tn * BN + at / BM, m = tm * BM + at % BM;
  if (n >= g.N || m >= g.M) return;
  const float* q = g.part + (int64_t)t * BM * BN + at;
  f32x4 v = *reinterpret_cast<const f32x4*>(q);
#pragma unroll 4
  for (int s = 1; s < g.splits; ++s) v += *reinterpret_cast<const f32x4*>(q + (int64_t)s * rest * (BM * BN));
  v *= g.alpha[0];
  if (g.add) v += *reinterpret_cast<const f32x4*>(g.add + (int64_t)n * g.ldadd + m);
  const int64_t o = (int64_t)n * g.ldc + m;
  if (g.c_f32) *reinterpret_cast<f32x4*>((float*)g.C + o) = v;
  else {
    typedef E e4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<e4*>((E*)g.C + o) = __builtin_convertvector(v, e4);
  }
}

// ---- fp32 -------------------------------------------------------------------------------------------------------------
// A block's 4096 logits of a row: their pair, the target's logit.  [row][ld], rows 16-byte aligned.
#define LCE_SEG 4096
__global__ __launch_bounds__(256) void lce_stat_f32_kernel(const float* logits, int64_t ld, int V, const int64_t* target, f32x2* stat, int64_t prow, float* lt) {
  __shared__ float red[16];
  const int segs = (V + LCE_SEG - 1) / LCE_SEG, n = blockIdx.x / segs, seg = blockIdx.x - n * segs, v0 = seg * LCE_SEG;
  const float* x = logits + (int64_t)n * ld + v0;
  f32x4 q[4];
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int v = k * 1024 + threadIdx.x * 4;
    q[k] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (v0 + v < V) q[k] = *reinterpret_cast<const f32x4*>(x + v);      // (the row's padding is within its stride)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (v0 + v + e >= V) q[k][e] = -INFINITY;
      top = fmaxf(top, q[k][e]);
    }
  }
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float ref = top == -INFINITY ? 0.f : top;
  f32x4 run = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) run[e] += lce_exp(q[k][e], ref);
  const float sum = dpc_block_sum((run.x + run.y) + (run.z + run.w), red);
  if (threadIdx.x == 0) {
    stat[(int64_t)seg * prow + n] = f32x2{ref, sum};
    const int64_t t = target[n] - v0;
    if (t >= 0 && t < LCE_SEG && v0 + t < V) lt[n] = x[t];
  }
}

// Logits to alpha * d, in place; the `copies` blocks behind them copy h with its ignored rows set to 0, one more takes the total.
__global__ __launch_bounds__(256) void lce_d_f32_kernel(float* logits, int64_t ld, int rows, int V, const int64_t* target, const f32x2* live, const float* pm1,
                                                        const float* alpha, const float* h, int64_t ldh, int D, float* hm, int copies, LceTotal all) {
  const int first = rows * ((V + LCE_SEG - 1) / LCE_SEG);
  if ((int)blockIdx.x >= first + copies) {
    lce_total<256>(all);
    return;
  }
  if ((int)blockIdx.x >= first) {
    for (int64_t i = (int64_t)(blockIdx.x - first) * 256 + threadIdx.x; i < (int64_t)rows * D; i += (int64_t)copies * 256) {
      const int64_t n = i / D;
      hm[i] = live[n].y != 0.f ? h[n * ldh + (i - n * D)] : 0.f;
    }
    return;
  }
  const int segs = (V + LCE_SEG - 1) / LCE_SEG, n = blockIdx.x / segs, seg = blockIdx.x - n * segs;
  const f32x2 gl = live[n];
  const bool on = gl.y != 0.f;
  const int64_t t = target[n];
  const float al = alpha[0], f = al * gl.y, pt = al * pm1[n];
  float* x = logits + (int64_t)n * ld;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int v = seg * LCE_SEG + k * 1024 + threadIdx.x * 4;
    if (v >= V) break;
    f32x4 q = *reinterpret_cast<const f32x4*>(x + v);
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = on ? (v + e == t ? pt : f * lce_exp(q[e], gl.x)) : 0.f;
    *reinterpret_cast<f32x4*>(x + v) = q;
  }
}

// out[n][m] = sum of the split product's slabs [n][M], in their order
__global__ __launch_bounds__(256) void lce_fold_f32_kernel(const float* slabs, int64_t slab, int splits, int M, float* out, int64_t ldo) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < slab; i += (int64_t)gridDim.x * 256) {
    float v = slabs[i];
#pragma unroll 16
    for (int s = 1; s < splits; ++s) v += slabs[s * slab + i];
    const int64_t n = i / M;
    out[n * ldo + (i - n * M)] = v;
  }
}

// At most 16 rows: reading W once - writing dW once - is all there is to it.  The logits take one wave per block and no LDS: a
// lane's 16 bytes of W are four k-steps of v_mfma_f32_16x16x4_f32 (step s takes element s of every lane, of W and of h alike),
// and a wave has 16 of them on their way.  One row, width 2048, vocabulary 131072 (1.07 GB): logits 547 -> 241 us (4.5 TB/s), dW
// 557 -> 161 against the tiled products; dh by these means took what the tiled product with its K cut takes, 260.  With 17 to
// 64 rows the logits were slower: too few waves for their work.
template <bool VEC>
__device__ __forceinline__ f32x4 lce_load4(const float* p, int left) {               // elements [0, left) of 4, 0 for the others
  if (VEC) return left > 0 ? *reinterpret_cast<const f32x4*>(p) : f32x4{0.f, 0.f, 0.f, 0.f};
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) x[e] = p[e];
  return x;
}
// logits[n][v] = h w^T, 32 vocabulary entries per wave.  VEC: rows 16-byte aligned, of whole 16 bytes.
template <bool VEC>
__global__ __launch_bounds__(64) void lce_few_logits_kernel(const float* w, int64_t ldw, const float* h, int64_t ldh, int rows, int D, int V, float* out,
                                                            int64_t ldo) {
  constexpr int NI = 2, U = 8;
  const int l16 = threadIdx.x & 15, G = threadIdx.x >> 4, v0 = blockIdx.x * 16 * NI;
  const float *pw[NI], *ph = h + (int64_t)min(l16, rows - 1) * ldh + 4 * G;           // (past the last row: that row again, and not stored)
#pragma unroll
  for (int i = 0; i < NI; ++i) pw[i] = w + (int64_t)min(v0 + i * 16 + l16, V - 1) * ldw + 4 * G;
  f32x4 acc[NI] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  for (int k = 0; k < D; k += 16 * U) {
    f32x4 a[U][NI];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < NI; ++i) a[u][i] = lce_load4<VEC>(pw[i] + k + 16 * u, D - k - 16 * u - 4 * G);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const f32x4 b = lce_load4<VEC>(ph + k + 16 * u, D - k - 16 * u - 4 * G);
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int i = 0; i < NI; ++i) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[u][i][s], b[s], acc[i], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int v = v0 + i * 16 + 4 * G;                                 // (ldo is a multiple of 4 and holds V)
    if (l16 < rows && v < V) *reinterpret_cast<f32x4*>(out + (int64_t)l16 * ldo + v) = acc[i];
  }
}
// dw[v][c] (+)= sum over the rows of d[n][v] hm[n][c]: a wave keeps 4 columns of every row per lane and walks 16 vocabulary entries.
template <int NR, bool VEC>
__global__ __launch_bounds__(256) void lce_few_dw_kernel(const float* __restrict__ d, int64_t ldd, const float* __restrict__ hm, int rows, int D, int V, int add,
                                                         float* dw, int64_t lddw) {
  __shared__ __attribute__((aligned(16))) float dv[64][NR + 4];         // d of this block's 64 entries
  const int cols = (D + 255) / 256, vb = blockIdx.x / cols, c = (blockIdx.x - vb * cols) * 256 + (threadIdx.x & 63) * 4, left = D - c;
  for (int i = threadIdx.x; i < 64 * NR; i += 256) {
    const int n = i >> 6, v = vb * 64 + (i & 63);
    dv[i & 63][n] = n < rows && v < V ? d[(int64_t)n * ldd + v] : 0.f;
  }
  f32x4 x[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) x[n] = lce_load4<VEC>(hm + (int64_t)n * D + c, n < rows ? left : 0);
  __syncthreads();
  if (left <= 0) return;
  const int first = (threadIdx.x >> 6) * 16;
  for (int k = first; k < first + 16 && vb * 64 + k < V; ++k) {
    float* o = dw + (int64_t)(vb * 64 + k) * lddw + c;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NR; n += 4) {
      const f32x4 q = *reinterpret_cast<const f32x4*>(&dv[k][n]);
#pragma unroll
      for (int m = 0; m < 4; ++m) y += q[m] * x[n + m];
    }
    if (add) y += lce_load4<VEC>(o, left);
    if (VEC) {
      *reinterpret_cast<f32x4*>(o) = y;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) o[e] = y[e];
    }
  }
}

// M 16-bit words of each of N rows set to 0 (the gradient of no rows at all)
__global__ __launch_bounds__(256) void lce_zero_kernel(uint16_t* out, int64_t ld, int64_t N, int M) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < N * M; i += (int64_t)gridDim.x * 256) {
    const int64_t n = i / M;
    out[n * ld + (i - n * M)] = 0;
  }
}

__global__ __launch_bounds__(1024) void lce_total_kernel(LceTotal a) { lce_total<1024>(a); }

// ---- host ------------------------------------------------------------------------------------------------------------
static int64_t lce_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
static int lce_size(int dtype) { return dtype == DPC_F32 ? 4 : 2; }

// Tiles of a product.  256 x 256 where that makes enough of them; else 128 x 128, four times as many and three to a CU; a
// kernel of their own for few rows of logits.  Enough is half a round of the chip for
// the logits (width 1024: 500 x 18000, 142 tiles, 32 against 38 us, 256 x 18000, 71 tiles, 30 against 26), and for the
// gradients, whose K - vocabulary or rows - is cut into ranges, 192 of at least 1024 each (all of the call, width 256:
// 1531 x 18000, dW with 71, 129 against 124 us; 4096 x 18000, dW with 284, 227 against 248; dh with 4, 73 against 59).
enum { LCE_BIG = 0, LCE_MID = 1, LCE_ROW = 2 };
static int64_t lce_tiles(int64_t M, int64_t N, int64_t bm, int64_t bn) { return dpc_cdiv(M, bm) * dpc_cdiv(N, bn); }
static int lce_tile_logits(int64_t V, int64_t rows) {
  if (rows <= LCE_FEW) return LCE_ROW;
  return lce_tiles(V, rows, 256, 256) >= 128 ? LCE_BIG : LCE_MID;
}
static int lce_tile_grad(int64_t M, int64_t N, int64_t K) { return lce_tiles(M, N, 256, 256) * (K < 1024 ? 1 : K / 1024) >= 192 ? LCE_BIG : LCE_MID; }
static int lce_slab_rows(int kind) { return kind == LCE_BIG ? 128 : 64; }

// The tiles of a product that make whole rounds of the chip (256 CUs, `per` blocks each), and the K ranges of the others:
// as many as fill a round, none shorter than `least`, 32 at most; not cut at all where two would be (a round of them saves less
// than writing and adding up their sums costs).  (Loss and dh in bf16, 32 ranges at most against 128: 4 x 64 x 18000 29 against 31 us, 64 x 128 x
// 18000 35 both, but 4 x 128 x 131072 80 against 60, 100 x 512 x 131072 156 against 127.)
struct LceCut { int whole, splits; int64_t part; };
static LceCut lce_cut(int64_t tiles, int kind, int64_t K) {
  const int64_t slots = kind == LCE_BIG ? 256 : 512, least = kind == LCE_BIG ? 1024 : 512;
  const int64_t rest = tiles % slots;
  int64_t s = rest ? slots / rest : 1;
  if (s > K / least) s = K / least;
  if (s > 32) s = 32;
  LceCut c = {(int)tiles, 1, 0};
  if (s >= 2) {
    const int edge = kind == LCE_BIG ? 256 : 128;
    c.whole = (int)(tiles - rest);
    c.splits = (int)s;
    c.part = s * rest * edge * edge * 4;
  }
  return c;
}
static int lce_edge(int kind) { return kind == LCE_BIG ? 256 : 128; }

// Where things lie in the workspace for pieces of `rows` rows.
struct LceLayout {
  int64_t rows, prow;           // rows of a piece; padded to whole tiles
  int64_t stat, lt, live, pm1, P, ldp, hm, hp, two, part, acc, bytes;   // byte offsets (ldp: fp32 logits' row length), and the whole
  int tile_l, tile_h, tile_w;   // kinds of the three products' tiles
  int splits;                   // fp32: K ranges of dh
  int pieces;
};

static LceLayout lce_layout(int64_t T, int D, int V, int dtype, bool grads, bool dw16, int64_t rows) {
  LceLayout l;
  memset(&l, 0, sizeof(l));
  l.rows = rows < T ? rows : T;
  if (l.rows < 1) l.rows = 1;
  l.pieces = (int)dpc_cdiv(T < 1 ? 1 : T, l.rows);
  l.prow = lce_up(l.rows, 256);
  int64_t at = 256;                                                    // head
  const auto take = [&](int64_t bytes) { const int64_t o = at; at += lce_up(bytes, 256); return o; };
  l.lt = take(l.prow * 4);
  l.live = take(l.prow * 8);
  l.pm1 = take(l.prow * 4);
  l.splits = 1;
  if (dtype == DPC_F32) {
    l.ldp = lce_up(V, 4);
    l.stat = take(dpc_cdiv(V, LCE_SEG) * l.prow * 8);
    l.P = take(l.rows * l.ldp * 4);
    if (grads) {
      // 64 x 64 tiles, three to a CU; no range shorter than 256, none empty, 32 at most (loss and dh, 32 against 128: 100 x 512 x
      // 131072 324 against 327 us, 64 x 128 x 18000 42 against 40, 4 x 128 x 131072 100 against 55)
      const int64_t tiles = lce_tiles(D, l.rows, 64, 64), kt = dpc_cdiv(V, 32);
      int64_t s = 768 / tiles;
      if (s > V / 256) s = V / 256;
      if (s > 32) s = 32;
      if (s > 1) {
        l.splits = (int)dpc_cdiv(kt, dpc_cdiv(kt, s));
        l.part = take(l.splits * l.rows * (int64_t)D * 4);
      }
      l.hm = take(l.rows * (int64_t)D * 4);
    }
  } else {
    l.tile_l = lce_tile_logits(V, l.rows);
    l.stat = take(dpc_cdiv(V, lce_slab_rows(l.tile_l)) * l.prow * 8);
    // Rows that do not start on 64 bytes: a K-tile's 64 bytes of them lie across two lines of the cache every so often.  h is
    // small and laid out anew for the logits where they are at least 2^36 multiplications.  The loss alone, with the copy and
    // without: bf16 1531 x 1160 x 50021 181 against 187 us, 4096 x 1160 x 50021 450 against 474, 900 x 2040 x 50021 208 against
    // 218, 8192 x 1000 x 18000 284 against 293; below the limit, 1024 x 1160 x 50021 142 against 148, 400 x 2040 x 50021 108 against 117,
    // 600 x 520 x 50021 61 against 59, 256 x 1000 x 30000 38 against 39 (fp16 the same within 2 %): wide rows gain there too,
    // narrow ones lose, small calls neither.
    if (D % 32 != 0 && l.rows * D >= (1ll << 36) / V) l.hp = take(l.rows * lce_up(D, 32) * 2);
    if (grads) {
      l.P = take(lce_up(V, 256) * l.prow * 2);
      l.hm = take(l.prow * (int64_t)D * 2);
      if (l.tile_l == LCE_ROW) l.two = take(2 * LCE_FEW * (int64_t)D * 4);
      l.tile_h = lce_tile_grad(D, l.rows, V);
      l.tile_w = lce_tile_grad(D, V, l.prow);
      const LceCut h = lce_cut(lce_tiles(D, l.rows, lce_edge(l.tile_h), lce_edge(l.tile_h)), l.tile_h, V);
      const LceCut w = lce_cut(lce_tiles(D, V, lce_edge(l.tile_w), lce_edge(l.tile_w)), l.tile_w, l.prow);
      // (the last piece has fewer rows: fewer tiles of dh, then cut into more ranges - a round of them at most)
      const int64_t most = 256ll * 256 * 256 * 4;
      const int64_t part = l.pieces > 1 ? most : (h.part > w.part ? h.part : w.part);
      if (part) l.part = take(part);
      if (dw16 && l.pieces > 1) l.acc = take((int64_t)V * D * 4);
    }
  }
  l.bytes = at;
  return l;
}

static int lce_check(int64_t T, int D, int V, int dtype) {
  DPC_CHECK_ARG(T >= 0 && T < (1ll << 31) && D >= 1 && V >= 1 && V <= (1 << 28), "linear_cross_entropy: bad size");
  DPC_CHECK_ARG(dtype == DPC_F32 || dtype == DPC_BF16 || dtype == DPC_F16, "linear_cross_entropy: unknown element type");
  DPC_CHECK_ARG(dtype == DPC_F32 || D % 8 == 0, "linear_cross_entropy: half-precision rows need a width that is a multiple of 8");
  return DPC_OK;
}

#define LCE_ROWS (1 << 21)      // rows of a piece at most (half precision, gradients: P's chunks within 32-bit offsets)
// Rows of the largest piece: a launch has less than 2^32 threads.  512 for each 256 x 256 tile (and one for each row and slab), 64 for
// each row's slabs; fp32: 256 for 4096 logits of a row.
static int64_t lce_rows_most(int V, int dtype, bool grads) {
  if (dtype == DPC_F32) return ((1ll << 23) - 1) / dpc_cdiv(V, LCE_SEG);
  const int64_t tiles = ((1ll << 22) - 1) / dpc_cdiv(V, 256) * 256, rows = grads ? LCE_ROWS : ((1ll << 22) - 2) * 16;
  return tiles < rows ? tiles : rows;
}
// Rows of a piece where the caller names none: pieces of about the same size, whole tiles, of as many rows as 1 GiB - or twice
// the fp32 sums of dW, which each piece reads and writes - holds of what a row leaves (d, or the slabs' pairs alone); all of
// them where the sums would take the rest's place.  (32768 x 2048 x 131072 in pieces of 4096 rows 45.1 ms, of 8192 43.4, at once
// 43.6; 32768 x 1024 x 50021 in 4 x 8192 rows 9.5, in 3 x 10496 and 1280 10.6, at once 9.1.)
static int64_t lce_rows_default(int64_t T, int D, int V, int dtype, bool grads, bool dw16) {
  const int64_t row = grads || dtype == DPC_F32 ? (int64_t)V * lce_size(dtype) : dpc_cdiv(V, 64) * 8;
  const int64_t sums = grads ? 2 * (int64_t)V * D * 4 : 0, room = sums > (1ll << 30) ? sums : 1ll << 30;
  int64_t limit = lce_rows_most(V, dtype, grads);
  if (limit > LCE_ROWS) limit = LCE_ROWS;
  if (T <= limit && T * row <= room + (grads && dw16 ? (int64_t)V * D * 4 : 0)) return T < 1 ? 1 : T;
  if (limit < 256) return limit;                                       // (fp32, V from 2^27 on)
  int64_t most = room / row;
  most = most < 256 ? 256 : (most > limit ? limit : most) / 256 * 256;
  const int64_t pieces = dpc_cdiv(T, most);
  return lce_up(dpc_cdiv(T, pieces), 256);
}

// Whether the sizes and the piece, as the caller names it or by default, are ones that a call takes.
static int lce_check_piece(int64_t T, int D, int V, int dtype, bool grads, bool dw16, int64_t& piece_rows) {
  const int rc = lce_check(T, D, V, dtype);
  if (rc != DPC_OK) return rc;
  if (piece_rows <= 0) piece_rows = lce_rows_default(T, D, V, dtype, grads, dw16);
  DPC_CHECK_ARG((piece_rows < T ? piece_rows : T) <= lce_rows_most(V, dtype, grads) && (dtype == DPC_F32 || dpc_cdiv(V, 256) * dpc_cdiv(D, 256) < (1ll << 22)),
                "linear_cross_entropy: the piece is too large");
  return DPC_OK;
}

extern "C" int64_t dpc_linear_cross_entropy_ws(int64_t T, int D, int V, int dtype, int grads, int dw_f32, int64_t piece_rows) {
  if (lce_check_piece(T, D, V, dtype, grads != 0, dtype != DPC_F32 && !dw_f32, piece_rows) != DPC_OK) return -1;
  return lce_layout(T, D, V, dtype, grads != 0, dtype != DPC_F32 && !dw_f32, piece_rows).bytes;
}

template <typename E, int MODE, int BM, int BN, int WM, int WN>
static void lce_launch_tile(LceArgs& g, int kind, hipStream_t st) {
  g.tiles_m = (int)dpc_cdiv(g.M, BM);
  g.tiles_n = (int)dpc_cdiv(g.N, BN);
  const int tiles = g.tiles_m * g.tiles_n;
  const LceCut c = MODE == LCE_LOGITS ? LceCut{tiles, 1, 0} : lce_cut(tiles, kind, g.K);
  g.whole = c.whole;
  g.splits = c.splits;
  g.kchunk = (int)lce_up(dpc_cdiv(g.K, g.splits), LCE_BK);
  hipLaunchKernelGGL((lce_product_kernel<E, MODE, BM, BN, WM, WN>), dim3(g.whole + (tiles - g.whole) * g.splits), dim3(WM * WN * 64), 0, st, g);
  if (MODE != LCE_LOGITS && g.whole < tiles)
    hipLaunchKernelGGL((lce_fold_kernel<E, BM, BN>), dim3((tiles - g.whole) * (BM * BN / 1024)), dim3(256), 0, st, g);
}
template <typename E, int MODE>
static void lce_launch(LceArgs& g, int kind, hipStream_t st) {
  if (kind == LCE_BIG) lce_launch_tile<E, MODE, 256, 256, MODE == LCE_LOGITS ? 2 : 4, MODE == LCE_LOGITS ? 4 : 2>(g, kind, st);
  else if (kind == LCE_MID) lce_launch_tile<E, MODE, 128, 128, 2, 2>(g, kind, st);
  else if constexpr (MODE == LCE_LOGITS) hipLaunchKernelGGL(lce_few_kernel<E>, dim3((unsigned)dpc_cdiv(g.M, 64)), dim3(64), 0, st, g);
}

struct LceCall {
  const char* h; int64_t ldh; const char* w; int64_t ldw;
  int dtype; const int64_t* target; int64_t ignore; int64_t T; int D, V;
  float* loss; float* lse; float* total;
  char* dh; int64_t lddh; char* dw; int64_t lddw; int dw_f32, accumulate;
  float gscale; int mean;
  char* ws;
};

static LceTotal lce_all(const LceCall& c) { return LceTotal{c.loss, c.target, c.T, c.ignore, c.mean, c.total}; }
// Whether piece `p` takes the total in the pass between the products.
static int lce_takes_total(const LceCall& c, const LceLayout& l, int p) { return c.total && p + 1 == l.pieces && !(c.T <= 16 && l.pieces == 1); }

// Rows of a piece: with the first one's the call's alpha, and the total where one block sees all rows.
static void lce_rows(const LceCall& c, LceRowArgs& a, int piece, const LceLayout& l, hipStream_t st) {
  const bool begin = piece == 0 && (c.dh || c.dw);
  a.alpha = begin ? (float*)c.ws : nullptr;
  a.scale = c.dtype == DPC_F16 ? c.gscale / Half<_Float16>::kUp : c.gscale;
  a.mean = c.mean; a.all = c.target; a.T = c.T;
  a.total = c.T <= 16 && l.pieces == 1 ? c.total : nullptr;
  hipLaunchKernelGGL(lce_rows_kernel, dim3((unsigned)dpc_cdiv(a.rows, 16) + begin), dim3(1024), 0, st, a);
}

template <typename E>
static int lce_half(const LceCall& c, const LceLayout& l, hipStream_t st) {
  float* head = (float*)c.ws;
  const bool grads = c.dh || c.dw;
  const int slab_rows = lce_slab_rows(l.tile_l), slabs = (int)dpc_cdiv(c.V, slab_rows);
  for (int p = 0; p < l.pieces; ++p) {
    const int64_t r0 = p * l.rows;
    const int rows = (int)(c.T - r0 < l.rows ? c.T - r0 : l.rows);
    const char* h = c.h + r0 * c.ldh * 2;
    LceArgs g;
    memset(&g, 0, sizeof(g));
    g.P = c.ws + l.P; g.prow = l.prow; g.alpha = head; g.target = c.target + r0;
    g.stat = (f32x2*)(c.ws + l.stat); g.lt = (float*)(c.ws + l.lt); g.grads = grads;
    g.A = c.w; g.lda = c.ldw * 2; g.B = h; g.ldb = c.ldh * 2;
    if (l.hp && (((uintptr_t)h | (uintptr_t)g.ldb) & 63)) {
      g.B = c.ws + l.hp; g.ldb = lce_up(c.D, 32) * 2;
      hipLaunchKernelGGL(lce_pitch_kernel, dim3(dpc_grid((int64_t)rows * (c.D / 8), 256)), dim3(256), 0, st, h, c.ldh * 2, rows, c.D / 8, c.ws + l.hp, g.ldb);
    }
    g.M = c.V; g.N = rows; g.K = c.D;
    lce_launch<E, LCE_LOGITS>(g, l.tile_l, st);
    LceRowArgs ra;
    ra.stat = g.stat; ra.prow = l.prow; ra.slabs = slabs; ra.rows = rows; ra.V = c.V; ra.lt = g.lt; ra.target = g.target; ra.ignore = c.ignore;
    ra.loss = c.loss + r0; ra.lse = c.lse ? c.lse + r0 : nullptr;
    ra.live = grads ? (f32x2*)(c.ws + l.live) : nullptr; ra.pm1 = (float*)(c.ws + l.pm1);
    lce_rows(c, ra, p, l, st);
    if (!grads) continue;
    const int row16 = c.D / 8;
    const bool few = l.tile_l == LCE_ROW;
    char* hm = c.ws + l.hm;
    if (few) {
      const int copies = c.dw ? dpc_grid(LCE_FEW * row16, 256) : 0;
      hipLaunchKernelGGL(lce_few_scale_kernel<E>, dim3((unsigned)(dpc_cdiv(slabs, 2) + copies + lce_takes_total(c, l, p))), dim3(256), 0, st, g.P, l.prow,
                         g.stat, slabs, rows, ra.live, ra.pm1, g.target, h, c.ldh * 2, row16, hm, copies, lce_all(c));
    } else {
      const auto scale = lce_up(c.V, 256) * l.prow * 2 > (1ll << 30) ? lce_scale_kernel<E, true> : lce_scale_kernel<E, false>;
      const int copies = c.dw ? dpc_grid(l.prow * row16, 256) : 0;
      hipLaunchKernelGGL(scale, dim3((unsigned)(l.prow / 256 * slabs + copies + lce_takes_total(c, l, p))), dim3(256), 0, st, g.P, l.prow, g.stat, slabs, rows,
                         slab_rows, ra.live, ra.pm1, g.target, h, c.ldh * 2, row16, hm, copies, lce_all(c));
    }
    if (c.dh) {
      LceArgs d = g;
      d.A = c.w; d.lda = c.ldw * 2; d.M = c.D; d.N = rows; d.K = c.V;
      E* dh = (E*)c.dh + r0 * c.lddh;
      float* two = (float*)(c.ws + l.two);
      d.C = few ? (void*)two : (void*)dh; d.ldc = few ? c.D : c.lddh; d.c_f32 = few; d.part = (float*)(c.ws + l.part);
      if (few) d.N = 2 * LCE_FEW;
      lce_launch<E, LCE_DH>(d, l.tile_h, st);
      if (few) hipLaunchKernelGGL(lce_few_join_kernel<E>, dim3(dpc_grid((int64_t)rows * c.D, 256)), dim3(256), 0, st, two, rows, c.D, dh, c.lddh);
    }
    if (c.dw) {
      LceArgs d = g;
      d.A = hm; d.lda = (int64_t)c.D * 2; d.M = c.D; d.N = c.V; d.K = few ? 2 * LCE_FEW : (int)lce_up(rows, LCE_BK); d.part = (float*)(c.ws + l.part);
      // where the piece's share goes: dW itself, or the fp32 sums over the pieces until the last one
      const bool last = p + 1 == l.pieces, via = !c.dw_f32 && l.pieces > 1;
      float* acc = (float*)(c.ws + l.acc);
      d.add = via ? (p > 0 ? acc : nullptr) : (c.dw_f32 && (p > 0 || c.accumulate) ? (const float*)c.dw : nullptr);
      d.ldadd = via ? c.D : c.lddw;
      d.C = via && !last ? (void*)acc : (void*)c.dw;
      d.ldc = via && !last ? c.D : c.lddw;
      d.c_f32 = via ? !last : c.dw_f32;
      lce_launch<E, LCE_DW>(d, l.tile_w, st);
    }
  }
  return DPC_OK;
}

// fp32: the framework's own products (no split with atomics: the sums keep one order)
static dpc_gemm_desc lce_desc(int M, int N, int K, const float* A, int64_t a_rs, int64_t a_cs, const float* B, int64_t b_rs, int64_t b_cs, float beta,
                              float* C, int64_t ldc) {
  dpc_gemm_desc d;
  memset(&d, 0, sizeof(d));
  d.M = M; d.N = N; d.K = K; d.alpha = 1.f; d.beta = beta; d.A = A; d.a_rs = a_rs; d.a_cs = a_cs; d.B = B; d.b_rs = b_rs; d.b_cs = b_cs;
  d.C = C; d.ldc = ldc; d.splitk = 1;
  return d;
}
static int lce_full(const LceCall& c, const LceLayout& l, hipStream_t st) {
  float* head = (float*)c.ws;
  const bool grads = c.dh || c.dw;
  for (int p = 0; p < l.pieces; ++p) {
    const int64_t r0 = p * l.rows;
    const int rows = (int)(c.T - r0 < l.rows ? c.T - r0 : l.rows);
    const float* h = (const float*)c.h + r0 * c.ldh;
    const float* w = (const float*)c.w;
    float* P = (float*)(c.ws + l.P);
    float* hm = (float*)(c.ws + l.hm);
    const int segs = (int)dpc_cdiv(c.V, LCE_SEG);
    LceRowArgs ra;
    memset(&ra, 0, sizeof(ra));
    ra.stat = (f32x2*)(c.ws + l.stat); ra.prow = l.prow; ra.slabs = segs; ra.rows = rows; ra.V = c.V; ra.lt = (float*)(c.ws + l.lt);
    ra.target = c.target + r0; ra.ignore = c.ignore; ra.loss = c.loss + r0; ra.lse = c.lse ? c.lse + r0 : nullptr;
    ra.live = grads ? (f32x2*)(c.ws + l.live) : nullptr; ra.pm1 = (float*)(c.ws + l.pm1);
    const bool few = l.rows <= LCE_FEW;
    const bool vec = (((uintptr_t)h | (uintptr_t)w) & 15) == 0 && ((c.ldh | c.ldw | c.D) & 3) == 0;
    int rc = DPC_OK;
    if (few) {
      const auto k = vec ? lce_few_logits_kernel<true> : lce_few_logits_kernel<false>;
      hipLaunchKernelGGL(k, dim3((unsigned)dpc_cdiv(c.V, 32)), dim3(64), 0, st, w, c.ldw, h, c.ldh, rows, c.D, c.V, P, l.ldp);
    } else {
      // (64 x 64 tiles below 1024 of 128 x 128: 500 x 18000 x 256 55 against 70 us, 700 x 18000 x 1024 226 against 259; 4096 x
      // 5000 x 512 193 against 180, 3000 x 18000 x 1024 940 against 884)
      dpc_gemm_desc lg = lce_desc(rows, c.V, c.D, h, c.ldh, 1, w, 1, c.ldw, 0.f, P, l.ldp);
      lg.tile = lce_tiles(rows, c.V, 128, 128) < 1024 ? 64 : 128;
      rc = dpc_gemm_f32_ex(&lg, 1, st);
    }
    if (rc != DPC_OK) return rc;
    hipLaunchKernelGGL(lce_stat_f32_kernel, dim3((unsigned)segs * rows), dim3(256), 0, st, P, l.ldp, c.V, ra.target, (f32x2*)(c.ws + l.stat), l.prow,
                       (float*)(c.ws + l.lt));
    lce_rows(c, ra, p, l, st);
    if (!grads) continue;
    const int copies = c.dw ? dpc_grid((int64_t)rows * c.D, 256) : 0;
    hipLaunchKernelGGL(lce_d_f32_kernel, dim3((unsigned)segs * rows + copies + lce_takes_total(c, l, p)), dim3(256), 0, st, P, l.ldp, rows, c.V, ra.target, ra.live,
                       ra.pm1, head, h, c.ldh, c.D, hm, copies, lce_all(c));
    if (c.dh) {
      float* dh = (float*)c.dh + r0 * c.lddh;
      const bool cut = l.splits > 1;
      const int64_t slab = (int64_t)rows * c.D;
      dpc_gemm_desc d = lce_desc(rows, c.D, c.V, P, l.ldp, 1, w, c.ldw, 1, 0.f, cut ? (float*)(c.ws + l.part) : dh, cut ? c.D : c.lddh);
      if (cut) { d.splitk = l.splits; d.tile = 64; d.split_slab = slab; }
      rc = dpc_gemm_f32_ex(&d, 1, st);
      if (rc != DPC_OK) return rc;
      if (cut)
        hipLaunchKernelGGL(lce_fold_f32_kernel, dim3(dpc_grid(slab, 256)), dim3(256), 0, st, (const float*)(c.ws + l.part), slab, l.splits, c.D, dh, c.lddh);
    }
    if (c.dw && few) {
      const bool wide = ((uintptr_t)c.dw & 15) == 0 && ((c.lddw | c.D) & 3) == 0;
      const auto k = rows <= 4 ? (wide ? lce_few_dw_kernel<4, true> : lce_few_dw_kernel<4, false>)
                               : (wide ? lce_few_dw_kernel<16, true> : lce_few_dw_kernel<16, false>);
      hipLaunchKernelGGL(k, dim3((unsigned)(dpc_cdiv(c.D, 256) * dpc_cdiv(c.V, 64))), dim3(256), 0, st, P, l.ldp, hm, rows, c.D, c.V, p > 0 || c.accumulate,
                         (float*)c.dw, c.lddw);
    } else if (c.dw) {
      // (64 x 64 tiles: 2 to 9 % less than the product's own choice at 500 x 256 x 18000, 700 x 1024 x 18000, 4096 x 512 x 5000)
      dpc_gemm_desc d = lce_desc(c.V, c.D, rows, P, 1, l.ldp, hm, c.D, 1, p > 0 || c.accumulate ? 1.f : 0.f, (float*)c.dw, c.lddw);
      d.tile = 64;
      rc = dpc_gemm_f32_ex(&d, 1, st);
      if (rc != DPC_OK) return rc;
    }
  }
  return DPC_OK;
}

// Rows of `width` bytes every `pitch` bytes, and whether two such lie over each other anywhere.
struct LceSpan { uintptr_t at; int64_t rows, width, pitch; };
static LceSpan lce_span(const void* p, int64_t rows, int64_t width, int64_t pitch) { return LceSpan{(uintptr_t)p, p && width ? rows : 0, width, pitch}; }
static bool lce_row_meets(uintptr_t at, int64_t width, const LceSpan& y) {
  const int64_t from = (int64_t)(at - y.at) - y.width;                 // the first row of y that ends behind `at`
  const int64_t j = from < 0 ? 0 : from / y.pitch + 1;
  return j < y.rows && y.at + j * y.pitch < at + width;
}
static bool lce_meet(const LceSpan& x, const LceSpan& y) {
  if (x.rows <= 0 || y.rows <= 0) return false;
  if (x.at + (x.rows - 1) * x.pitch + x.width <= y.at || y.at + (y.rows - 1) * y.pitch + y.width <= x.at) return false;
  if (x.rows > y.rows) return lce_meet(y, x);
  // (of one pitch: rows that meet are the same number of rows apart everywhere, so one of them is a first row somewhere)
  if (x.pitch == y.pitch) return lce_row_meets(x.at, x.width, y) || lce_row_meets(y.at, y.width, x);
  for (int64_t i = 0; i < x.rows; ++i)
    if (lce_row_meets(x.at + i * x.pitch, x.width, y)) return true;
  return false;
}

extern "C" int dpc_linear_cross_entropy(const void* h, int64_t ldh, const void* w, int64_t ldw, int dtype, const int64_t* target,
                                        int64_t ignore_index, int64_t T, int D, int V, float* loss, float* lse, float* total, void* dh,
                                        int64_t lddh, void* dw, int64_t lddw, int dw_f32, int accumulate, float gscale, int mean,
                                        int64_t piece_rows, void* ws, int64_t ws_bytes, void* stream) {
  const bool f32 = dtype == DPC_F32, grads = dh || dw;
  const int rc0 = lce_check_piece(T, D, V, dtype, grads, !f32 && !dw_f32, piece_rows);
  if (rc0 != DPC_OK) return rc0;
  DPC_CHECK_ARG(w && ws && (T == 0 || (h && target && loss)), "linear_cross_entropy: null pointer");
  DPC_CHECK_ARG(ldh >= D && ldw >= D && (!dh || lddh >= D) && (!dw || lddw >= D), "linear_cross_entropy: a leading dimension is smaller than the width");
  DPC_CHECK_ARG(!accumulate || (dw && (dw_f32 || dtype == DPC_F32)), "linear_cross_entropy: accumulation goes into an fp32 dw");
  if (!f32) {
    const uintptr_t al = (uintptr_t)h | (uintptr_t)w | (uintptr_t)dh | (uintptr_t)dw | (uintptr_t)(ldh * 2) | (uintptr_t)(ldw * 2);
    DPC_CHECK_ARG((al & 15) == 0, "linear_cross_entropy: half-precision rows must be 16-byte aligned");
    DPC_CHECK_ARG(ldh < (1 << 21) && ldw < (1 << 21), "linear_cross_entropy: rows are too long");     // (256 rows within 32-bit offsets)
    DPC_CHECK_ARG((!dh || lddh % 8 == 0) && (!dw || lddw % (dw_f32 ? 4 : 8) == 0), "linear_cross_entropy: gradient rows must be 16-byte aligned");
  }
  DPC_CHECK_ARG(((uintptr_t)ws & 255) == 0, "linear_cross_entropy: the workspace must be 256-byte aligned");
  const LceLayout l = lce_layout(T, D, V, dtype, grads, !f32 && !dw_f32, piece_rows);
  const int64_t size = lce_size(dtype), size_w = dw_f32 ? 4 : size;
  const LceSpan spans[] = {lce_span(ws, 1, l.bytes, l.bytes), lce_span(loss, 1, T * 4, T * 4), lce_span(lse, 1, T * 4, T * 4), lce_span(total, 1, 4, 4),
                           lce_span(dh, T, D * size, lddh * size), lce_span(dw, V, D * size_w, lddw * size_w),                 // what is written: 6
                           lce_span(h, T, D * size, ldh * size), lce_span(w, V, D * size, ldw * size), lce_span(target, 1, T * 8, T * 8)};
  for (int i = 0; i < 6; ++i)
    for (int j = i + 1; j < 9; ++j)
      DPC_CHECK_ARG(!lce_meet(spans[i], spans[j]), "linear_cross_entropy: an output or the workspace must not lie over an operand or another output");
  DPC_CHECK_ARG(ws_bytes >= l.bytes, "linear_cross_entropy: the workspace is smaller than dpc_linear_cross_entropy_ws says");
  hipStream_t st = (hipStream_t)stream;
  LceCall c;
  c.h = (const char*)h; c.ldh = ldh; c.w = (const char*)w; c.ldw = ldw; c.dtype = dtype; c.target = target; c.ignore = ignore_index; c.T = T;
  c.D = D; c.V = V; c.loss = loss; c.lse = lse; c.total = total; c.dh = (char*)dh; c.lddh = lddh; c.dw = (char*)dw; c.lddw = lddw;
  c.dw_f32 = dw_f32 || f32; c.accumulate = accumulate; c.gscale = gscale; c.mean = mean; c.ws = (char*)ws;
  if (T == 0 && dw && !accumulate)
    hipLaunchKernelGGL(lce_zero_kernel, dim3(dpc_grid((int64_t)V * D, 256)), dim3(256), 0, st, (uint16_t*)dw, c.dw_f32 ? 2 * lddw : lddw, (int64_t)V,
                       c.dw_f32 ? 2 * D : D);
  const int rc = T == 0 ? DPC_OK : f32 ? lce_full(c, l, st) : (dtype == DPC_BF16 ? lce_half<__bf16>(c, l, st) : lce_half<_Float16>(c, l, st));
  if (rc != DPC_OK) return rc;
  if (total && (T == 0 || (!grads && (T > 16 || l.pieces > 1)))) hipLaunchKernelGGL(lce_total_kernel, dim3(1), dim3(1024), 0, st, lce_all(c));
  DPC_LAUNCH_CHECK();
  return DPC_OK;
}
