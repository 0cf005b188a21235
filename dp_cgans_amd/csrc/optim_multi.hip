// Many tensors in one launch: the global gradient norm with its clip factor, and a decoupled-weight-decay Adam step
// with states in 32 or in 8 bits.  A PLAN (device memory of the caller) lists the tensors and cuts them into chunks;
// block b of a launch works on chunk b, so a launch costs the same for one tensor as for hundreds.
#include "dpc_common.h"
#include "../../include/dpcgan_hip.h"
#include <math.h>
#include <string.h>

#define MT_BLOCK8 128           // elements that share one scale of an 8-bit state = 16 lanes x 8 elements
#define MT_SUB 2048             // elements one block handles per pass: 256 threads x 8

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// One tensor of a plan, as the kernels see it.
struct MtRec {
  void* p; const void* g; void* m; void* v;
  float* ms; float* vs;                 // scales of the 8-bit states (null: 32-bit states)
  void* cp;
  const uint16_t* dith;
  int64_t n;
  int64_t draw8;                        // first Philox block of this tensor (one block per 8 elements)
  int32_t p_t, g_t, c_t;
  float wd;
  int32_t vec;                          // 8-element accesses are aligned in every buffer
  int32_t pad;
};
// Chunk b of a plan: elements [start, start + MT_SUB) of tensor t.
struct MtChunk { int32_t t; int32_t pad; int64_t start; };

struct MtPlan { const MtRec* rec; const MtChunk* chunk; int blocks; };

#define MT_GROUPS 16             // groups of blocks that count their ends apart, each on a line of its own
#define MT_LINE 64               // words between two counts
#define MT_COUNTS 4608           // bytes of the counts, (1 + MT_GROUPS) lines

static int64_t mt_align(int64_t x) { return (x + 255) & ~(int64_t)255; }

// 8 consecutive elements, as loaded: two halves of fp32, one of 16 bits.  Loading and converting are apart so that a
// block has all its loads in flight before the first wait (the element types are branches the whole block takes).
struct Raw8 { u32x4 a, b; };
template <bool FULL>
__device__ __forceinline__ Raw8 mt_load(const void* base, int64_t i, int type, int left) {
  Raw8 o = {u32x4{0u, 0u, 0u, 0u}, u32x4{0u, 0u, 0u, 0u}};
  if (type == DPC_F32) {
    const uint32_t* q = (const uint32_t*)base + i;
    if (FULL) {
      o.a = reinterpret_cast<const u32x4*>(q)[0];
      o.b = reinterpret_cast<const u32x4*>(q)[1];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) { if (e < 4) o.a[e] = q[e]; else o.b[e - 4] = q[e]; }
    }
  } else {
    const uint16_t* q = (const uint16_t*)base + i;
    if (FULL) {
      o.a = *reinterpret_cast<const u32x4*>(q);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) o.a[e >> 1] |= (uint32_t)q[e] << (16 * (e & 1));
    }
  }
  return o;
}
__device__ __forceinline__ f32x8 mt_float(const Raw8& r, int type) {
  if (type == DPC_F32) {
    const f32x4 a = __builtin_bit_cast(f32x4, r.a), b = __builtin_bit_cast(f32x4, r.b);
    return f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  }
  if (type == DPC_BF16) return __builtin_convertvector(__builtin_bit_cast(bf16x8, r.a), f32x8);
  return __builtin_convertvector(__builtin_bit_cast(f16x8, r.a), f32x8);
}

template <bool FULL>
__device__ __forceinline__ void mt_store(void* base, int64_t i, int type, int left, f32x8 x) {
  if (FULL) {
    if (type == DPC_F32) {
      f32x4* q = reinterpret_cast<f32x4*>((float*)base + i);
      q[0] = f32x4{x[0], x[1], x[2], x[3]};
      q[1] = f32x4{x[4], x[5], x[6], x[7]};
    } else if (type == DPC_BF16) {
      *reinterpret_cast<bf16x8*>((uint16_t*)base + i) = __builtin_convertvector(x, bf16x8);
    } else {
      *reinterpret_cast<f16x8*>((uint16_t*)base + i) = __builtin_convertvector(x, f16x8);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (e < left) {
      if (type == DPC_F32) ((float*)base)[i + e] = x[e];
      else if (type == DPC_BF16) ((__bf16*)base)[i + e] = (__bf16)x[e];
      else ((_Float16*)base)[i + e] = (_Float16)x[e];
    }
  }
}

// ---- global norm ---------------------------------------------------------------------------------------------------
// out = {norm, coef} from the partial sums; a norm that is not finite gives coef 0 (the step that reads it is not taken) and
// leaves *t alone.
struct ClipArgs { double max_norm, gscale; float* out; int32_t* t; };
__device__ __forceinline__ void grad_clip_finish(const double* part, int n, const ClipArgs& a, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 256)
    s += __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<const uint64_t*>(part) + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  s = dpc_block_sum(s, red);
  if (threadIdx.x == 0) {
    const double norm = a.gscale * sqrt(s);
    const bool ok = norm <= 1.7976931348623157e308;        // false for NaN too
    a.out[0] = (float)norm;
    // (never 0 for a finite norm, however small the factor: 0 skips the step)
    a.out[1] = ok ? fmaxf((float)(norm > a.max_norm ? a.gscale * (a.max_norm / norm) : a.gscale), 1.17549435e-38f) : 0.f;
    if (ok && a.t) *a.t += 1;
  }
}
__global__ __launch_bounds__(256) void grad_clip_none_kernel(ClipArgs a) {      // (a plan without elements: norm 0)
  __shared__ double red[16];
  grad_clip_finish(nullptr, 0, a, red);
}

// sum of g^2 in fp64 (the square of an fp32 gradient overflows at 2e19 and vanishes below 1e-23): one partial per
// block, chunks b, b + gridDim, ... in that order; the block that ends last adds up the partials, in theirs, so the sum does
// not depend on which one that is (with a second launch for it a call took the host 7.0 us instead of 3.5, the GPU as long).
// What crosses between blocks is written through and read past the XCDs' own L2s, word by word: an acquire and a release,
// which write back and empty an L2 for every block, made the norm of 0.8 GB 208 us long instead of 124.
// NT: the gradients are larger than the 256 MB of the last-level cache and are read past it.
template <bool NT>
__device__ __forceinline__ Raw8 mt_load_norm(const MtRec& r, int64_t i, int64_t end, bool full) {
  if (!full) return mt_load<false>(r.g, i, r.g_t, (int)max((int64_t)0, min((int64_t)8, end - i)));
  Raw8 o = {u32x4{0u, 0u, 0u, 0u}, u32x4{0u, 0u, 0u, 0u}};
  const u32x4* q = reinterpret_cast<const u32x4*>((const char*)r.g + i * (r.g_t == DPC_F32 ? 4 : 2));
  o.a = NT ? __builtin_nontemporal_load(q) : q[0];
  if (r.g_t == DPC_F32) o.b = NT ? __builtin_nontemporal_load(q + 1) : q[1];
  return o;
}
__device__ __forceinline__ uint32_t mt_add(uint32_t* p) { return __hip_atomic_fetch_add(p, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void mt_put(uint32_t* p, uint32_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <bool NT>
__global__ __launch_bounds__(256) void grad_clip_kernel(MtPlan pl, double* part, uint32_t* ended, ClipArgs a) {
  __shared__ double red[16];
  __shared__ bool last;
  double s = 0.0;
  // four chunks at a time: their loads are in flight together
  for (int c0 = blockIdx.x * 4; c0 < pl.blocks; c0 += gridDim.x * 4) {
    Raw8 raw[4];
    int type[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const MtChunk ch = pl.chunk[min(c0 + k, pl.blocks - 1)];
      const MtRec r = pl.rec[ch.t];
      const int64_t end = c0 + k < pl.blocks ? min(ch.start + MT_SUB, r.n) : ch.start;         // (past the last chunk: nothing of it)
      type[k] = r.g_t;
      raw[k] = mt_load_norm<NT>(r, ch.start + 8 * threadIdx.x, end, r.vec && end - ch.start >= MT_SUB);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x8 g = mt_float(raw[k], type[k]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fma((double)g[e], (double)g[e], s);
    }
  }
  s = dpc_block_sum(s, red);
  if (threadIdx.x == 0) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(part) + blockIdx.x, __builtin_bit_cast(uint64_t, s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                   // (written through: it is there for every XCD)
    // (counted in MT_GROUPS groups, then the groups: adds to one word follow one another, 10 ns each)
    const uint32_t group = blockIdx.x % MT_GROUPS, groups = min(gridDim.x, (uint32_t)MT_GROUPS), size = (gridDim.x - group + MT_GROUPS - 1) / MT_GROUPS;
    uint32_t* own = ended + (1 + group) * MT_LINE;
    last = false;
    if (mt_add(own) + 1 == size) {
      mt_put(own, 0u);                                                 // for the next call
      last = mt_add(ended) + 1 == groups;
      if (last) mt_put(ended, 0u);
    }
  }
  __syncthreads();
  if (!last) return;
  grad_clip_finish(part, gridDim.x, a, red);
}

// ---- AdamW ---------------------------------------------------------------------------------------------------------
struct AdamwArgs {
  MtPlan pl;
  float lr, b1, b2, c1, c2, eps;        // c = 1 - b, taken in fp64
  float eps8;                           // eps, but a normal number
  double b1d, b2d, c1d, c2d;
  float step_size, inv_bc2s;            // lr / (1 - b1^t), 1 / sqrt(1 - b2^t) where the step count is the host's
  const float* coef; float gscale;
  const int32_t* t_dev; int t_host;
  const uint64_t* rng; uint32_t site;
};

// The parameter after a step of `up` and a decay by `decay` = lr wd: what leaves it is added up before its one rounding.  (A
// factor 1 - decay is a multiple of 2^-24: 1.5 % off at a decay of 2e-6, 19 % at 1e-7, 1 below 3e-8.)  The clamp keeps an infinite
// parameter infinite.  Contraction off here and below: the vector and the element-wise paths give the same bits.
__device__ __forceinline__ float adamw_param(float p, float up, float decay) {
#pragma clang fp contract(off)
  return p - (decay * __builtin_amdgcn_fmed3f(p, -3.402823466e38f, 3.402823466e38f) + up);
}

// ---- 8-bit states.  The moments are updated in fp64 from what is held and rounded ONCE, to 4 significant bits, so what
// is held is the exact rounding for the given random bits (an update in fp32 lands on the other side of a border for one
// element in 10^6).  The vector units bound this - the counters show them busy all the time - so it is written for few
// instructions: 66 M parameters in bf16 took 205 us with a library square root and every case of the rounding per element,
// 186 us with the hardware's reciprocal root, 156 us with the usual case on its own.
struct Hold8 { double x[8]; };

#define MT_ONE8 0x3f900000u      // high word of 2^-6, the smallest normal e4m3 number (code 8)
#define MT_BIAS8 (1016u << 20)   // fp64's exponent bias less e4m3's, where the high word has its exponent
#define MT_SOME 1e-300           // added to a second moment: 0 becomes a number with a root

// sqrt(v) to 2^-46, v >= MT_SOME: the hardware's reciprocal root (2^-24, the whole range of fp64) and one Newton step.
// NaN for infinities and NaN, which are held as NaN anyway.
__device__ __forceinline__ double mt_root(double v) {
  const double q = __builtin_amdgcn_rsq(v), r = v * q;
  return fma(fma(-r, r, v), 0.5 * q, r);
}

// Largest of a value over the 16 lanes that hold a state block (rotations inside a DPP row).
template <int CTRL>
__device__ __forceinline__ double mt_ror(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double mt_max16(double v) {
  v = fmax(v, mt_ror<0x128>(v));
  v = fmax(v, mt_ror<0x124>(v));
  v = fmax(v, mt_ror<0x122>(v));
  return fmax(v, mt_ror<0x121>(v));
}

template <bool FULL>
__device__ __forceinline__ u32x2 mt_load8(const void* base, int64_t i, int left) {
  if (FULL) return *reinterpret_cast<const u32x2*>((const uint8_t*)base + i);
  u32x2 q = {0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < left) q[e >> 2] |= (uint32_t)((const uint8_t*)base)[i + e] << (8 * (e & 3));
  return q;
}
__device__ __forceinline__ f32x8 mt_float8(u32x2 q) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(q.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(q.x, true);
  const f32x2 c = __builtin_amdgcn_cvt_pk_f32_fp8(q.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8(q.y, true);
  return f32x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// 448 / top a little up (2^-48): top times it is not below 448.
__device__ __forceinline__ double mt_scale8(double top) {
  double q = __builtin_amdgcn_rcp(top);
  q = fma(fma(-top, q, 1.0), q, q);
  q = fma(fma(-top, q, 1.0), q, q);
  return q * (448.0 * (1.0 + 0x1p-48));
}

// Hold the 8 values x of this lane, part of a 128-element block, in 8 bits: the block's largest finite value as 448, the
// largest e4m3 number; the others y = 448 x / largest as the code below or above, above where the fraction between them
// plus d / 65536 reaches 1: 2 d (`d2`, less the exponents' biases) is added to the high word of the fp64 number, whose lowest
// 17 bits go; the carry rounds up.  ROOT: the value is a square root, not negative, and not held as 0 unless it is 0 (a
// root held as 0 would divide its moment by eps alone).
// The usual case has normal numbers only.  `odd`: some value of this wave is not finite.
template <bool FULL, bool ROOT>
__device__ __forceinline__ void mt_hold8(void* base, float* scales, int64_t i, int left, const Hold8& h, const uint32_t d2[8], bool odd) {
  double top = 0.0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = fmax(top, fabs(h.x[e]));
  const double most = 3.4028234663852886e38, least = 7.888609052210118e-31;        // (at least 2^-100: the fp32 scale stays normal)
  top = fmax(mt_max16(top), least);
  double inv = mt_scale8(top);
  uint32_t hi[8], low = ~0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    hi[e] = (uint32_t)(__builtin_bit_cast(uint64_t, fabs(h.x[e]) * inv) >> 32);
    low = min(low, hi[e]);
  }
  uint32_t q[2] = {0u, 0u};
  if (!__any(odd || low < MT_ONE8)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t c = (hi[e] + d2[e]) >> 17;
      if (!ROOT) c |= (uint32_t)(__builtin_bit_cast(uint64_t, h.x[e]) >> 56) & 0x80u;
      q[e >> 2] |= c << (8 * (e & 3));
    }
  } else {
    // small numbers: below 2^-6 the grid keeps its step of 2^-9, as a mantissa does when 2^-6 is added.  What is not finite
    // counts for no largest value and is held as NaN.
    if (odd) {
      top = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmax(top, fabs(h.x[e]) <= most ? fabs(h.x[e]) : 0.0);
      top = fmax(mt_max16(top), least);
      inv = mt_scale8(top);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double ax = fabs(h.x[e]), y = ax * inv;
      const bool small = y < 0.015625;
      const uint32_t z = (uint32_t)(__builtin_bit_cast(uint64_t, small ? y + 0.015625 : y) >> 32);
      uint32_t c = ((z + d2[e]) >> 17) - (small ? 8u : 0u);
      if (ROOT) c = max(c, ax > 1e-140 ? 1u : 0u);                     // (the root of MT_SOME stands for 0)
      if (!(ax <= most)) c = 0x7fu;
      c |= (uint32_t)(__builtin_bit_cast(uint64_t, h.x[e]) >> 56) & 0x80u;
      q[e >> 2] |= c << (8 * (e & 3));
    }
  }
  if (FULL) {
    *reinterpret_cast<u32x2*>((uint8_t*)base + i) = u32x2{q[0], q[1]};
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) ((uint8_t*)base)[i + e] = (uint8_t)(q[e >> 2] >> (8 * (e & 3)));
  }
  if ((threadIdx.x & 15) == 0 && left > 0) scales[i / MT_BLOCK8] = (float)(top * (1.0 / 448.0));
}

// lr / (1 - b1^t) and 1 / sqrt(1 - b2^t): of the host, or of the step count on the device by repeated squaring, as in
// dpc_adam_step's kernel, one thread's work.  8-bit states: with the block's loads on their way (404 M fp32 parameters and gradients,
// Philox bits: 1282 -> 1234 us; now 1220, and 1160 with the host's count); 32-bit states: before them (2111 us against 2149, and
// 2105 with the host's).
struct AdamwBias { float step_size, inv_bc2s; };
__device__ __forceinline__ AdamwBias adamw_bias(const AdamwArgs& a, float* bc) {
  if (!a.t_dev) return AdamwBias{a.step_size, a.inv_bc2s};
  if (threadIdx.x == 0) {
    double p1 = 1.0, p2 = 1.0, x1 = a.b1d, x2 = a.b2d;
    for (int e = a.t_dev[0] + a.t_host; e > 0; e >>= 1) {
      if (e & 1) { p1 *= x1; p2 *= x2; }
      x1 *= x1; x2 *= x2;
    }
    bc[0] = (float)((double)a.lr / (1.0 - p1));
    bc[1] = (float)(1.0 / sqrt(1.0 - p2));
  }
  __syncthreads();
  return AdamwBias{bc[0], bc[1]};
}

// One pass of a block: 8 elements of each thread from i.  FULL: all of them exist and every buffer is aligned.
template <bool S8, bool FULL>
__device__ __forceinline__ void adamw_pass(const AdamwArgs& a, const MtRec& r, int64_t i, int left, double gs, float decay, AdamwBias bias, float* bc) {
#pragma clang fp contract(off)
  const Raw8 graw = mt_load<FULL>(r.g, i, r.g_t, left), praw = mt_load<FULL>(r.p, i, r.p_t, left);
  f32x8 p;
  if (S8) {
    const u32x2 mc = mt_load8<FULL>(r.m, i, left), rc = mt_load8<FULL>(r.v, i, left);
    const double ms = FULL || left > 0 ? r.ms[i / MT_BLOCK8] : 0.f, vs = FULL || left > 0 ? r.vs[i / MT_BLOCK8] : 0.f;
    u32x4 dw;
    if (r.dith) {
      dw = mt_load<FULL>(r.dith, i, DPC_F16, left).a;
    } else {
      const DpcPhilox4 ph = dpc_philox(a.rng[0], a.rng[1], a.site, (uint64_t)(r.draw8 + (i >> 3)));
      dw = u32x4{ph.v[0], ph.v[1], ph.v[2], ph.v[3]};
    }
    bias = adamw_bias(a, bc);
    const f32x8 g = mt_float(graw, r.g_t), mf = mt_float8(mc), rf = mt_float8(rc);
    p = mt_float(praw, r.p_t);
    uint32_t d2[8];
    Hold8 m, rt;
    float odd = 0.f;
    const double am = a.b1d * ms, ag = a.c1d * gs, bv = a.b2d * (vs * vs), bg = a.c2d * gs * gs;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      d2[e] = ((e & 1 ? dw[e >> 1] >> 15 : dw[e >> 1] << 1) & 0x1fffeu) - MT_BIAS8;
      const double ge = (double)g[e];
      m.x[e] = fma((double)mf[e], am, ag * ge);
      rt.x[e] = mt_root(fma(bg * ge, ge, fma((double)(rf[e] * rf[e]), bv, MT_SOME)));           // (the square of a code is exact in fp32)
      const float m32 = (float)m.x[e], r32 = (float)rt.x[e];
      // (1-ulp reciprocal: the step is rounded to the parameter's last bit anyway; eps8 is a normal number)
      p[e] = adamw_param(p[e], bias.step_size * (m32 * __builtin_amdgcn_rcpf(fmaf(r32, bias.inv_bc2s, a.eps8))), decay);
      odd = fmaf(p[e], 0.f, odd);                                      // NaN once a moment, and so the parameter, is not finite
    }
    const bool bad = __any(odd != 0.f);
    mt_hold8<FULL, false>(r.m, r.ms, i, left, m, d2, bad);
    mt_hold8<FULL, true>(r.v, r.vs, i, left, rt, d2, bad);
  } else {
    const Raw8 mraw = mt_load<FULL>(r.m, i, DPC_F32, left), vraw = mt_load<FULL>(r.v, i, DPC_F32, left);
    const f32x8 g = mt_float(graw, r.g_t);
    f32x8 m = mt_float(mraw, DPC_F32), v = mt_float(vraw, DPC_F32);
    p = mt_float(praw, r.p_t);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float ge = g[e] * (float)gs;
      m[e] = a.b1 * m[e] + a.c1 * ge;
      v[e] = a.b2 * v[e] + a.c2 * ge * ge;
      p[e] = adamw_param(p[e], bias.step_size * (m[e] / (sqrtf(v[e]) * bias.inv_bc2s + a.eps)), decay);
    }
    mt_store<FULL>(r.m, i, DPC_F32, left, m);
    mt_store<FULL>(r.v, i, DPC_F32, left, v);
  }
  mt_store<FULL>(r.p, i, r.p_t, left, p);
  if (r.cp) mt_store<FULL>(r.cp, i, r.c_t, left, p);
}

template <bool S8>
__global__ __launch_bounds__(256) void adamw_kernel(AdamwArgs a) {
  __shared__ float bc[2];
  const float coef = a.coef ? a.coef[0] : 1.f;
  if (a.coef && coef == 0.f) return;            // the clip factor of a gradient that is not finite
  const MtChunk ch = a.pl.chunk[blockIdx.x];
  const MtRec r = a.pl.rec[ch.t];
  AdamwBias bias = {0.f, 0.f};
  if (!S8) bias = adamw_bias(a, bc);
  const double gs = (double)a.gscale * coef;
  const float decay = a.lr * r.wd;
  // (the block stays whole where the tensor ends inside it: so do the 16 lanes of a state block)
  const int64_t i = ch.start + 8 * threadIdx.x;
  if (r.vec && r.n - ch.start >= MT_SUB)
    adamw_pass<S8, true>(a, r, i, 8, gs, decay, bias, bc);
  else
    adamw_pass<S8, false>(a, r, i, (int)max((int64_t)0, min((int64_t)8, r.n - i)), gs, decay, bias, bc);
}

// ---- host ----------------------------------------------------------------------------------------------------------
static int mt_size(int type) { return type == DPC_F32 ? 4 : 2; }
static bool mt_type_ok(int type) { return type == DPC_F32 || type == DPC_BF16 || type == DPC_F16; }
static bool mt_al(const void* p, int bytes) { return ((uintptr_t)p % (uintptr_t)bytes) == 0; }
#define MT_PARTS 2048            // partial sums of the global norm: its blocks at most

static int mt_check(const dpc_multi_tensor* t, int count, dpc_multi_info* info) {
  DPC_CHECK_ARG(count >= 0 && (t || count == 0) && info, "multi_plan: null pointer or negative count");
  int64_t grad_bytes = 0;
  int kinds = 0;
  for (int k = 0; k < count; ++k) {
    const dpc_multi_tensor& x = t[k];
    DPC_CHECK_ARG(x.n >= 0 && x.n < (1ll << 46), "multi_plan: bad tensor size");
    DPC_CHECK_ARG(mt_type_ok(x.g_type) && mt_type_ok(x.p_type) && mt_type_ok(x.copy_type), "multi_plan: unknown element type");
    if (x.n == 0) continue;
    DPC_CHECK_ARG(x.g && mt_al(x.g, mt_size(x.g_type)), "multi_plan: null or misaligned gradient");
    if (x.p) {
      DPC_CHECK_ARG(x.m && x.v, "multi_plan: a parameter needs both moments");
      DPC_CHECK_ARG(mt_al(x.p, mt_size(x.p_type)) && (!x.copy || mt_al(x.copy, mt_size(x.copy_type))), "multi_plan: misaligned tensor");
      DPC_CHECK_ARG(!x.m_scale == !x.v_scale, "multi_plan: both 8-bit states need their scales");
      DPC_CHECK_ARG(x.m_scale ? (mt_al(x.m_scale, 4) && mt_al(x.v_scale, 4)) : (mt_al(x.m, 4) && mt_al(x.v, 4)), "multi_plan: misaligned state");
      DPC_CHECK_ARG(!x.dither || (x.m_scale && mt_al(x.dither, 2)), "multi_plan: random bits go with 8-bit states");
      DPC_CHECK_ARG(x.wd >= 0.f && x.wd <= 3.402823466e38f, "multi_plan: weight decay must be finite and not negative");
      kinds |= x.m_scale ? (x.dither ? 4 : 2) : 1;
    } else {
      DPC_CHECK_ARG(!x.m && !x.v && !x.copy && !x.m_scale && !x.v_scale, "multi_plan: states without a parameter");
      kinds |= 8;
    }
    grad_bytes += x.n * mt_size(x.g_type);
  }
  DPC_CHECK_ARG(kinds == 0 || kinds == 1 || kinds == 2 || kinds == 4 || kinds == 8,
                "multi_plan: the tensors of a plan are of one kind (gradients only, 32-bit states, or 8-bit states with or without given random bits)");
  // (a chunk is one pass of a block: with two, four and eight the step of 404 M parameters took 2142, 2165 and 2214 us
  // against 2114)
  int64_t blocks = 0;
  for (int k = 0; k < count; ++k) blocks += dpc_cdiv(t[k].n, MT_SUB);
  DPC_CHECK_ARG(blocks < (1ll << 24), "multi_plan: too many elements");      // (a launch has less than 2^32 threads)
  info->kind = kinds;
  info->grad_bytes = grad_bytes;
  info->count = count;
  info->blocks = (int)blocks;
  info->rec_off = 0;
  info->chunk_off = mt_align((int64_t)count * sizeof(MtRec));
  info->part_off = info->chunk_off + mt_align(blocks * (int64_t)sizeof(MtChunk)) + MT_COUNTS;      // (before it the counts of blocks that have ended)
  info->bytes = info->part_off + MT_PARTS * sizeof(double);
  return DPC_OK;
}

extern "C" int dpc_multi_plan_size(const dpc_multi_tensor* t, int count, dpc_multi_info* info) { return mt_check(t, count, info); }

extern "C" int dpc_multi_plan(const dpc_multi_tensor* t, int count, const dpc_multi_info* info, void* plan, int64_t bytes) {
  DPC_CHECK_ARG(info && plan, "multi_plan: null pointer");
  dpc_multi_info in;
  const int rc = mt_check(t, count, &in);
  if (rc != DPC_OK) return rc;
  DPC_CHECK_ARG(in.bytes == info->bytes && in.blocks == info->blocks && in.kind == info->kind && bytes >= in.bytes,
                "multi_plan: the buffer or the sizes are not those of dpc_multi_plan_size");
  memset(plan, 0, (size_t)in.bytes);
  MtRec* rec = (MtRec*)((char*)plan + in.rec_off);
  MtChunk* chunk = (MtChunk*)((char*)plan + in.chunk_off);
  int64_t draw = 0, b = 0;
  for (int k = 0; k < count; ++k) {
    const dpc_multi_tensor& x = t[k];
    MtRec& r = rec[k];
    r.p = x.p; r.g = x.g; r.m = x.m; r.v = x.v; r.ms = x.m_scale; r.vs = x.v_scale; r.cp = x.copy; r.dith = x.dither;
    r.n = x.n; r.draw8 = draw; r.p_t = x.p_type; r.g_t = x.g_type; r.c_t = x.copy_type; r.wd = x.wd;
    r.vec = mt_al(x.g, 16) && (!x.p || (mt_al(x.p, 16) && mt_al(x.m, x.m_scale ? 8 : 16) && mt_al(x.v, x.m_scale ? 8 : 16) &&
                                        mt_al(x.copy, 16) && mt_al(x.dither, 16)));
    draw += dpc_cdiv(x.n, 8);
    for (int64_t s = 0; s < x.n; s += MT_SUB) { chunk[b].t = k; chunk[b].start = s; ++b; }
  }
  return DPC_OK;
}

static MtPlan mt_view(const dpc_multi_info* info, const void* plan) {
  MtPlan pl;
  pl.rec = (const MtRec*)((const char*)plan + info->rec_off);
  pl.chunk = (const MtChunk*)((const char*)plan + info->chunk_off);
  pl.blocks = info->blocks;
  return pl;
}

extern "C" int dpc_grad_clip(const dpc_multi_info* info, void* plan, double max_norm, double gscale, float* out, int32_t* t_dev, void* stream) {
  DPC_CHECK_ARG(info && plan && out, "grad_clip: null pointer");
  DPC_CHECK_ARG(max_norm > 0.0 && gscale > 0.0 && gscale <= 3.402823466e38, "grad_clip: max_norm and gscale must be positive");
  double* part = (double*)((char*)plan + info->part_off);
  const ClipArgs a = {max_norm, gscale, out, t_dev};
  const int64_t quads = dpc_cdiv(info->blocks, 4);
  const int nb = (int)(quads < MT_PARTS ? quads : MT_PARTS);
  const auto clip = info->grad_bytes > (256ll << 20) ? grad_clip_kernel<true> : grad_clip_kernel<false>;
  if (nb > 0) hipLaunchKernelGGL(clip, dim3(nb), dim3(256), 0, (hipStream_t)stream, mt_view(info, plan), part, (uint32_t*)((char*)part - MT_COUNTS), a);
  else hipLaunchKernelGGL(grad_clip_none_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, a);
  DPC_LAUNCH_CHECK();
  return DPC_OK;
}

extern "C" int dpc_adamw_step(const dpc_multi_info* info, const void* plan, double lr, double b1, double b2, double eps,
                              const float* coef, float gscale, const int32_t* t_dev, int t_host, const uint64_t* rng,
                              uint32_t site, void* stream) {
  DPC_CHECK_ARG(info && plan, "adamw: null pointer");
  DPC_CHECK_ARG(info->kind != 8, "adamw: the plan lists gradients only");
  DPC_CHECK_ARG(b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0 && eps >= 0.0 && lr >= 0.0 && lr <= 3.402823466e38, "adamw: betas must lie in [0, 1), lr and eps must not be negative");
  DPC_CHECK_ARG(t_host >= 1 || (t_host == 0 && t_dev), "adamw: the step count starts at 1 (t_host 0 goes with a device counter)");
  DPC_CHECK_ARG(info->kind != 2 || rng, "adamw: 8-bit states need random bits (rng, or dither in the plan)");
  if (info->blocks == 0) return DPC_OK;
  AdamwArgs a;
  a.pl = mt_view(info, plan);
  a.lr = (float)lr; a.b1 = (float)b1; a.b2 = (float)b2; a.c1 = (float)(1.0 - b1); a.c2 = (float)(1.0 - b2); a.eps = (float)eps;
  a.eps8 = a.eps < 1.17549435e-38f ? 1.17549435e-38f : a.eps;
  a.b1d = b1; a.b2d = b2; a.c1d = 1.0 - b1; a.c2d = 1.0 - b2;
  a.step_size = a.inv_bc2s = 0.f;
  if (!t_dev) {
    a.step_size = (float)(lr / (1.0 - pow(b1, t_host)));
    a.inv_bc2s = (float)(1.0 / sqrt(1.0 - pow(b2, t_host)));
  }
  a.coef = coef; a.gscale = gscale; a.t_dev = t_dev; a.t_host = t_host; a.rng = rng; a.site = site;
  if (info->kind == 1) hipLaunchKernelGGL(adamw_kernel<false>, dim3(info->blocks), dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(adamw_kernel<true>, dim3(info->blocks), dim3(256), 0, (hipStream_t)stream, a);
  DPC_LAUNCH_CHECK();
  return DPC_OK;
}
