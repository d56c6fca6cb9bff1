// AdamW over many tensors and the sum of squares that clips it: the local work of a rank between a reduce-scatter of
// gradients and an all-gather of parameters.  Element-wise, bound by HBM: every element is read once and written once.
#include <hip/hip_runtime.h>
#include "local_ops.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
// The same with the alignment of one element: tensors are views at any element of a flat buffer.  Unaligned vector
// accesses are legal on gfx950, so one code path serves all of them.
typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef f16x4 f16x4_u __attribute__((aligned(2)));
typedef bf16x4 bf16x4_u __attribute__((aligned(2)));
typedef uint32_t u32_u __attribute__((aligned(1)));

template <typename T> struct Vec;
template <> struct Vec<float> { typedef f32x4_u four; };
template <> struct Vec<_Float16> { typedef f16x4_u four; };
template <> struct Vec<__bf16> { typedef bf16x4_u four; };

template <typename T> static __device__ __forceinline__ f32x4 load4(const T* p) {
  return __builtin_convertvector(__builtin_nontemporal_load((const typename Vec<T>::four*)p), f32x4);
}
template <typename T> static __device__ __forceinline__ void store4(T* p, f32x4 x) {
  typedef T vec __attribute__((ext_vector_type(4)));
  __builtin_nontemporal_store(__builtin_convertvector(x, vec), (typename Vec<T>::four*)p);
}
// The same where only `left` (1 .. 3) of the four elements exist; the others are zeros.
template <typename T> static __device__ __forceinline__ f32x4 load4(const T* p, int left) {
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  x[0] = (float)p[0];
  if (left > 1) x[1] = (float)p[1];
  if (left > 2) x[2] = (float)p[2];
  return x;
}
template <typename T> static __device__ __forceinline__ void store4(T* p, f32x4 x, int left) {
  p[0] = (T)x[0];
  if (left > 1) p[1] = (T)x[1];
  if (left > 2) p[2] = (T)x[2];
}

// 32 bits that depend on all of x: two rounds of xor-shift and multiplication by an odd constant (2^32 over the golden
// ratio, and a multiplier of L'Ecuyer's tables of linear congruential generators).
static __device__ __forceinline__ uint32_t mix(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x9E3779B1u;
  x = (x ^ (x >> 15)) * 0xAC564B05u;
  return x ^ (x >> 16);
}
static __device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
static __device__ __forceinline__ float uniform(float x) { return __uint_as_float(uniform(__float_as_uint(x))); }

// Which of the launch's tensors chunk b belongs to: the number of tensors that begin at or before it, less one.  All loads
// are on their way before the first is waited for.
template <int MAX> static __device__ __forceinline__ uint32_t findTensor(const uint32_t* first, uint32_t n, uint32_t b) {
  if (n == 1) return 0;
  uint32_t f[(MAX + 63) / 64], t = 0;
  const uint32_t lane = threadIdx.x & 63;
#pragma unroll
  for (int k = 0; k < (MAX + 63) / 64; k++) f[k] = k * 64 + lane < n ? first[k * 64 + lane] : ~0u;
#pragma unroll
  for (int k = 0; k < (MAX + 63) / 64; k++) t += (uint32_t)__popcll(__ballot(f[k] <= b));
  return uniform(t - 1);
}

// x^n by squaring, in 64 bits; the host computes its bias corrections with the same steps.
static __device__ __forceinline__ double powN(double x, int64_t n) {
  double r = 1.0;
  for (; n > 0; n >>= 1, x *= x) if (n & 1) r *= x;
  return r;
}

struct Scalars { float b1, omb1, b2, omb2, eps, decay, stepSize, rootC2, coef; };

// ------------------------------------------------------------------ 8-bit states
// 2^(X-127), for the scaled conversions: they take the exponent field of their scale alone, and for them 0 is 2^-127 and 255 NaN.
static __device__ __forceinline__ float powerOf(uint32_t scale) { return __uint_as_float(scale << 23); }
static __device__ __forceinline__ f32x4 decode4(uint32_t code, uint32_t scale) {
  const f32x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(code, powerOf(scale), false), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(code, powerOf(scale), true);
  return f32x4{lo[0], lo[1], hi[0], hi[1]};
}
static __device__ __forceinline__ uint32_t maxOf8(uint32_t a) {      // over the 8 lanes that hold a block, with DPP moves
  uint32_t o;
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0xB1, 0xF, 0xF, true); a = a > o ? a : o;      // lane ^ 1
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x4E, 0xF, 0xF, true); a = a > o ? a : o;      // lane ^ 2
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x141, 0xF, 0xF, true); return a > o ? a : o;  // 7 - lane
}
// The scale of a block: the smallest power of two with which its largest magnitude (bit pattern `most`) is at most 448.
static __device__ __forceinline__ uint32_t scaleOf(uint32_t most) {
  const int x = (int)((most + 0x1FFFFFu) >> 23) - 8;
  return (uint32_t)(x < 1 ? 1 : x > 247 ? 247 : x);
}
// Stochastic rounding to the e4m3 grid, by the instruction for it: of x / scale, the 20 high bits of `rnd` are added below the
// third bit of the mantissa (below 2^-9 in the subnormal range) and what is below it is cut off.  Values that are not
// finite become NaN.  Written out in integer operations this took a third of the kernel's VALU time.
static __device__ __forceinline__ uint32_t encode4(f32x4 x, uint32_t scale, const uint32_t (&rnd)[4]) {
  const float f = powerOf(scale);
  uint32_t c = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(0, x[0], rnd[0], f, 0);
  c = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(c, x[1], rnd[1], f, 1);
  c = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(c, x[2], rnd[2], f, 2);
  return __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(c, x[3], rnd[3], f, 3);
}
// Largest magnitude of a block, as a bit pattern.  What is not finite does not count: it becomes NaN, and the others of its
// block keep their scale.  That costs a second pass, which only waves that hold such an element take.
static __device__ __forceinline__ uint32_t largestOf8(f32x4 x) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) { const uint32_t b = __float_as_uint(x[i]) & 0x7FFFFFFFu; a = a > b ? a : b; }
  a = maxOf8(a);
  if (__any(a >= 0x7F800000u)) {
    a = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) { const uint32_t b = __float_as_uint(x[i]) & 0x7FFFFFFFu; a = b > a && b < 0x7F800000u ? b : a; }
    a = maxOf8(a);
  }
  return a;
}

// ------------------------------------------------------------------ AdamW
// A workgroup of four waves takes one chunk of one tensor; a wave takes rows of 256 elements, 4 for each lane, so that
// every access of a row is one contiguous run and a block of an 8-bit state lies in 8 neighbouring lanes.
template <typename P, typename G, bool MX> struct Row {
  P* param; const G* grad;
  float *m, *v;                         // fp32 states
  uint8_t *cm, *cv, *sm, *sv;           // 8-bit states
  void* copy; int copyType;
  f32x4 p, g, fm, fv;
  uint32_t qm, qv, xm, xv;

  // A lane's elements of a row are at .. at + 3; `left` of them exist (4 in every lane where WHOLE).
  template <bool WHOLE> __device__ __forceinline__ void load(size_t at, int left) {
    if (WHOLE || left >= 4) {
      p = load4(param + at); g = load4(grad + at);
      if constexpr (MX) { qm = __builtin_nontemporal_load((const u32_u*)(cm + at)); qv = __builtin_nontemporal_load((const u32_u*)(cv + at)); }
      else { fm = load4(m + at); fv = load4(v + at); }
    } else {
      p = g = fm = fv = f32x4{0.f, 0.f, 0.f, 0.f};
      qm = qv = 0;
      if (left > 0) {
        p = load4(param + at, left); g = load4(grad + at, left);
        if constexpr (MX) {
          qm = cm[at]; qv = cv[at];
          if (left > 1) { qm |= (uint32_t)cm[at + 1] << 8; qv |= (uint32_t)cv[at + 1] << 8; }
          if (left > 2) { qm |= (uint32_t)cm[at + 2] << 16; qv |= (uint32_t)cv[at + 2] << 16; }
        } else { fm = load4(m + at, left); fv = load4(v + at, left); }
      }
    }
    if constexpr (MX) {
      xm = xv = 0;
      if (WHOLE || left > 0) { xm = sm[at / RCCL_AMD_STATE_BLOCK]; xv = sv[at / RCCL_AMD_STATE_BLOCK]; }
    }
  }
  template <typename C> __device__ __forceinline__ void storeAs(C* to, bool whole, int left) {
    if (whole) store4(to, p);
    else if (left > 0) store4(to, p, left);
  }
  __device__ __forceinline__ void storeCopy(size_t at, bool whole, int left) {
    if (copyType < 0) return;
    if (copyType == ncclFloat32) storeAs((float*)copy + at, whole, left);
    else if (copyType == ncclBfloat16) storeAs((__bf16*)copy + at, whole, left);
    else storeAs((_Float16*)copy + at, whole, left);
  }
  // Square roots are the correctly rounded ones and nothing is contracted, so that a rounding of an 8-bit state does not depend
  // on how this is compiled.  So is the quotient with fp32 states; with 8-bit states, where VALU time counts, it is a product
  // with the reciprocal instruction's result, which is off by at most one unit of the last place.  That instruction takes
  // subnormal numbers for zero and gives none.  The divisor is zero or from 2^-126 to 2^126: with eps = 0 a root of an fp32
  // number, 2^-75 at least; otherwise eps, which the host holds to that range, or more by a root of at most 2^64 and its
  // correction of at most 2^27, which next to 2^126 is rounded away.  (Where g^2 is infinite, so is the divisor, and its reciprocal 0.)
  template <bool WHOLE> __device__ __forceinline__ void update(const Scalars& s, size_t at, int left, uint32_t key) {
    f32x4 r;
    if constexpr (MX) { fm = decode4(qm, xm); r = decode4(qv, xv); fv = r * r; }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float gi = g[i] * s.coef;
      fm[i] = s.b1 * fm[i] + s.omb1 * gi;
      fv[i] = s.b2 * fv[i] + s.omb2 * (gi * gi);
      r[i] = __builtin_sqrtf(fv[i]);
      const float down = r[i] * s.rootC2 + s.eps;
      p[i] = p[i] * s.decay - s.stepSize * (MX ? fm[i] * __builtin_amdgcn_rcpf(down) : fm[i] / down);
    }
    const bool whole = WHOLE || left >= 4;
    storeAs(param + at, whole, left);
    storeCopy(at, whole, left);
    if constexpr (MX) {
      // (what does not exist is zero: its gradient and its moments were)
      const uint32_t em = scaleOf(largestOf8(fm)), ev = scaleOf(largestOf8(r));
      const float least = powerOf(ev) * 0x1p-9f;            // a second moment over zero stays over zero
      uint32_t rm[4], rv[4];                                // 16 random bits, and a half of the last of them
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t h = mix((uint32_t)at + (uint32_t)i + key);
        rm[i] = h << 16 | 0x8000u;
        rv[i] = (h & 0xFFFF0000u) | 0x8000u;
        if (r[i] > 0.f) r[i] = r[i] > least ? r[i] : least;
      }
      const uint32_t nm = encode4(fm, em, rm), nv = encode4(r, ev, rv);
      if (whole) { __builtin_nontemporal_store(nm, (u32_u*)(cm + at)); __builtin_nontemporal_store(nv, (u32_u*)(cv + at)); }
      else if (left > 0) {
        cm[at] = (uint8_t)nm; cv[at] = (uint8_t)nv;
        if (left > 1) { cm[at + 1] = (uint8_t)(nm >> 8); cv[at + 1] = (uint8_t)(nv >> 8); }
        if (left > 2) { cm[at + 2] = (uint8_t)(nm >> 16); cv[at + 2] = (uint8_t)(nv >> 16); }
      }
      if ((threadIdx.x & 7) == 0 && (WHOLE || left > 0)) { sm[at / RCCL_AMD_STATE_BLOCK] = (uint8_t)em; sv[at / RCCL_AMD_STATE_BLOCK] = (uint8_t)ev; }
    } else if (whole) { store4(m + at, fm); store4(v + at, fv); }
    else if (left > 0) { store4(m + at, fm, left); store4(v + at, fv, left); }
  }
};

template <typename P, typename G, bool MX>
__global__ __launch_bounds__(RA_ADAMW_THREADS) __attribute__((amdgpu_waves_per_eu(1, MX && sizeof(P) == 2 ? 8 : 4))) void raLocalKernelAdamW(RaAdamWArgs a) {
  // Rows in flight for each wave, and no more than 16 waves on a compute unit, so that the workgroups that run at a time
  // stream through one window of memory.  fp32 states: one row for each wave in all, a shard of 67 million elements (1.88 GB) 0.302 ms
  // = 6.2 TB/s; with 2, 4 and 16 rows for each wave 0.313, 0.320 and 0.350, with 32 waves 0.311, with accesses that are not streaming
  // 0.369.  8-bit states: two rows at once and in all (the start of a workgroup counts for more), 33.5 million elements of fp32
  // (541 MB) 0.089 ms = 6.1 TB/s, of four rows 0.094.  With parameters in 16 bits arithmetic is what bounds
  // it: 66 VALU instructions for each element keep the SIMDs' issue busy for nine tenths of the kernel's cycles (68 and seven tenths with
  // fp32 parameters).  32 waves, two rows 0.080 ms (fp16, fp32 gradients, bf16 copy, 477 MB; four rows 0.085), and four rows where nothing but
  // 16-bit parameters and gradients is moved beside the states 0.064 (340 MB; two rows 0.067).
  constexpr int U = MX ? 2 : 1;
  constexpr uint32_t STEP = RA_ADAMW_THREADS / 64 * RA_ADAMW_ROW;
  uint32_t t, chunk0;
  size_t count, offset = 0;
  const uint64_t* w;
  if (a.stride) {
    t = findTensor<RA_ADAMW_MAX>(a.general.first, a.n, blockIdx.x);
    chunk0 = a.general.first[t];
    w = a.general.words + (size_t)t * a.stride;
    count = w[RA_W_COUNT];
  } else {
    t = findTensor<RA_ADAMW_FLAT>(a.flat.first, a.n, blockIdx.x);
    chunk0 = a.flat.first[t];
    w = a.flat.base;
    count = a.flat.count[t];
    offset = a.flat.offset[t];
  }
  const size_t begin = (size_t)(blockIdx.x - chunk0) * a.chunk;
  const size_t end = begin + a.chunk < count ? begin + a.chunk : count;

  Scalars s = {a.b1, a.omb1, a.b2, a.omb2, a.eps, a.decay, a.stepSize, a.rootC2, a.coef};
  int64_t step = a.step;
  if (a.stepPtr || a.lrPtr) {
    if (a.stepPtr) step = *a.stepPtr > 1 ? *a.stepPtr : 1;
    const double lr = a.lrPtr ? (double)*a.lrPtr : a.lr;
    s.decay = uniform((float)(1.0 - lr * a.weightDecay));
    s.stepSize = uniform((float)(lr / (1.0 - powN(a.beta1, step))));
    s.rootC2 = uniform((float)(1.0 / __builtin_sqrt(1.0 - powN(a.beta2, step))));
  }
  bool go = true;
  if (a.sumSq) {
    const double sq = *a.sumSq;
    go = __builtin_isfinite(sq);
    const double c = a.maxNorm / (a.gradScale * __builtin_sqrt(sq) + 1e-6);
    s.coef = uniform((float)(a.gradScale * (c < 1.0 ? c : 1.0)));
  }

  Row<P, G, MX> row[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    row[u].param = (P*)w[RA_W_PARAM] + offset; row[u].grad = (const G*)w[RA_W_GRAD] + offset;
    if constexpr (MX) {
      row[u].cm = (uint8_t*)w[RA_W_M] + offset; row[u].cv = (uint8_t*)w[RA_W_V] + offset;
      row[u].sm = (uint8_t*)w[RA_W_MS] + offset / RCCL_AMD_STATE_BLOCK; row[u].sv = (uint8_t*)w[RA_W_VS] + offset / RCCL_AMD_STATE_BLOCK;
    } else { row[u].m = (float*)w[RA_W_M] + offset; row[u].v = (float*)w[RA_W_V] + offset; }
    row[u].copy = a.copyWord >= 0 ? (void*)w[a.copyWord] : nullptr;
    row[u].copyType = row[u].copy ? a.copyType : -1;
    if (row[u].copy) row[u].copy = (char*)row[u].copy + offset * (a.copyType == ncclFloat32 ? 4 : 2);
  }
  const uint32_t lane4 = (threadIdx.x & 63) * 4;
  size_t r = begin + uniform(threadIdx.x >> 6) * RA_ADAMW_ROW;
  uint32_t key = 0;
  if constexpr (MX) {
    key = mix((uint32_t)a.seed + 0x9E3779B9u);
    key = mix(key ^ (uint32_t)(a.seed >> 32));
    key = mix(key + (uint32_t)step);
    key = uniform(mix(a.ordinal + t + key));
  }
  // (the high word of an element's index belongs to its random bits too)
  if (U > 1 && go)
    for (; r + (U - 1) * STEP + RA_ADAMW_ROW <= end; r += U * STEP) {
#pragma unroll
      for (int u = 0; u < U; u++) row[u].template load<true>(r + u * STEP + lane4, 4);
#pragma unroll
      for (int u = 0; u < U; u++) {
        const size_t at = r + u * STEP;
        row[u].template update<true>(s, at + lane4, 4, at >> 32 ? mix(key ^ (uint32_t)(at >> 32)) : key);
      }
    }
  for (; r < end; r += STEP) {
    const size_t at = r + lane4;
    const int left = at < end ? (end - at < 4 ? (int)(end - at) : 4) : 0;
    if (go) {
      row[0].template load<false>(at, left);
      row[0].template update<false>(s, at, left, r >> 32 ? mix(key ^ (uint32_t)(r >> 32)) : key);
    } else if (row[0].copyType >= 0) {                      // a skipped step: only the copies are written
      if (left >= 4) row[0].p = load4(row[0].param + at);
      else if (left > 0) row[0].p = load4(row[0].param + at, left);
      row[0].storeCopy(at, left >= 4, left);
    }
  }
}

template <typename P, typename G>
static hipError_t adamW(const RaAdamWArgs& a, bool mx, uint32_t grid, hipStream_t s) {
  return mx ? raLaunch(raLocalKernelAdamW<P, G, true>, grid, RA_ADAMW_THREADS, 0, s, a) : raLaunch(raLocalKernelAdamW<P, G, false>, grid, RA_ADAMW_THREADS, 0, s, a);
}
template <typename P>
static hipError_t adamWGrad(const RaAdamWArgs& a, int gradType, bool mx, uint32_t grid, hipStream_t s) {
  switch (gradType) {
    case ncclFloat32: return adamW<P, float>(a, mx, grid, s);
    case ncclBfloat16: return adamW<P, __bf16>(a, mx, grid, s);
    case ncclFloat16: return adamW<P, _Float16>(a, mx, grid, s);
    default: return hipErrorInvalidValue;
  }
}
hipError_t raLaunchAdamW(const RaAdamWArgs& a, int paramType, int gradType, bool mx, uint32_t grid, hipStream_t s) {
  switch (paramType) {
    case ncclFloat32: return adamWGrad<float>(a, gradType, mx, grid, s);
    case ncclBfloat16: return adamWGrad<__bf16>(a, gradType, mx, grid, s);
    case ncclFloat16: return adamWGrad<_Float16>(a, gradType, mx, grid, s);
    default: return hipErrorInvalidValue;
  }
}

// ------------------------------------------------------------------ sum of squares
// One partial sum for each chunk, in 64 bits, then one workgroup that adds the partial sums in a fixed order: the result
// does not depend on which chunk is done first.  Squares of fp32 values overflow fp32 long before their norm does, so
// the products are 64-bit too.
static __device__ __forceinline__ double waveSum(double x) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
  return x;
}
template <int THREADS> static __device__ __forceinline__ double blockSum(double x) {      // valid in thread 0
  __shared__ double sums[THREADS / 64];
  x = waveSum(x);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = x;
  __syncthreads();
  x = 0.0;
  if (threadIdx.x == 0) for (int i = 0; i < THREADS / 64; i++) x += sums[i];
  return x;
}
template <typename T> static __device__ __forceinline__ f32x4 load4Cached(const T* p) {   // AdamW reads the gradients next
  return __builtin_convertvector(*(const typename Vec<T>::four*)p, f32x4);
}
template <typename T>
__global__ __launch_bounds__(RA_SUMSQ_THREADS) void raLocalKernelSumSq(RaSumSqArgs a) {
  const uint32_t t = findTensor<RA_SUMSQ_MAX>(a.first, a.n, blockIdx.x);
  const T* x = (const T*)a.ptr[t];
  const uint32_t count = a.count[t];
  const uint64_t begin = (uint64_t)(blockIdx.x - a.first[t]) * a.chunk;
  const uint64_t end = begin + a.chunk < count ? begin + a.chunk : count;
  constexpr int U = 4;
  constexpr uint32_t STEP = RA_SUMSQ_THREADS * 4;
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  uint64_t r = begin + threadIdx.x * 4;
  for (; r + (U - 1) * STEP + 4 <= end; r += U * STEP) {
    f32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; u++) v[u] = load4Cached(x + r + u * STEP);
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int i = 0; i < 4; i++) sum[i] = __builtin_fma((double)v[u][i], (double)v[u][i], sum[i]);
  }
  for (; r < end; r += STEP) {
    const f32x4 v = end - r < 4 ? load4(x + r, (int)(end - r)) : load4Cached(x + r);
#pragma unroll
    for (int i = 0; i < 4; i++) sum[i] = __builtin_fma((double)v[i], (double)v[i], sum[i]);
  }
  const double all = blockSum<RA_SUMSQ_THREADS>((sum[0] + sum[1]) + (sum[2] + sum[3]));
  if (threadIdx.x == 0) {
    if (a.out) *a.out = (a.accumulate ? *a.out : 0.0) + all;
    else a.partial[blockIdx.x] = all;
  }
}
__global__ __launch_bounds__(1024) void raLocalKernelSumSqJoin(const double* __restrict__ partial, uint32_t n, double* out, int accumulate) {
  double sum = 0.0;
  for (uint32_t i = threadIdx.x; i < n; i += 1024) sum += partial[i];
  sum = blockSum<1024>(sum);
  if (threadIdx.x == 0) *out = (accumulate ? *out : 0.0) + sum;
}

hipError_t raLaunchSumSq(const RaSumSqArgs& a, int type, uint32_t grid, hipStream_t s) {
  switch (type) {
    case ncclFloat32: return raLaunch(raLocalKernelSumSq<float>, grid, RA_SUMSQ_THREADS, 0, s, a);
    case ncclBfloat16: return raLaunch(raLocalKernelSumSq<__bf16>, grid, RA_SUMSQ_THREADS, 0, s, a);
    case ncclFloat16: return raLaunch(raLocalKernelSumSq<_Float16>, grid, RA_SUMSQ_THREADS, 0, s, a);
    default: return hipErrorInvalidValue;
  }
}
hipError_t raLaunchSumSqJoin(const double* partial, uint32_t n, double* out, int accumulate, hipStream_t s) {
  return raLaunch(raLocalKernelSumSqJoin, 1, 1024, 0, s, partial, n, out, accumulate);
}
