// Token slots sorted by expert, and token rows moved to that order and back: the local work of a rank that holds some of
// a model's experts, between an all-gather of tokens and a reduce-scatter of their outputs.
#include <hip/hip_runtime.h>
#include "local_ops.h"

static __device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

// ------------------------------------------------------------------ sort
// A stable counting sort.  A tile of RA_SORT_THREADS * ROUNDS slots belongs to one workgroup, a run of 64 * ROUNDS of them
// to a wave, 64 at a time: lanes with the same key find one another by a ballot for each bit of the key, a slot's rank is
// the wave's running count of the key plus the peers in lower lanes.  Counts of the waves, then of the tiles before this
// one, then of the experts before this one are added: nothing depends on the order in which anything runs.
static __device__ __forceinline__ int keyOf(const RaSortArgs& a, uint32_t slot) {
  const int64_t e = (a.idBytes == 8 ? ((const int64_t*)a.ids)[slot] : (int64_t)((const int32_t*)a.ids)[slot]);
  const uint64_t k = (uint64_t)e - (uint64_t)a.firstExpert;
  return k < (uint64_t)a.nExperts ? (int)k : a.nExperts;
}

// Slots of each expert in each tile; only for more than one tile.
__global__ __launch_bounds__(RA_SORT_THREADS) void raLocalKernelSortCount(RaSortArgs a, uint32_t tileSlots) {
  extern __shared__ int hist[];
  for (int e = threadIdx.x; e < a.nExperts; e += RA_SORT_THREADS) hist[e] = 0;
  __syncthreads();
  const uint32_t lo = blockIdx.x * tileSlots;                       // (tiles * tileSlots stays below 2^32)
  const uint32_t hi = a.slots - lo < tileSlots ? a.slots : lo + tileSlots;
  for (uint32_t i = lo + threadIdx.x; i < hi; i += RA_SORT_THREADS) {
    const int k = keyOf(a, i);
    if (k < a.nExperts) atomicAdd(&hist[k], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.nExperts; e += RA_SORT_THREADS) a.tileCounts[(size_t)blockIdx.x * a.nExperts + e] = hist[e];
}

template <int ROUNDS>
__global__ __launch_bounds__(RA_SORT_THREADS) void raLocalKernelSort(RaSortArgs a) {
  constexpr int WAVES = RA_SORT_THREADS / 64;
  extern __shared__ int lds[];
  const int n = a.nExperts;
  int* base = lds;                                                  // [n] first row of this tile's slots of an expert
  int* total = lds + n;                                             // [n] slots of an expert in all tiles
  int* sums = lds + 2 * n;                                          // [WAVES + 1]
  volatile uint16_t* wc = (volatile uint16_t*)(lds + 2 * n + WAVES + 1);   // [WAVES][n] counts of each wave, at most 64 * ROUNDS
  const int lane = threadIdx.x & 63, wave = (int)uniform(threadIdx.x >> 6);
  for (int i = threadIdx.x; i < WAVES * n; i += RA_SORT_THREADS) wc[i] = 0;
  for (int e = threadIdx.x; e < n; e += RA_SORT_THREADS) { base[e] = 0; total[e] = 0; }
  __syncthreads();

  const uint32_t first = (blockIdx.x * WAVES + wave) * (64u * ROUNDS);
  const int bits = 32 - __builtin_clz((unsigned)n);                 // keys are 0 .. n
  int key[ROUNDS], rank[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; r++) {
    const uint32_t slot = first + r * 64 + lane;
    key[r] = slot < a.slots ? keyOf(a, slot) : n;
  }
#pragma unroll
  for (int r = 0; r < ROUNDS; r++) {
    uint64_t peers = ~0ull;
    for (int b = 0; b < bits; b++) {
      const bool one = (key[r] >> b) & 1;
      const uint64_t ones = __ballot(one);
      peers &= one ? ones : ~ones;
    }
    const int below = __builtin_amdgcn_mbcnt_hi((uint32_t)(peers >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)peers, 0));
    int before = 0;
    if (key[r] < n) {
      before = wc[wave * n + key[r]];                               // LDS operations of one wave are done in order
      if (below == 0) wc[wave * n + key[r]] = (uint16_t)(before + __popcll(peers));
    }
    rank[r] = before + below;
  }
  if (a.tiles > 1)
    for (uint32_t i = threadIdx.x; i < a.tiles * (uint32_t)n; i += RA_SORT_THREADS) {
      const int c = a.tileCounts[i];
      if (c) {
        atomicAdd(&total[i % n], c);
        if (i / n < blockIdx.x) atomicAdd(&base[i % n], c);
      }
    }
  __syncthreads();
  // Thread e: the expert's counts of the waves before each wave; its slots in all tiles.
  int padded = 0;
  const int e = threadIdx.x;
  if (e < n) {
    int run = 0;
    for (int w = 0; w < WAVES; w++) { const int c = wc[w * n + e]; wc[w * n + e] = (uint16_t)run; run += c; }
    if (a.tiles == 1) total[e] = run;
    padded = (total[e] + a.rowAlign - 1) / a.rowAlign * a.rowAlign;
  }
  int scan = padded;                                                // inclusive over the wave, then over the waves
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(scan, d); if (lane >= d) scan += o; }
  if (lane == 63) sums[wave] = scan;
  __syncthreads();
  if (threadIdx.x == 0) { int run = 0; for (int w = 0; w < WAVES; w++) { const int c = sums[w]; sums[w] = run; run += c; } sums[WAVES] = run; }
  __syncthreads();
  const int start = sums[wave] + scan - padded;                     // first row of expert e
  if (e < n) {
    base[e] += start;
    if (blockIdx.x == 0) {
      if (a.offsets) { a.offsets[e] = start; if (e == n - 1) a.offsets[n] = start + padded; }
      if (a.counts) a.counts[e] = total[e];
    }
    // Rows without a slot: the padding of each expert by one workgroup, what is behind the last expert by all of them.
    if (a.source && e % a.tiles == blockIdx.x)
      for (int row = start + total[e]; row < start + padded; row++) a.source[row] = -1;
  }
  if (a.source)
    for (uint32_t row = (uint32_t)sums[WAVES] + blockIdx.x * RA_SORT_THREADS + threadIdx.x; row < a.rows; row += a.tiles * RA_SORT_THREADS)
      a.source[row] = -1;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; r++) {
    const uint32_t slot = first + r * 64 + lane;
    if (slot >= a.slots) continue;
    int row = -1;
    if (key[r] < n) {
      row = base[key[r]] + wc[wave * n + key[r]] + rank[r];
      if (a.source) a.source[row] = (int32_t)slot;
    }
    a.position[slot] = row;
  }
}

hipError_t raLaunchSort(const RaSortArgs& a, hipStream_t s) {
  const uint32_t rounds = raSortRounds(a.slots);
  const int waves = RA_SORT_THREADS / 64;
  if (a.tiles > 1) hipLaunchKernelGGL(raLocalKernelSortCount, dim3(a.tiles), dim3(RA_SORT_THREADS), a.nExperts * sizeof(int), s, a, RA_SORT_THREADS * rounds);
  const size_t lds = (2 * (size_t)a.nExperts + waves + 1) * sizeof(int) + (size_t)waves * a.nExperts * sizeof(uint16_t);
  switch (rounds) {
    case 1: hipLaunchKernelGGL((raLocalKernelSort<1>), dim3(a.tiles), dim3(RA_SORT_THREADS), lds, s, a); break;
    case 4: hipLaunchKernelGGL((raLocalKernelSort<4>), dim3(a.tiles), dim3(RA_SORT_THREADS), lds, s, a); break;
    default: hipLaunchKernelGGL((raLocalKernelSort<8>), dim3(a.tiles), dim3(RA_SORT_THREADS), lds, s, a); break;
  }
  return hipGetLastError();
}

// ------------------------------------------------------------------ rows
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// 16 bytes with the alignment of one element: strides and row lengths may be odd, and unaligned vector accesses are legal.
typedef u32x4 u32x4_u2 __attribute__((aligned(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Pack {};                               // 16 bytes of a row, and the same as floats
template <> struct Pack<float> { static constexpr int N = 4; typedef f32x4 floats; };
template <> struct Pack<__bf16> { static constexpr int N = 8; typedef f32x8 floats; };
template <> struct Pack<_Float16> { static constexpr int N = 8; typedef f32x8 floats; };
template <typename T> static __device__ __forceinline__ typename Pack<T>::floats toFloats(u32x4 p) {
  typedef T vec __attribute__((ext_vector_type(Pack<T>::N)));
  return __builtin_convertvector(__builtin_bit_cast(vec, p), typename Pack<T>::floats);
}
template <typename T> static __device__ __forceinline__ u32x4 fromFloats(typename Pack<T>::floats f) {
  typedef T vec __attribute__((ext_vector_type(Pack<T>::N)));
  return __builtin_bit_cast(u32x4, __builtin_convertvector(f, vec));
}
// The pack at element `at` of a row of `hidden` elements; past its end there are zeros, and nothing is written.
template <typename T> static __device__ __forceinline__ u32x4 loadPack(const T* row, size_t at, size_t hidden) {
  constexpr int N = Pack<T>::N;
  if (at + N <= hidden) return *(const u32x4_u2*)(row + at);
  typedef T vec __attribute__((ext_vector_type(N)));
  vec v = {};
#pragma unroll
  for (int i = 0; i < N; i++) if (at + i < hidden) v[i] = row[at + i];
  return __builtin_bit_cast(u32x4, v);
}
template <typename T> static __device__ __forceinline__ void storePack(T* row, size_t at, size_t hidden, u32x4 p) {
  constexpr int N = Pack<T>::N;
  if (at + N <= hidden) { *(u32x4_u2*)(row + at) = p; return; }
  typedef T vec __attribute__((ext_vector_type(N)));
  const vec v = __builtin_bit_cast(vec, p);
#pragma unroll
  for (int i = 0; i < N; i++) if (at + i < hidden) row[at + i] = v[i];
}
static __device__ __forceinline__ float weightOf(const void* w, int type, size_t i) {
  if (type == ncclFloat32) return ((const float*)w)[i];
  if (type == ncclBfloat16) return (float)((const __bf16*)w)[i];
  return (float)((const _Float16*)w)[i];
}
// Lane k of the wave holds what belongs to slot k of its token.
static __device__ __forceinline__ int laneInt(int x, int k) { return __builtin_amdgcn_readlane(x, k); }
static __device__ __forceinline__ float laneFloat(float x, int k) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), k)); }

// The padding rows of the segments are set to zero by the workgroups behind those of the tokens, RA_PAD_GROUPS for each expert.
#define RA_PAD_GROUPS 4
template <typename T> static __device__ __forceinline__ void padRows(const RaRowsArgs& a, uint32_t group) {
  const int e = (int)(group / RA_PAD_GROUPS);
  const int waves = (int)(blockDim.x >> 6);
  int64_t row = (int64_t)a.offsets[e] + a.counts[e] + (int)(group % RA_PAD_GROUPS) * waves + (int)uniform(threadIdx.x >> 6);
  const int64_t end = a.offsets[e + 1] < (int64_t)a.rows ? a.offsets[e + 1] : (int64_t)a.rows;
  if (row < 0) return;
  for (; row < end; row += RA_PAD_GROUPS * waves)
    for (size_t at = (threadIdx.x & 63) * Pack<T>::N; at < a.hidden; at += 64 * Pack<T>::N)
      storePack((T*)a.out + (size_t)row * a.outStride, at, a.hidden, u32x4{0, 0, 0, 0});
}

// Dispatch.  A wave takes 64 * U packs of one token's row, reads them once and writes them to each of the token's slots.
#define RA_ROWS_THREADS 256
template <typename T, int U>
__global__ __launch_bounds__(RA_ROWS_THREADS) void raLocalKernelDispatch(RaRowsArgs a, uint32_t groups, uint32_t parts) {
  if (blockIdx.x >= groups) { padRows<T>(a, blockIdx.x - groups); return; }
  const int lane = threadIdx.x & 63;
  const uint64_t unit = (uint64_t)blockIdx.x * (RA_ROWS_THREADS / 64) + uniform(threadIdx.x >> 6);
  const size_t token = unit / parts;
  if (token >= a.tokens) return;
  const int32_t pos = lane < a.topk ? a.position[token * a.topk + lane] : -1;
  uint64_t slots = __ballot(pos >= 0 && (size_t)pos < a.rows);
  if (!slots) return;
  const T* x = (const T*)a.in + token * a.inStride;
  const size_t at = ((size_t)(unit % parts) * 64 * U + lane) * Pack<T>::N;
  u32x4 p[U];
#pragma unroll
  for (int u = 0; u < U; u++) p[u] = loadPack(x, at + u * 64 * Pack<T>::N, a.hidden);
  for (; slots; slots &= slots - 1) {
    T* row = (T*)a.out + (size_t)laneInt(pos, __builtin_ctzll(slots)) * a.outStride;
#pragma unroll
    for (int u = 0; u < U; u++) storePack(row, at + u * 64 * Pack<T>::N, a.hidden, p[u]);
  }
}

// Combine.  A wave takes 64 * U packs of one token's row and adds those of its slots in the order of k, four rows in flight.
template <typename T, int U>
__global__ __launch_bounds__(RA_ROWS_THREADS) void raLocalKernelCombine(RaRowsArgs a, uint32_t parts) {
  constexpr int N = Pack<T>::N, F = 4;
  typedef typename Pack<T>::floats floats;
  const int lane = threadIdx.x & 63;
  const uint64_t unit = (uint64_t)blockIdx.x * (RA_ROWS_THREADS / 64) + uniform(threadIdx.x >> 6);
  const size_t token = unit / parts;
  if (token >= a.tokens) return;
  int32_t pos = -1;
  float w = 1.f;
  if (lane < a.topk) {
    pos = a.position[token * a.topk + lane];
    if (a.weightType >= 0) w = weightOf(a.weights, a.weightType, token * a.topk + lane);
  }
  uint64_t slots = __ballot(pos >= 0 && (size_t)pos < a.rows);
  const size_t at = ((size_t)(unit % parts) * 64 * U + lane) * N;
  floats sum[U];
#pragma unroll
  for (int u = 0; u < U; u++) sum[u] = floats{};
  while (slots) {
    u32x4 p[F][U];
    float wk[F];
    int have = 0;
#pragma unroll
    for (int f = 0; f < F; f++) {
      if (!slots) break;
      const int k = __builtin_ctzll(slots);
      slots &= slots - 1;
      have = f + 1;
      wk[f] = laneFloat(w, k);
      const T* z = (const T*)a.in + (size_t)laneInt(pos, k) * a.inStride;
#pragma unroll
      for (int u = 0; u < U; u++) p[f][u] = loadPack(z, at + u * 64 * N, a.hidden);
    }
#pragma unroll
    for (int f = 0; f < F; f++) {
      if (f >= have) break;
#pragma unroll
      for (int u = 0; u < U; u++) {
        const floats z = toFloats<T>(p[f][u]);
#pragma unroll
        for (int i = 0; i < N; i++) sum[u][i] = __builtin_fmaf(wk[f], z[i], sum[u][i]);
      }
    }
  }
  T* y = (T*)a.out + token * a.outStride;
#pragma unroll
  for (int u = 0; u < U; u++) storePack(y, at + u * 64 * N, a.hidden, fromFloats<T>(sum[u]));
}

// The gradients of combine.  A workgroup takes one token: its row of dy stays in registers (a part of the row at a time,
// where it is longer than the workgroup holds) while the rows of its slots pass; each wave adds its part of a slot's
// product into its own word in LDS.
template <typename T>
__global__ __launch_bounds__(1024) void raLocalKernelCombineBackward(RaRowsArgs a, uint32_t groups) {
  constexpr int N = Pack<T>::N, U = 2;
  typedef typename Pack<T>::floats floats;
  __shared__ float dots[16][RA_ROWS_MAX_TOPK];
  if (blockIdx.x >= groups) { padRows<T>(a, blockIdx.x - groups); return; }
  const int lane = threadIdx.x & 63, wave = (int)uniform(threadIdx.x >> 6), waves = (int)(blockDim.x >> 6);
  const size_t token = blockIdx.x;
  int32_t pos = -1;
  float w = 0.f;
  if (lane < a.topk) {
    pos = a.position[token * a.topk + lane];
    w = weightOf(a.weights, a.weightType, token * a.topk + lane);
    dots[wave][lane] = 0.f;
  }
  const uint64_t all = __ballot(pos >= 0 && (size_t)pos < a.rows);
  const T* dy = (const T*)a.in + token * a.inStride;
  if (all)
    for (size_t part = 0; part < a.hidden; part += (size_t)waves * 64 * U * N) {
      const size_t at = part + ((size_t)wave * 64 * U + lane) * N;
      floats d[U];
#pragma unroll
      for (int u = 0; u < U; u++) d[u] = toFloats<T>(loadPack(dy, at + u * 64 * N, a.hidden));
      for (uint64_t slots = all; slots; slots &= slots - 1) {
        const int k = __builtin_ctzll(slots);
        const size_t row = (size_t)laneInt(pos, k);
        const float wk = laneFloat(w, k);
        const T* z = (const T*)a.z + row * a.zStride;
        T* dz = (T*)a.out + row * a.outStride;
        float dot = 0.f;
#pragma unroll
        for (int u = 0; u < U; u++) {
          const floats zf = toFloats<T>(loadPack(z, at + u * 64 * N, a.hidden));
          floats g;
#pragma unroll
          for (int i = 0; i < N; i++) { dot = __builtin_fmaf(d[u][i], zf[i], dot); g[i] = wk * d[u][i]; }
          storePack(dz, at + u * 64 * N, a.hidden, fromFloats<T>(g));
        }
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) dot += __shfl_xor(dot, s);
        if (lane == 0) dots[wave][k] += dot;
      }
    }
  __syncthreads();
  if (wave == 0 && lane < a.topk) {
    float sum = 0.f;
    for (int v = 0; v < waves; v++) sum += dots[v][lane];
    const size_t slot = token * a.topk + lane;
    if (a.weightType == ncclFloat32) ((float*)a.dweights)[slot] = sum;
    else if (a.weightType == ncclBfloat16) ((__bf16*)a.dweights)[slot] = (__bf16)sum;
    else ((_Float16*)a.dweights)[slot] = (_Float16)sum;
  }
}

static uint32_t padGroups(const RaRowsArgs& a) { return a.offsets ? (uint32_t)a.nExperts * RA_PAD_GROUPS : 0; }

template <typename T> static hipError_t dispatch(const RaRowsArgs& a, hipStream_t s) {
  constexpr int U = 2;
  const uint64_t parts = (a.hidden + 64 * U * Pack<T>::N - 1) / (64 * U * Pack<T>::N);
  const uint64_t groups = (a.tokens * parts + RA_ROWS_THREADS / 64 - 1) / (RA_ROWS_THREADS / 64);
  if (groups + padGroups(a) > 0x7FFFFFFF) return hipErrorInvalidValue;
  if (groups + padGroups(a) == 0) return hipSuccess;
  hipLaunchKernelGGL((raLocalKernelDispatch<T, U>), dim3((uint32_t)groups + padGroups(a)), dim3(RA_ROWS_THREADS), 0, s, a, (uint32_t)groups, (uint32_t)parts);
  return hipGetLastError();
}
template <typename T> static hipError_t combine(const RaRowsArgs& a, hipStream_t s) {
  constexpr int U = 2;
  const uint64_t parts = (a.hidden + 64 * U * Pack<T>::N - 1) / (64 * U * Pack<T>::N);
  const uint64_t groups = (a.tokens * parts + RA_ROWS_THREADS / 64 - 1) / (RA_ROWS_THREADS / 64);
  if (groups > 0x7FFFFFFF) return hipErrorInvalidValue;
  hipLaunchKernelGGL((raLocalKernelCombine<T, U>), dim3((uint32_t)groups), dim3(RA_ROWS_THREADS), 0, s, a, (uint32_t)parts);
  return hipGetLastError();
}
template <typename T> static hipError_t combineBackward(const RaRowsArgs& a, hipStream_t s) {
  const size_t packs = (a.hidden + Pack<T>::N - 1) / Pack<T>::N;
  const size_t waves = packs <= 128 ? 1 : packs >= 16 * 128 ? 16 : (packs + 127) / 128;
  if (a.tokens + padGroups(a) > 0x7FFFFFFF) return hipErrorInvalidValue;
  hipLaunchKernelGGL((raLocalKernelCombineBackward<T>), dim3((uint32_t)a.tokens + padGroups(a)), dim3((uint32_t)waves * 64), 0, s, a, (uint32_t)a.tokens);
  return hipGetLastError();
}
#define RA_BY_TYPE(fn)                                    \
  switch (type) {                                         \
    case ncclFloat32: return fn<float>(a, s);             \
    case ncclBfloat16: return fn<__bf16>(a, s);           \
    case ncclFloat16: return fn<_Float16>(a, s);          \
    default: return hipErrorInvalidValue;                 \
  }
hipError_t raLaunchDispatch(const RaRowsArgs& a, int type, hipStream_t s) { RA_BY_TYPE(dispatch) }
hipError_t raLaunchCombine(const RaRowsArgs& a, int type, hipStream_t s) { RA_BY_TYPE(combine) }
hipError_t raLaunchCombineBackward(const RaRowsArgs& a, int type, hipStream_t s) { RA_BY_TYPE(combineBackward) }
