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

// Workgroups of consecutive numbers run on the eight XCDs in turn.  Each XCD takes consecutive tiles, whose runs of rows meet
// in its L2 (524288 slots of 384 experts 14.1 us, tile by tile 14.9).
static __device__ __forceinline__ uint32_t tileOf(uint32_t b, uint32_t tiles) {
  const uint32_t q = tiles / 8, r = tiles % 8, x = b % 8;
  return x * q + (x < r ? x : r) + b / 8;
}

// Slots of each expert in each tile; only for more than one tile.
__global__ __launch_bounds__(RA_SORT_THREADS) void raLocalKernelSortCount(RaSortArgs a, uint32_t tileSlots) {
  extern __shared__ int hist[];
  for (int e = threadIdx.x; e < a.nExperts; e += RA_SORT_THREADS) hist[e] = 0;
  __syncthreads();
  const uint32_t tile = tileOf(blockIdx.x, a.tiles), lo = tile * tileSlots;      // (tiles * tileSlots stays below 2^32)
  const uint32_t hi = a.slots - lo < tileSlots ? a.slots : lo + tileSlots;
#pragma unroll 4
  for (uint32_t i = lo + threadIdx.x; i < hi; i += RA_SORT_THREADS) {
    const int k = keyOf(a, i);
    if (k < a.nExperts) atomicAdd(&hist[k], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.nExperts; e += RA_SORT_THREADS) a.tileCounts[(size_t)tile * a.nExperts + e] = hist[e];
}

// Where there are many counts: each becomes the sum of those of the tiles before it, and the row behind the last tile the sum
// of all.  A workgroup takes 16 experts, which lie side by side in memory, a group of 16 threads a run of tiles (1024 tiles of
// 128 experts 5.5 us; a wave for each expert, its lanes' loads a run of tiles apart, 17 with half as many).
__global__ __launch_bounds__(RA_SORT_THREADS) void raLocalKernelSortScan(RaSortArgs a) {
  __shared__ int part[RA_SORT_THREADS / 16][16];                    // a run's columns are turned by its number / 4: every bank once
  const uint32_t x = threadIdx.x & 15, group = threadIdx.x >> 4, e = blockIdx.x * 16 + x, n = (uint32_t)a.nExperts;
  const uint32_t run = (a.tiles + 63) / 64, lo = group * run, hi = e >= n ? 0 : lo + run < a.tiles ? lo + run : a.tiles;
  int sum = 0;
#pragma unroll 8
  for (uint32_t t = lo; t < hi; t++) sum += a.tileCounts[(size_t)t * n + e];
  part[group][(x + (group >> 2)) & 15] = sum;
  __syncthreads();
  const uint32_t wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;        // a wave scans one expert's 64 runs
  int* mine = &part[lane][(wave + (lane >> 2)) & 15];
  const int own = *mine;
  int scan = own;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(scan, d); if (lane >= (uint32_t)d) scan += o; }
  if (lane == 63 && blockIdx.x * 16 + wave < n) a.tileCounts[(size_t)a.tiles * n + blockIdx.x * 16 + wave] = scan;
  *mine = scan - own;
  __syncthreads();
  sum = part[group][(x + (group >> 2)) & 15];
#pragma unroll 8
  for (uint32_t t = lo; t < hi; t++) { const int c = a.tileCounts[(size_t)t * n + e]; a.tileCounts[(size_t)t * n + e] = sum; sum += c; }
}

// LDS of the sort: three words for each expert, one for each wave, and for each expert a count of each wave.
static size_t sortLds(int n) { return (3 * (size_t)n + RA_SORT_THREADS / 64 + 1) * sizeof(int) + (size_t)(RA_SORT_THREADS / 64) * ((n + 1) / 2) * 2 * sizeof(uint16_t); }

template <int ROUNDS>
__global__ __launch_bounds__(RA_SORT_THREADS) void raLocalKernelSort(RaSortArgs a) {
  constexpr int WAVES = RA_SORT_THREADS / 64;
  extern __shared__ int lds[];
  const int n = a.nExperts, pitch = (n + 1) / 2 * 2;
  int* base = lds;                                                  // [n] slots of an expert in earlier tiles, then its first row here
  int* total = lds + n;                                             // [n] slots of an expert in all tiles
  int* start = lds + 2 * n;                                         // [n] first row of an expert
  int* sums = lds + 3 * n;                                          // [WAVES + 1]
  uint16_t* wc = (uint16_t*)(lds + 3 * n + WAVES + 1);              // [WAVES][pitch] counts of each wave, at most 64 * ROUNDS
  const int lane = threadIdx.x & 63, wave = (int)uniform(threadIdx.x >> 6);
  const uint32_t tile = tileOf(blockIdx.x, a.tiles), first = (tile * WAVES + wave) * (64u * ROUNDS);
  int key[ROUNDS], rank[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; r++) {
    const uint32_t slot = first + r * 64 + lane;
    key[r] = slot < a.slots ? keyOf(a, slot) : n;
  }
  for (int i = lane; i < pitch / 2; i += 64) ((int*)(wc + wave * pitch))[i] = 0;     // a wave clears its own
  for (int e = threadIdx.x; e < n; e += RA_SORT_THREADS) {
    base[e] = a.scanned ? a.tileCounts[(size_t)tile * n + e] : 0;
    total[e] = a.scanned ? a.tileCounts[(size_t)a.tiles * n + e] : 0;
  }
  __syncthreads();
  // The slots of each expert in all tiles, and in those before this one: groups of threads that hold one expert each take
  // the tiles in turn.
  if (a.tiles > 1 && !a.scanned) {
    const int width = (int)raSortWidth(n);
    const int e = threadIdx.x & (width - 1);
    const uint32_t step = RA_SORT_THREADS / width;
    if (e < n) {
      int all = 0, before = 0;
#pragma unroll 8
      for (uint32_t t = threadIdx.x / width; t < a.tiles; t += step) {
        const int c = a.tileCounts[(size_t)t * n + e];
        all += c;
        before += t < tile ? c : 0;
      }
      if (all) atomicAdd(&total[e], all);
      if (before) atomicAdd(&base[e], before);
    }
  }
  const int bits = 32 - __builtin_clz((unsigned)n);                 // keys are 0 .. n
  volatile uint16_t* mine = wc + wave * pitch;                      // LDS operations of one wave are done in order
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
      before = mine[key[r]];
      if (below == 0) mine[key[r]] = (uint16_t)(before + __popcll(peers));
    }
    rank[r] = before + below;
  }
  __syncthreads();
  // Thread e: the expert's counts of the waves before each wave, its rows.
  int padded = 0;
  const int e = threadIdx.x;
  if (e < n) {
    int c[WAVES], run = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) c[w] = wc[w * pitch + e];
#pragma unroll
    for (int w = 0; w < WAVES; w++) { wc[w * pitch + e] = (uint16_t)run; run += c[w]; }
    if (a.tiles == 1) total[e] = run;
    padded = (total[e] + a.rowAlign - 1) / a.rowAlign * a.rowAlign;
  }
  int scan = padded;                                                // inclusive over the wave, then over the waves
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(scan, d); if (lane >= d) scan += o; }
  if (lane == 63) sums[wave] = scan;
  __syncthreads();
  int earlier = 0, used = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) { const int c = sums[w]; earlier += w < wave ? c : 0; used += c; }
  if (e < n) {
    const int from = earlier + scan - padded;
    base[e] += from;
    start[e] = from;
    if (blockIdx.x == 0) {
      if (a.offsets) { a.offsets[e] = from; if (e == n - 1) a.offsets[n] = from + padded; }
      if (a.counts) a.counts[e] = total[e];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; r++) {
    const uint32_t slot = first + r * 64 + lane;
    if (slot >= a.slots) continue;
    int row = -1;
    if (key[r] < n) {
      row = base[key[r]] + wc[wave * pitch + key[r]] + rank[r];
      if (a.source) a.source[row] = (int32_t)slot;
    }
    a.position[slot] = row;
  }
  if (!a.source) return;
  // Rows without a slot: the padding of an expert by a wave of one workgroup, what is behind the last expert by all of them.
  for (uint32_t x = blockIdx.x + wave * a.tiles; x < (uint32_t)n; x += WAVES * a.tiles) {
    const int from = start[x] + total[x], to = x + 1 < (uint32_t)n ? start[x + 1] : used;
    for (int row = from + lane; row < to; row += 64) a.source[row] = -1;
  }
  for (uint32_t row = (uint32_t)used + blockIdx.x * RA_SORT_THREADS + threadIdx.x; row < a.rows; row += a.tiles * RA_SORT_THREADS) a.source[row] = -1;
}

hipError_t raLaunchSort(const RaSortArgs& a, hipStream_t s) {
  const uint32_t rounds = raSortRounds(a.slots);
  hipError_t e = hipSuccess;
  if (a.tiles > 1) e = raLaunch(raLocalKernelSortCount, a.tiles, RA_SORT_THREADS, a.nExperts * sizeof(int), s, a, RA_SORT_THREADS * rounds);
  if (a.scanned && e == hipSuccess) e = raLaunch(raLocalKernelSortScan, (a.nExperts + 15) / 16, RA_SORT_THREADS, 0, s, a);
  if (e != hipSuccess) return e;
  switch (rounds) {
    case 1: return raLaunch(raLocalKernelSort<1>, a.tiles, RA_SORT_THREADS, sortLds(a.nExperts), s, a);
    case 2: return raLaunch(raLocalKernelSort<2>, a.tiles, RA_SORT_THREADS, sortLds(a.nExperts), s, a);
    default: return raLaunch(raLocalKernelSort<4>, a.tiles, RA_SORT_THREADS, sortLds(a.nExperts), s, a);
  }
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
// A pack of a row.  STREAM: the access does not ask for a place in the caches.
template <bool STREAM, typename T> static __device__ __forceinline__ u32x4 wholePack(const T* p) {
  return STREAM ? __builtin_nontemporal_load((const u32x4_u2*)p) : *(const u32x4_u2*)p;
}
template <bool STREAM, typename T> static __device__ __forceinline__ void storeWhole(T* p, u32x4 x) {
  if (STREAM) __builtin_nontemporal_store(x, (u32x4_u2*)p);
  else *(u32x4_u2*)p = x;
}
// The pack at element `at` of a row of `hidden` elements, where the row may end inside it: there are zeros past its end, and
// nothing is written there.
template <bool STREAM, typename T> static __device__ __forceinline__ u32x4 loadPack(const T* row, size_t at, size_t hidden) {
  constexpr int N = Pack<T>::N;
  if (at + N <= hidden) return wholePack<STREAM>(row + at);
  typedef T vec __attribute__((ext_vector_type(N)));
  vec v = {};
#pragma unroll
  for (int i = 0; i < N - 1; i++) if (at + i < hidden) v[i] = row[at + i];
  return __builtin_bit_cast(u32x4, v);
}
template <bool STREAM, typename T> static __device__ __forceinline__ void storePack(T* row, size_t at, size_t hidden, u32x4 p) {
  constexpr int N = Pack<T>::N;
  if (at + N <= hidden) { storeWhole<STREAM>(row + at, p); return; }
  typedef T vec __attribute__((ext_vector_type(N)));
  const vec v = __builtin_bit_cast(vec, p);
#pragma unroll
  for (int i = 0; i < N - 1; i++) if (at + i < hidden) row[at + i] = v[i];
}
static __device__ __forceinline__ float weightOf(const void* w, int type, size_t i) {
  if (type == ncclFloat32) return ((const float*)w)[i];
  if (type == ncclBfloat16) return (float)((const __bf16*)w)[i];
  return (float)((const _Float16*)w)[i];
}
static __device__ __forceinline__ void storeWeight(void* w, int type, size_t i, float x) {
  if (type == ncclFloat32) ((float*)w)[i] = x;
  else if (type == ncclBfloat16) ((__bf16*)w)[i] = (__bf16)x;
  else ((_Float16*)w)[i] = (_Float16)x;
}
// Lane k of the wave holds what belongs to slot k of its token.
static __device__ __forceinline__ int laneInt(int x, int k) { return __builtin_amdgcn_readlane(x, k); }
static __device__ __forceinline__ float laneFloat(float x, int k) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), k)); }

// The padding rows of the segments are set to zero by the workgroups behind those of the slots, RA_PAD_GROUPS for each expert.
#define RA_PAD_GROUPS 4
template <typename T> static __device__ __forceinline__ void padRows(const RaRowsArgs& a, uint32_t group) {
  const int e = (int)(group / RA_PAD_GROUPS);
  const int waves = (int)(blockDim.x >> 6);
  int64_t row = (int64_t)a.offsets[e] + a.counts[e] + (int)(group % RA_PAD_GROUPS) * waves + (int)uniform(threadIdx.x >> 6);
  const int64_t end = a.offsets[e + 1] < (int64_t)a.rows ? a.offsets[e + 1] : (int64_t)a.rows;
  if (row < 0) return;
  for (; row < end; row += RA_PAD_GROUPS * waves)
    for (size_t at = (threadIdx.x & 63) * Pack<T>::N; at < a.hidden; at += 64 * Pack<T>::N)
      storePack<false>((T*)a.out + (size_t)row * a.outStride, at, a.hidden, u32x4{0, 0, 0, 0});
}

// How a row is cut: `head` single elements up to the first 16-byte boundary of the row that is written, then `body`
// elements in packs, then single ones again.  Stores of 16 bytes that are not aligned cost up to half of the bandwidth,
// loads that are not cost little.  The at most 14 single elements are one access of a wave: see elementOf.
struct RowCut { uint32_t head, body, single; };         // single = hidden - body
template <typename T> static __device__ __forceinline__ RowCut cutRow(const T* out, size_t hidden) {
  constexpr uint32_t N = Pack<T>::N;
  uint32_t head = (uint32_t)((16 - ((uintptr_t)out & 15)) & 15) / (uint32_t)sizeof(T);
  if (head > hidden) head = (uint32_t)hidden;
  const uint32_t body = ((uint32_t)hidden - head) / N * N;
  return RowCut{head, body, (uint32_t)hidden - body};
}
// Which element is a lane's single one, of `singles` in the row.
static __device__ __forceinline__ uint32_t elementOf(uint32_t head, size_t hidden, uint32_t singles, uint32_t lane) { return lane < head ? lane : (uint32_t)hidden - singles + lane; }

// Dispatch and the gradient of combine: a workgroup of eight waves takes `each` slots in a row, every lane of a wave loads the
// position of one, and the waves take the slots that are kept in turn, S rows at a time.
#define RA_SLOT_WAVES 8
// What a launch over slots needs before all else, in few 32-bit steps, so that a workgroup without work ends soon.
struct RaSlots {
  const int32_t* end;                // how many rows are kept at most (offsets[nExperts]), or null
  uint32_t slots, rows, groups;      // groups: workgroups of the slots; those behind them clear padding rows
  uint32_t inverse, shift;           // slot / topk = slot * inverse >> shift, for slots below 2^31
  uint32_t few[3];                   // `each` doubles where fewer rows than this are kept, and again, and again
};
// `each`: 8 S slots where all are kept, so that every wave has a row (S of them), writes it and ends: a wave that goes on to a second row
// waits for the stores of the first, and with 64 slots in any case 16384 tokens of 8 slots, rows of 8 KiB, take 245 us, with 8 216.
// More where a rank holds few of the experts and most slots are dropped, so that a wave does not live for one position alone:
// 65536 tokens of 8 slots, one in eight kept, rows of 8, 4 and 2 KiB 154, 57 and 27 us, a wave for each slot 217, 118
// and 82 (the gradients 177, 113 and 50 against 312, 291 and 130; one set of inputs again and again, part of which stays in the
// Infinity Cache).  What is kept stands on the device, so the grid fits `rows`
// and workgroups too many end at once: that is 40 us of the 154.  half: more slots for a workgroup already where half are dropped
// (dispatch of 16384 tokens of 8 KiB rows 111 us, not so 132; the gradients 184 and 180).
static RaSlots slotsOf(const RaRowsArgs& a, int S, bool half) {
  uint32_t l = 0;
  while ((1 << l) < a.topk) l++;     // 2^(31 + l) / topk, rounded up, is below 2^32; over 2^31 slots its error stays below 1 / topk
  const uint64_t slots = a.tokens * a.topk;
  RaSlots n = {a.offsets ? a.offsets + a.nExperts : nullptr, (uint32_t)slots, (uint32_t)a.rows, 0, (uint32_t)(((1ull << (31 + l)) + a.topk - 1) / a.topk), 31 + l, {0, 0, 0}};
  for (int i = 0; i < 3 && (RA_SLOT_WAVES * S << i) < 64; i++) n.few[i] = (uint32_t)(half && i == 0 ? slots * 3 / 5 : slots / (3 << i)) + 1;
  return n;
}
static __host__ __device__ __forceinline__ uint32_t doublings(const RaSlots& n, uint32_t kept) { return (kept < n.few[0]) + (kept < n.few[1]) + (kept < n.few[2]); }
template <int S> static __device__ __forceinline__ uint32_t slotsEach(const RaSlots& n) {
  uint32_t kept = n.rows;
  if (n.end) { const uint32_t end = (uint32_t)*n.end; kept = end < kept ? end : kept; }
  return RA_SLOT_WAVES * S << doublings(n, kept);
}
// The lanes of the kept slots that are this wave's.
template <int S> static __device__ __forceinline__ uint64_t sharedOut(bool keep, uint32_t wave) {
  const uint64_t kept = __ballot(keep);
  const uint32_t rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(kept >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)kept, 0));
  return __ballot(keep && rank / S % RA_SLOT_WAVES == wave);
}

// Dispatch.  V = 8 / S packs in flight for each lane and row: one row with rows over 256 packs (parts of a row, where there are too
// few slots to fill the GPU), more with shorter ones.  Long runs of one row are what the
// time follows: 16384 tokens of 8 slots, 4096 bf16 elements (1.24 GB to move): 8 KiB in one go 0.218 ms, 4 KiB 0.225, 2 KiB
// 0.235; a wave that reads a row once and writes all of the token's rows 0.236, the same through LDS 0.236; streaming accesses
// 0.225 to 0.250.  The waves that write a token's rows are in one workgroup, so that its row comes from HBM once.
// Sixteen waves of a compute unit at a time: with 20, 24 and 32 the runs of more rows mix, and the time is 0.226, 0.239 and 0.244 ms.
#define RA_FEW_WAVES(most) __attribute__((amdgpu_waves_per_eu(4, most)))
template <typename T, int S>
__global__ __launch_bounds__(RA_SLOT_WAVES * 64) RA_FEW_WAVES(S == 1 ? 4 : 8) void raLocalKernelDispatch(RaSlots n, RaRowsArgs a, uint32_t parts, uint32_t partElems) {
  constexpr uint32_t N = Pack<T>::N, U = 8, V = S == 1 ? 4 : U / S;      // V: packs of a slot in what is left of its row
  if (blockIdx.x >= n.groups) { padRows<T>(a, blockIdx.x - n.groups); return; }
  const uint32_t wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const bool split = S == 1 && parts > 1;                              // a wave takes a part of one slot's row
  const uint32_t each = split ? 1 : slotsEach<S>(n);
  const uint32_t units = split ? n.slots * parts : (n.slots + each - 1) / each;
  for (uint32_t unit = split ? blockIdx.x * RA_SLOT_WAVES + wave : blockIdx.x; unit < units; unit += split ? n.groups * RA_SLOT_WAVES : n.groups) {
    const uint32_t slot = (split ? unit / parts : unit * each) + lane;      // (below 2^31 + 64)
    int32_t pos = -1;
    if (lane < each && slot < n.slots) pos = a.position[slot];
    const uint32_t token = (uint32_t)((uint64_t)slot * n.inverse >> n.shift);
    const bool keep = pos >= 0 && (uint32_t)pos < n.rows;
    for (uint64_t kept = split ? __ballot(keep) : sharedOut<S>(keep, wave); kept;) {
      const T* x[S];
      T* out[S];
      RowCut c[S];
      bool go[S];
#pragma unroll
      for (int s = 0; s < S; s++) {
        go[s] = kept != 0;
        const int k = go[s] ? __builtin_ctzll(kept) : 0;
        kept &= kept - 1;
        x[s] = (const T*)a.in + (size_t)(uint32_t)laneInt(token, k) * a.inStride;
        out[s] = (T*)a.out + (size_t)(go[s] ? laneInt(pos, k) : 0) * a.outStride;
        c[s] = cutRow(out[s], a.hidden);
      }
      uint32_t run = 0;
      if (split) {
        const uint32_t part = unit % parts;
        run = part * partElems;
        if (part) c[0].single = 0;                           // (the single elements go with the first part)
        if (run + partElems < c[0].body) c[0].body = run + partElems;
      }
      for (; S == 1 && run + U * 64 * N <= c[0].body; run += U * 64 * N) {
        u32x4 p[U];
        const T* from = x[0] + c[0].head + run + lane * N;
        T* to = out[0] + c[0].head + run + lane * N;
#pragma unroll
        for (uint32_t u = 0; u < U; u++) p[u] = wholePack<false>(from + u * 64 * N);
#pragma unroll
        for (uint32_t u = 0; u < U; u++) storeWhole<false>(to + u * 64 * N, p[u]);
      }
      T single[S];
      if (S == 1 && lane < c[0].single) single[0] = x[0][elementOf(c[0].head, a.hidden, c[0].single, lane)];
      do {
        u32x4 p[S][V];
#pragma unroll
        for (int s = 0; s < S; s++) {
          const T* from = x[s] + c[s].head + run + lane * N;
#pragma unroll
          for (uint32_t v = 0; v < V; v++) if (go[s] && run + (v * 64 + lane) * N < c[s].body) p[s][v] = wholePack<false>(from + v * 64 * N);
          if (S > 1 && go[s] && lane < c[s].single) single[s] = x[s][elementOf(c[s].head, a.hidden, c[s].single, lane)];
        }
#pragma unroll
        for (int s = 0; s < S; s++) {
          T* to = out[s] + c[s].head + run + lane * N;
#pragma unroll
          for (uint32_t v = 0; v < V; v++) if (go[s] && run + (v * 64 + lane) * N < c[s].body) storeWhole<false>(to + v * 64 * N, p[s][v]);
          if (S > 1 && go[s] && lane < c[s].single) out[s][elementOf(c[s].head, a.hidden, c[s].single, lane)] = single[s];
        }
        run += V * 64 * N;
      } while (S == 1 && run < c[0].body);
      if (S == 1 && lane < c[0].single) out[0][elementOf(c[0].head, a.hidden, c[0].single, lane)] = single[0];
    }
  }
}

// Rows of at most 32 packs: a group of `1 << shift` lanes takes one, so that a wave moves several at a time, and each lane one
// of two rows at a time where there are many (524288 slots of 128 bf16, gradients: 53 us, one 58, four 64).
#define RA_NARROW_THREADS 256
#define RA_NARROW_ROWS 2
// A lane's pack of a narrow row.  The last one ends where the row ends and so repeats elements of the one before it (`twice`), which
// both lanes read and write alike (the lanes of a row are one wave's: all have read before one writes).  Rows of 100 elements take 25, 28 and 83 us
// for dispatch, combine and its gradients this way, 39, 47 and 108 with single elements at the end (524288 slots, one set of inputs
// again and again; three sets in turn 45, 29 and 82).  Rows that do not end on a cache line take up to twice the time
// for their bytes: 128 elements 38, 27 and 54 us, 256 84, 50 and 105, 255 133, 62 and 170.  !WHOLE: a row shorter than a
// pack, moved element by element.
template <typename T, bool WHOLE> struct Narrow {
  size_t at; int twice; bool any;
  __device__ __forceinline__ Narrow(size_t hidden, uint32_t shift) {
    constexpr int N = Pack<T>::N;
    at = (threadIdx.x & ((1u << shift) - 1)) * N;
    any = at < hidden;
    twice = WHOLE && any && at + N > hidden ? (int)(at + N - hidden) : 0;
    at -= twice;
  }
  template <bool STREAM> __device__ __forceinline__ u32x4 load(const T* row, size_t hidden) const { return WHOLE ? wholePack<STREAM>(row + at) : loadPack<STREAM>(row, at, hidden); }
  template <bool STREAM> __device__ __forceinline__ void store(T* row, size_t hidden, u32x4 p) const {
    if (WHOLE) storeWhole<STREAM>(row + at, p);
    else storePack<STREAM>(row, at, hidden, p);
  }
};
template <typename T, bool WHOLE>
__global__ __launch_bounds__(RA_NARROW_THREADS) void raLocalKernelDispatchNarrow(RaRowsArgs a, uint32_t groups, uint32_t shift) {
  constexpr int F = RA_NARROW_ROWS;
  if (blockIdx.x >= groups) { padRows<T>(a, blockIdx.x - groups); return; }
  const size_t slots = a.tokens * a.topk, step = (size_t)groups * RA_NARROW_THREADS >> shift;
  const Narrow<T, WHOLE> mine(a.hidden, shift);
  if (!mine.any) return;
  for (size_t slot = ((size_t)blockIdx.x * RA_NARROW_THREADS + threadIdx.x) >> shift; slot < slots; slot += F * step) {
    int32_t pos[F];
    u32x4 p[F];
#pragma unroll
    for (int f = 0; f < F; f++) pos[f] = slot + f * step < slots ? a.position[slot + f * step] : -1;
#pragma unroll
    for (int f = 0; f < F; f++)
      if (pos[f] >= 0 && (size_t)pos[f] < a.rows) p[f] = mine.template load<false>((const T*)a.in + (size_t)((uint32_t)(slot + f * step) / (uint32_t)a.topk) * a.inStride, a.hidden);
#pragma unroll
    for (int f = 0; f < F; f++)
      if (pos[f] >= 0 && (size_t)pos[f] < a.rows) mine.template store<false>((T*)a.out + (size_t)pos[f] * a.outStride, a.hidden, p[f]);
  }
}

// Combine.  A wave takes 64 * U packs of one token's row (64 where there are few tokens) and adds those of its slots in the order
// of k, F rows in flight.  The same micro-batch back (1.21 GB):
// U = 4 and F = 4 0.205 ms, U = 2 0.209, U = 4 and F = 2 0.206 (F = 8 0.202, but with more registers than eight waves of a
// compute unit's SIMD have), accesses that are not streaming 0.235.
#define RA_COMBINE_THREADS 256
// WHOLE: all of the packs at element `at` + ... exist; otherwise those before `end` do.
template <typename T, int U, bool WHOLE>
static __device__ __forceinline__ void combineAt(const RaRowsArgs& a, T* y, uint32_t at, uint32_t end, uint64_t slots, int32_t pos, float w) {
  constexpr int N = Pack<T>::N, F = 4;
  typedef typename Pack<T>::floats floats;
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
      for (int u = 0; u < U; u++) if (WHOLE || at + u * 64 * N < end) p[f][u] = wholePack<true>(z + at + u * 64 * N); else p[f][u] = u32x4{0, 0, 0, 0};
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
#pragma unroll
  for (int u = 0; u < U; u++) if (WHOLE || at + u * 64 * N < end) storeWhole<true>(y + at + u * 64 * N, fromFloats<T>(sum[u]));
}
// The same for one element of each lane that has one.  All lanes run through it: what a slot has lies in the lane of its number.
template <typename T> static __device__ __forceinline__ void combineElement(const RaRowsArgs& a, T* y, uint32_t at, bool go, uint64_t slots, int32_t pos, float w) {
  constexpr int F = 8;
  float sum = 0.f;
  while (slots) {
    float z[F], wk[F];
#pragma unroll
    for (int f = 0; f < F; f++) {
      z[f] = wk[f] = 0.f;
      if (!slots) continue;
      const int k = __builtin_ctzll(slots);
      slots &= slots - 1;
      wk[f] = laneFloat(w, k);
      const size_t row = (size_t)laneInt(pos, k) * a.inStride;
      if (go) z[f] = (float)((const T*)a.in)[row + at];
    }
#pragma unroll
    for (int f = 0; f < F; f++) sum = __builtin_fmaf(wk[f], z[f], sum);      // (a slot that is not there adds 0 * 0)
  }
  if (go) y[at] = (T)sum;
}
template <typename T>
__global__ __launch_bounds__(RA_COMBINE_THREADS) void raLocalKernelCombine(RaRowsArgs a, uint32_t parts, uint32_t partElems) {
  constexpr uint32_t N = Pack<T>::N, U = 4;
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t units = (uint64_t)a.tokens * parts;
  for (uint64_t unit = (uint64_t)blockIdx.x * (RA_COMBINE_THREADS / 64) + uniform(threadIdx.x >> 6); unit < units;
       unit += (uint64_t)gridDim.x * (RA_COMBINE_THREADS / 64)) {
    const size_t token = unit / parts;
    int32_t pos = -1;
    float w = 1.f;
    if (lane < (uint32_t)a.topk) {
      pos = a.position[token * a.topk + lane];
      if (a.weightType >= 0) w = weightOf(a.weights, a.weightType, token * a.topk + lane);
    }
    const uint64_t slots = __ballot(pos >= 0 && (size_t)pos < a.rows);
    T* y = (T*)a.out + token * a.outStride;
    const RowCut c = cutRow(y, a.hidden);
    const uint32_t run = (uint32_t)(unit % parts) * partElems;
    const uint32_t at = c.head + run + lane * N, end = c.head + (run + partElems < c.body ? run + partElems : c.body);
    if (partElems == 64 * N) combineAt<T, 1, false>(a, y, at, end, slots, pos, w);
    else if (c.head + run + U * 64 * N <= end) combineAt<T, U, true>(a, y, at, end, slots, pos, w);
    else combineAt<T, U, false>(a, y, at, end, slots, pos, w);
    if (run == 0 && c.single) combineElement(a, y, elementOf(c.head, a.hidden, c.single, lane), lane < c.single, slots, pos, w);
  }
}

// Rows of at most 32 packs: `1 << shift` lanes for each token.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(RA_NARROW_THREADS) void raLocalKernelCombineNarrow(RaRowsArgs a, uint32_t shift) {
  constexpr int N = Pack<T>::N, F = 4;
  typedef typename Pack<T>::floats floats;
  const size_t step = (size_t)gridDim.x * RA_NARROW_THREADS >> shift;
  const Narrow<T, WHOLE> mine(a.hidden, shift);
  if (!mine.any) return;
  for (size_t token = ((size_t)blockIdx.x * RA_NARROW_THREADS + threadIdx.x) >> shift; token < a.tokens; token += step) {
    floats sum = {};
    for (int k = 0; k < a.topk; k += F) {
      u32x4 p[F];
      float w[F];
#pragma unroll
      for (int f = 0; f < F; f++) {
        p[f] = u32x4{0, 0, 0, 0};
        w[f] = 0.f;
        if (k + f >= a.topk) continue;
        const size_t slot = token * a.topk + k + f;
        const int32_t pos = a.position[slot];
        if (pos < 0 || (size_t)pos >= a.rows) continue;
        w[f] = a.weightType >= 0 ? weightOf(a.weights, a.weightType, slot) : 1.f;
        p[f] = mine.template load<true>((const T*)a.in + (size_t)pos * a.inStride, a.hidden);
      }
#pragma unroll
      for (int f = 0; f < F; f++) {                        // (a slot that is not there adds 0 * 0)
        const floats z = toFloats<T>(p[f]);
#pragma unroll
        for (int i = 0; i < N; i++) sum[i] = __builtin_fmaf(w[f], z[i], sum[i]);
      }
    }
    mine.template store<true>((T*)a.out + token * a.outStride, a.hidden, fromFloats<T>(sum));
  }
}

// The sum of x over the wave, in lane 63: inside rows of 16 lanes, then rows 0 and 2 into 1 and 3, then 1 into 3 (DPP moves).
template <int CTRL, int ROWS> static __device__ __forceinline__ float dppAdd(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, ROWS, 0xF, false));
}
static __device__ __forceinline__ float waveSum63(float x) {
  x = dppAdd<0xB1, 0xF>(x);
  x = dppAdd<0x4E, 0xF>(x);
  x = dppAdd<0x141, 0xF>(x);
  x = dppAdd<0x140, 0xF>(x);
  x = dppAdd<0x142, 0xA>(x);
  return dppAdd<0x143, 0xC>(x);
}

// w * dy of a pack; the pack's part of <dy, z> is added to `dot`.
template <typename T> static __device__ __forceinline__ u32x4 gradients(u32x4 z, u32x4 dy, float w, float& dot) {
  const typename Pack<T>::floats zf = toFloats<T>(z), d = toFloats<T>(dy);
  typename Pack<T>::floats g;
#pragma unroll
  for (int i = 0; i < Pack<T>::N; i++) { dot = __builtin_fmaf(d[i], zf[i], dot); g[i] = w * d[i]; }
  return fromFloats<T>(g);
}

// The gradients of combine.  A wave takes S slots: dz's rows are written while z's rows pass, and their products stay in the
// wave.  Runs of 8 KiB as in dispatch: half of the slots of 16384 tokens (1.17 to 1.38 GB, as routing goes) 0.211 to 0.246 ms = 5.5 TB/s, a copy
// has 6.3; runs of 4 KiB 3 % slower, 2 KiB 5 %; a workgroup for each token, its row in registers, no faster.
template <typename T, int S>
__global__ __launch_bounds__(RA_SLOT_WAVES * 64) RA_FEW_WAVES(S == 1 ? 4 : 8) void raLocalKernelCombineBackward(RaSlots n, RaRowsArgs a) {
  constexpr uint32_t N = Pack<T>::N, V = S == 1 ? 4 : 4 / S;      // packs of a slot in what is left of its row
  if (blockIdx.x >= n.groups) { padRows<T>(a, blockIdx.x - n.groups); return; }
  const uint32_t wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t each = slotsEach<S>(n);
  const uint32_t units = (n.slots + each - 1) / each;
  for (uint32_t unit = blockIdx.x; unit < units; unit += n.groups) {
    const uint32_t slot = unit * each + lane;
    const bool exists = lane < each && slot < n.slots;
    int32_t pos = -1;
    float weight = 0.f;
    if (exists) { pos = a.position[slot]; weight = weightOf(a.weights, a.weightType, slot); }
    const uint32_t token = (uint32_t)((uint64_t)slot * n.inverse >> n.shift);
    const bool keep = pos >= 0 && (uint32_t)pos < n.rows;
    if (wave == 0 && exists && !keep) storeWeight(a.dweights, a.weightType, slot, 0.f);
    for (uint64_t kept = sharedOut<S>(keep, wave); kept;) {
      const T* dy[S];
      const T* z[S];
      T* dz[S];
      RowCut c[S];
      bool go[S];
      uint32_t from[S];
      float w[S], dot[S];
#pragma unroll
      for (int s = 0; s < S; s++) {
        go[s] = kept != 0;
        const int k = go[s] ? __builtin_ctzll(kept) : 0;
        from[s] = (uint32_t)k;
        kept &= kept - 1;
        w[s] = laneFloat(weight, k);
        dot[s] = 0.f;
        const size_t row = go[s] ? laneInt(pos, k) : 0;
        dy[s] = (const T*)a.in + (size_t)(uint32_t)laneInt(token, k) * a.inStride;
        z[s] = (const T*)a.z + row * a.zStride;
        dz[s] = (T*)a.out + row * a.outStride;
        c[s] = cutRow(dz[s], a.hidden);
      }
      uint32_t run = 0;
      if (S == 1) {
        constexpr uint32_t U = 8;
        for (; run + U * 64 * N <= c[0].body; run += U * 64 * N) {
          const uint32_t at = c[0].head + run + lane * N;
          u32x4 p[U], q[U];
#pragma unroll
          for (uint32_t u = 0; u < U; u++) { p[u] = wholePack<true>(z[0] + at + u * 64 * N); q[u] = wholePack<false>(dy[0] + at + u * 64 * N); }
#pragma unroll
          for (uint32_t u = 0; u < U; u++) {
            storeWhole<true>(dz[0] + at + u * 64 * N, gradients<T>(p[u], q[u], w[0], dot[0]));
            __builtin_amdgcn_sched_barrier(0);               // one pack as floats at a time: the packs take half of the registers
          }
        }
      }
      do {
        u32x4 p[S][V], q[S][V];
#pragma unroll
        for (int s = 0; s < S; s++) {
          const uint32_t at = c[s].head + run + lane * N;
#pragma unroll
          for (uint32_t v = 0; v < V; v++)
            if (go[s] && run + (v * 64 + lane) * N < c[s].body) { p[s][v] = wholePack<true>(z[s] + at + v * 64 * N); q[s][v] = wholePack<false>(dy[s] + at + v * 64 * N); }
        }
#pragma unroll
        for (int s = 0; s < S; s++) {
          const uint32_t at = c[s].head + run + lane * N;
#pragma unroll
          for (uint32_t v = 0; v < V; v++)
            if (go[s] && run + (v * 64 + lane) * N < c[s].body) storeWhole<true>(dz[s] + at + v * 64 * N, gradients<T>(p[s][v], q[s][v], w[s], dot[s]));
        }
        run += V * 64 * N;
      } while (S == 1 && run < c[0].body);
#pragma unroll
      for (int s = 0; s < S; s++) {
        if (go[s] && lane < c[s].single) {
          const uint32_t i = elementOf(c[s].head, a.hidden, c[s].single, lane);
          const float d = (float)dy[s][i];
          dot[s] = __builtin_fmaf(d, (float)z[s][i], dot[s]);
          dz[s][i] = (T)(w[s] * d);
        }
      }
#pragma unroll
      for (int s = 0; s < S; s++) {
        const float sum = laneFloat(waveSum63(dot[s]), 63);
        if (go[s] && lane == from[s]) storeWeight(a.dweights, a.weightType, slot, sum);
      }
    }
  }
}

// Rows of at most 32 packs: `1 << shift` lanes for each slot.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(RA_NARROW_THREADS) void raLocalKernelCombineBackwardNarrow(RaRowsArgs a, uint32_t groups, uint32_t shift) {
  constexpr int N = Pack<T>::N, F = RA_NARROW_ROWS;
  if (blockIdx.x >= groups) { padRows<T>(a, blockIdx.x - groups); return; }
  const size_t slots = a.tokens * a.topk, step = (size_t)groups * RA_NARROW_THREADS >> shift;
  const Narrow<T, WHOLE> mine(a.hidden, shift);
  for (size_t slot = ((size_t)blockIdx.x * RA_NARROW_THREADS + threadIdx.x) >> shift; slot < slots; slot += F * step) {
    int32_t pos[F];
    float w[F], dot[F];
    u32x4 p[F], q[F];
#pragma unroll
    for (int f = 0; f < F; f++) {
      pos[f] = slot + f * step < slots ? a.position[slot + f * step] : -1;
      if ((size_t)(uint32_t)pos[f] >= a.rows) pos[f] = -1;
      dot[f] = 0.f;
    }
#pragma unroll
    for (int f = 0; f < F; f++)
      if (pos[f] >= 0 && mine.any) {
        w[f] = weightOf(a.weights, a.weightType, slot + f * step);
        q[f] = mine.template load<false>((const T*)a.in + (size_t)((uint32_t)(slot + f * step) / (uint32_t)a.topk) * a.inStride, a.hidden);
        p[f] = mine.template load<true>((const T*)a.z + (size_t)pos[f] * a.zStride, a.hidden);
      }
#pragma unroll
    for (int f = 0; f < F; f++)
      if (pos[f] >= 0 && mine.any) {
        const typename Pack<T>::floats z = toFloats<T>(p[f]), d = toFloats<T>(q[f]);
        typename Pack<T>::floats g;
#pragma unroll
        for (int i = 0; i < N; i++) { dot[f] = i >= mine.twice ? __builtin_fmaf(d[i], z[i], dot[f]) : dot[f]; g[i] = w[f] * d[i]; }
        mine.template store<true>((T*)a.out + (size_t)pos[f] * a.outStride, a.hidden, fromFloats<T>(g));
      }
#pragma unroll
    for (int f = 0; f < F; f++) {
      for (int s = 1; s < 1 << shift; s <<= 1) dot[f] += __shfl_xor(dot[f], s);      // (the lanes of a slot run together)
      if ((threadIdx.x & ((1u << shift) - 1)) == 0 && slot + f * step < slots) storeWeight(a.dweights, a.weightType, slot + f * step, dot[f]);
    }
  }
}

static uint32_t padGroups(const RaRowsArgs& a) { return a.offsets ? (uint32_t)a.nExperts * RA_PAD_GROUPS : 0; }

// Workgroups for so many waves: one each, up to 2^20 workgroups, beyond which a wave takes several in turn (a launch has fewer
// than 2^32 threads).
static uint32_t groupsOf(uint64_t units, int threads) {
  const uint64_t g = (units + threads / 64 - 1) / (threads / 64);
  return (uint32_t)(g < 1u << 20 ? g : 1u << 20);
}

// Workgroups for slots of which as many may be kept as there are rows.
static uint32_t slotGroups(const RaSlots& n, int S) { return groupsOf((((uint64_t)n.slots - 1) >> doublings(n, n.rows)) / (RA_SLOT_WAVES * S) + 1, 64); }

// Workgroups for narrow rows: two rows for each lane where that leaves 8192 waves.
static uint32_t narrowGroups(uint64_t rows, uint32_t shift) {
  const uint64_t waves = (rows + (63 >> shift)) >> (6 - shift);
  return groupsOf(waves >= 8192 * RA_NARROW_ROWS ? (waves + RA_NARROW_ROWS - 1) / RA_NARROW_ROWS : waves, RA_NARROW_THREADS);
}

// Lanes for a row of few packs, as a power of two; 6 (a whole wave): the row is not narrow.
template <typename T> static uint32_t narrowShift(const RaRowsArgs& a) {
  uint32_t shift = 0;
  while (shift < 6 && ((uint64_t)Pack<T>::N << shift) < a.hidden) shift++;
  return shift;
}
template <typename T, int S>
static hipError_t launchDispatch(const RaRowsArgs& a, uint32_t parts, uint32_t partElems, hipStream_t s) {
  RaSlots n = slotsOf(a, S, true);
  n.groups = n.slots == 0 ? 0 : parts > 1 ? groupsOf((uint64_t)n.slots * parts, RA_SLOT_WAVES * 64) : slotGroups(n, S);
  return raLaunch(raLocalKernelDispatch<T, S>, n.groups + padGroups(a), RA_SLOT_WAVES * 64, 0, s, n, a, parts, partElems);
}
template <typename T> static hipError_t dispatch(const RaRowsArgs& a, hipStream_t s) {
  const uint32_t shift = narrowShift<T>(a);
  const uint64_t slots = (uint64_t)a.tokens * a.topk, step = 64 * Pack<T>::N;
  if (shift < 6) {
    const uint32_t groups = narrowGroups(slots, shift);
    return raLaunch(a.hidden >= Pack<T>::N ? raLocalKernelDispatchNarrow<T, true> : raLocalKernelDispatchNarrow<T, false>, groups + padGroups(a), RA_NARROW_THREADS, 0, s, a, groups, shift);
  }
  // Short rows: several slots for a wave, where that leaves 4096 waves
  const uint64_t runs = (a.hidden + step - 1) / step;
  if (runs <= 1 && slots >= 8 * 4096) return launchDispatch<T, 8>(a, 1, 0, s);
  if (runs <= 2 && slots >= 4 * 4096) return launchDispatch<T, 4>(a, 1, 0, s);
  if (runs <= 4 && slots >= 2 * 4096) return launchDispatch<T, 2>(a, 1, 0, s);
  // parts of a row, down to 64 packs, where there are fewer than 4096 waves otherwise
  uint64_t parts = 1;
  while (parts < runs && slots * parts < 4096) parts *= 2;
  const uint64_t partElems = ((a.hidden + parts - 1) / parts + step - 1) / step * step;
  parts = (a.hidden + partElems - 1) / partElems;
  return launchDispatch<T, 1>(a, (uint32_t)parts, (uint32_t)partElems, s);
}
template <typename T> static hipError_t combine(const RaRowsArgs& a, hipStream_t s) {
  const uint32_t shift = narrowShift<T>(a);
  if (shift < 6) {
    return raLaunch(a.hidden >= Pack<T>::N ? raLocalKernelCombineNarrow<T, true> : raLocalKernelCombineNarrow<T, false>, groupsOf((a.tokens + (63 >> shift)) >> (6 - shift), RA_NARROW_THREADS), RA_NARROW_THREADS, 0, s, a, shift);
  }
  const uint64_t step = 64 * Pack<T>::N;
  // four runs of 64 packs for each wave, or one where that leaves fewer than 4096 waves
  const size_t partElems = a.tokens * ((a.hidden + 4 * step - 1) / (4 * step)) < 4096 ? step : 4 * step;
  const uint64_t parts = (a.hidden + partElems - 1) / partElems;
  return raLaunch(raLocalKernelCombine<T>, groupsOf(a.tokens * parts, RA_COMBINE_THREADS), RA_COMBINE_THREADS, 0, s, a, (uint32_t)parts, (uint32_t)partElems);
}
template <typename T> static hipError_t combineBackward(const RaRowsArgs& a, hipStream_t s) {
  const uint32_t shift = narrowShift<T>(a);
  if (shift < 6) {
    const uint32_t groups = narrowGroups((uint64_t)a.tokens * a.topk, shift);
    return raLaunch(a.hidden >= Pack<T>::N ? raLocalKernelCombineBackwardNarrow<T, true> : raLocalKernelCombineBackwardNarrow<T, false>, groups + padGroups(a), RA_NARROW_THREADS, 0, s, a, groups, shift);
  }
  const uint64_t slots = (uint64_t)a.tokens * a.topk, runs = (a.hidden + 64 * Pack<T>::N - 1) / (64 * Pack<T>::N);
  const int at = runs <= 1 && slots >= 4096 * 4 ? 4 : runs <= 2 && slots >= 4096 * 2 ? 2 : 1;
  RaSlots n = slotsOf(a, at, false);
  n.groups = n.slots ? slotGroups(n, at) : 0;
  const uint32_t groups = n.groups + padGroups(a);
  return at == 4 ? raLaunch(raLocalKernelCombineBackward<T, 4>, groups, RA_SLOT_WAVES * 64, 0, s, n, a)
       : at == 2 ? raLaunch(raLocalKernelCombineBackward<T, 2>, groups, RA_SLOT_WAVES * 64, 0, s, n, a)
                 : raLaunch(raLocalKernelCombineBackward<T, 1>, groups, RA_SLOT_WAVES * 64, 0, s, n, a);
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
