// Kernel arguments and launchers of the local operators of a sharded training step (kernels_shard.hip, kernels_expert.hip).
#pragma once
#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#include "rccl_amd.h"

// Launches a kernel and returns what that launch says.  (The error that hipGetLastError gives may be an older one of the
// caller's program, which is not this library's to report or to clear.)
template <typename T> struct RaSame { typedef T type; };
template <typename... A>
static inline hipError_t raLaunch(void (*kernel)(A...), uint32_t grid, int block, size_t lds, hipStream_t s, const typename RaSame<A>::type&... args) {
  void* p[] = {(void*)&args...};
  return hipLaunchKernel((const void*)kernel, dim3(grid), dim3((unsigned)block), p, lds, s);
}

// ------------------------------------------------------------------ AdamW, sum of squares
// Everything a launch needs travels in its arguments (at most 4 KiB): no table in device memory, nothing to allocate or to
// keep alive, and a captured launch stays valid.  In the general form a tensor takes `stride` words: the pointers the launch
// uses (a form without copies or scales leaves theirs out, so that more tensors fit) and its element count.  Tensors that
// lie alike in flat buffers, as shards do, need only their element offset and count: 300 fit into a launch.
#define RA_ADAMW_WORDS 414           // 8-byte words of tensor descriptions: 82 tensors of 5 words, 51 of 8
#define RA_ADAMW_MAX 82
#define RA_ADAMW_FLAT 300
#define RA_ADAMW_THREADS 256
#define RA_ADAMW_ROW 256             // elements a wave takes in one step: 4 for each lane
enum { RA_W_COUNT = 0, RA_W_PARAM = 1, RA_W_GRAD = 2, RA_W_M = 3, RA_W_V = 4, RA_W_MS = 5, RA_W_VS = 6 };   // then copy

struct RaAdamWGeneral {
  uint64_t words[RA_ADAMW_WORDS];
  uint32_t first[RA_ADAMW_MAX];      // first chunk (= workgroup) of each tensor
};
struct RaAdamWFlat {
  uint64_t base[8];                  // the pointers of the tensor at offset 0, in the places of a general tensor's words
  uint32_t offset[RA_ADAMW_FLAT], count[RA_ADAMW_FLAT], first[RA_ADAMW_FLAT];
};
struct RaAdamWArgs {
  union { RaAdamWGeneral general; RaAdamWFlat flat; };
  double lr, beta1, beta2, weightDecay, gradScale, maxNorm;
  const int64_t* stepPtr;
  const float* lrPtr;
  const double* sumSq;
  int64_t step;
  uint64_t seed;
  float b1, omb1, b2, omb2, eps, decay, stepSize, rootC2, coef;   // the same in fp32, where nothing is read from the device
  uint32_t n, stride, chunk;         // tensors, words for each (0: flat), elements of a chunk (a multiple of 4 rows)
  uint32_t ordinal;                  // place of the first tensor in the call
  int copyWord, copyType;            // word of the copy's pointer (-1: none), its ncclDataType_t
};
static_assert(sizeof(RaAdamWArgs) <= 4096, "kernel arguments");
hipError_t raLaunchAdamW(const RaAdamWArgs& a, int paramType, int gradType, bool mx, uint32_t grid, hipStream_t s);

#define RA_SUMSQ_MAX 248
#define RA_SUMSQ_THREADS 256
struct RaSumSqArgs {
  const void* ptr[RA_SUMSQ_MAX];
  uint32_t count[RA_SUMSQ_MAX];
  uint32_t first[RA_SUMSQ_MAX];      // first chunk of each tensor
  double* partial;                   // where the sum of this launch's chunk 0 goes
  double* out;                       // not null: the launch is the whole call and has one chunk
  uint32_t n, chunk;
  int accumulate;
};
static_assert(sizeof(RaSumSqArgs) <= 4096, "kernel arguments");
hipError_t raLaunchSumSq(const RaSumSqArgs& a, int type, uint32_t grid, hipStream_t s);
hipError_t raLaunchSumSqJoin(const double* partial, uint32_t n, double* out, int accumulate, hipStream_t s);

// ------------------------------------------------------------------ expert order
#define RA_SORT_THREADS 1024
#define RA_SORT_MAX_EXPERTS 1024
struct RaSortArgs {
  const void* ids;
  int64_t firstExpert;
  int32_t* position;
  int32_t* source;
  int32_t* offsets;
  int32_t* counts;
  int32_t* tileCounts;               // [tiles + 1][nExperts], tiles > 1
  uint32_t slots, rows, tiles;
  int nExperts, rowAlign, idBytes;
  bool scanned;                      // raSortScanned
};
// Rounds of 64 slots a wave takes in one tile (a tile is RA_SORT_THREADS * rounds): one tile up to 4096 slots, which is one
// launch; beyond that 2, and 4 for many tiles.  In us, with 2, 4 and 8 rounds: 131072 slots of 256 experts 11.0, 13.5, 18.7; 524288 of 128
// experts 13.2, 14.6, 18.4; 1 million 16.6, 17.6, 21.7; 2 million of 64 experts 25.4, 23.0, 24.8; 4.2 million of 128 experts 46.6, 42.1, 45.3.
static inline uint32_t raSortRounds(uint64_t slots) {
  return slots <= 1024 ? 1 : slots <= 2048 ? 2 : slots <= 4096 ? 4 : slots <= 1u << 20 ? 2 : 4;
}
static inline uint64_t raSortTiles(uint64_t slots) {
  const uint64_t tile = (uint64_t)RA_SORT_THREADS * raSortRounds(slots);
  return (slots + tile - 1) / tile;
}
// The next power of two of the number of experts.
static inline __host__ __device__ uint32_t raSortWidth(int nExperts) { return nExperts <= 1 ? 1 : 1u << (32 - __builtin_clz((unsigned)nExperts - 1)); }
// Every tile adds up the counts of all tiles by itself where that is at most 8 steps of its threads; otherwise a launch between
// the two does it once (524288 slots of 16 experts: 8.8 us without it, 10.9 with it; 131072 of 128 experts 9.8 and 10.5, of 256
// experts 12.5 and 11.0).
static inline bool raSortScanned(uint64_t tiles, int nExperts) { return tiles > 1 && tiles * raSortWidth(nExperts) > 8 * RA_SORT_THREADS; }
hipError_t raLaunchSort(const RaSortArgs& a, hipStream_t s);

#define RA_ROWS_MAX_TOPK 64
struct RaRowsArgs {
  const void* in;                    // dispatch: x; combine: z; backward: dy
  const void* z;                     // backward
  void* out;                         // dispatch: out; combine: y; backward: dz
  const void* weights;
  void* dweights;
  const int32_t* position;
  const int32_t* offsets;            // of the padding rows of `out`, or null
  const int32_t* counts;
  size_t inStride, zStride, outStride;   // elements
  size_t tokens, hidden, rows;
  int topk, nExperts, weightType;    // weightType -1: no weights
};
hipError_t raLaunchDispatch(const RaRowsArgs& a, int type, hipStream_t s);
hipError_t raLaunchCombine(const RaRowsArgs& a, int type, hipStream_t s);
hipError_t raLaunchCombineBackward(const RaRowsArgs& a, int type, hipStream_t s);
