// The exported local operators of a sharded training step: argument checks, how work is cut, launches.
#include <float.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "comm.h"
#include "debug.h"
#include "local_ops.h"

#define RA_API extern "C" __attribute__((visibility("default")))

// A refused argument: the message for ncclGetLastError, and the code.
#define RA_REFUSE(...) do { RA_WARN(__VA_ARGS__); return ncclInvalidArgument; } while (0)
#define RA_LAUNCH(what, call)                                                        \
  do {                                                                               \
    hipError_t e_ = (call);                                                          \
    if (e_ != hipSuccess) {                                                          \
      RA_WARN("%s: launch failed: %s", what, hipGetErrorString(e_));                 \
      return ncclUnhandledCudaError;                                                 \
    }                                                                                \
  } while (0)

// Kernels run on the current device; a stream of another one would take them, and buffers they may not reach, there.
static ncclResult_t checkStream(const char* fn, hipStream_t stream) {
  int own = 0, current = 0;
  if ((uintptr_t)stream <= (uintptr_t)hipStreamPerThread) return ncclSuccess;      // the default streams are the current device's
  if (hipStreamGetDevice(stream, &own) != hipSuccess || hipGetDevice(&current) != hipSuccess) RA_REFUSE("%s: the stream has no device", fn);
  if (own != current) RA_REFUSE("%s: the stream belongs to device %d, the current device is %d", fn, own, current);
  return ncclSuccess;
}
static bool isFloat(int t) { return t == ncclFloat32 || t == ncclBfloat16 || t == ncclFloat16; }
static bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
static const uint64_t kMaxElements = 1ull << 40;      // of one call: byte offsets and chunk numbers stay far from overflow
static const size_t kMaxRow = 1u << 28;               // elements of a row and its stride: so do the offsets of 2^31 rows

// x^n by squaring, in the same steps as the kernel that reads the step number from the device.
static double powN(double x, int64_t n) {
  double r = 1.0;
  for (; n > 0; n >>= 1, x *= x) if (n & 1) r *= x;
  return r;
}

// The words of a tensor: its count and the pointers that its form of the call uses.
static void describe(const rcclAmdAdamWTensor_t& t, bool mx, bool copies, uint64_t* w) {
  w[RA_W_COUNT] = t.count;
  w[RA_W_PARAM] = (uint64_t)t.param; w[RA_W_GRAD] = (uint64_t)t.grad; w[RA_W_M] = (uint64_t)t.expAvg; w[RA_W_V] = (uint64_t)t.expAvgSq;
  if (mx) { w[RA_W_MS] = (uint64_t)t.expAvgScale; w[RA_W_VS] = (uint64_t)t.expAvgSqScale; }
  if (copies) w[mx ? RA_W_VS + 1 : RA_W_V + 1] = (uint64_t)t.copy;
}

// Whether every tensor is the same run of elements of its flat buffers, counted from the tensor with the lowest address,
// whose pointers go to `base`: param + o, grad + o, the moments + o (their scales + o / 32) and the copy + o, or no copies.
static bool liesFlat(const rcclAmdAdamWTensor_t* tensors, int n, bool mx, size_t ps, size_t gs, size_t cs, uint64_t* base) {
  const rcclAmdAdamWTensor_t* b = nullptr;
  for (int i = 0; i < n; i++) if (tensors[i].count && (!b || tensors[i].param < b->param)) b = &tensors[i];
  if (!b) return false;
  const size_t ss = mx ? 1 : 4;
  for (int i = 0; i < n; i++) {
    const rcclAmdAdamWTensor_t& t = tensors[i];
    if (t.count == 0) continue;
    const uintptr_t bytes = (uintptr_t)t.param - (uintptr_t)b->param, o = bytes / ps;
    if (bytes % ps || o > 0xFFFFFFFF || t.count > 0xFFFFFFFF) return false;
    if ((uintptr_t)t.grad - (uintptr_t)b->grad != o * gs || (uintptr_t)t.expAvg - (uintptr_t)b->expAvg != o * ss || (uintptr_t)t.expAvgSq - (uintptr_t)b->expAvgSq != o * ss) return false;
    if (mx && (o % RCCL_AMD_STATE_BLOCK || (uintptr_t)t.expAvgScale - (uintptr_t)b->expAvgScale != o / RCCL_AMD_STATE_BLOCK ||
               (uintptr_t)t.expAvgSqScale - (uintptr_t)b->expAvgSqScale != o / RCCL_AMD_STATE_BLOCK)) return false;
    if (!t.copy != !b->copy || (t.copy && (uintptr_t)t.copy - (uintptr_t)b->copy != o * cs)) return false;
  }
  describe(*b, mx, b->copy != nullptr, base);
  return true;
}

RA_API ncclResult_t rcclAmdAdamW(const rcclAmdAdamWTensor_t* tensors, int ntensors, ncclDataType_t paramType, ncclDataType_t gradType,
                                 ncclDataType_t copyType, rcclAmdStateType_t stateType, const rcclAmdAdamWConfig_t* config,
                                 hipStream_t stream) {
  const char* fn = "rcclAmdAdamW";
  if (ntensors < 0 || (ntensors > 0 && !tensors) || !config) RA_REFUSE("%s: %d tensors, null argument", fn, ntensors);
  if (!isFloat(paramType) || !isFloat(gradType)) RA_REFUSE("%s: parameter type %d / gradient type %d is not float32, bfloat16 or float16", fn, (int)paramType, (int)gradType);
  if (stateType != rcclAmdStateF32 && stateType != rcclAmdStateMx8) RA_REFUSE("%s: unknown state type %d", fn, (int)stateType);
  const rcclAmdAdamWConfig_t& c = *config;
  if (!isfinite(c.lr) || !isfinite(c.weightDecay) || !isfinite(c.gradScale) || !isfinite(c.eps) || c.eps < 0.0 || c.gradScale < 0.0)
    RA_REFUSE("%s: lr, weightDecay, gradScale and eps must be finite, gradScale and eps not negative", fn);
  if ((c.eps > 0.0 && c.eps < FLT_MIN) || c.eps > FLT_MAX) RA_REFUSE("%s: eps %g is %s normal fp32 number", fn, c.eps, c.eps < 1.0 ? "below the smallest" : "above the largest");
  // (the kernel of the 8-bit states multiplies with the divisor's reciprocal, which has to be a normal number too)
  if (stateType == rcclAmdStateMx8 && c.eps > 0x1p126) RA_REFUSE("%s: eps %g is above 2^126, the largest with 8-bit states", fn, c.eps);
  if (!(c.beta1 >= 0.0 && c.beta1 < 1.0 && c.beta2 >= 0.0 && c.beta2 < 1.0)) RA_REFUSE("%s: beta1 = %g, beta2 = %g outside 0 <= beta < 1", fn, c.beta1, c.beta2);
  if (!c.stepPtr && c.step < 1) RA_REFUSE("%s: step %lld: the first step is 1", fn, (long long)c.step);
  if (c.sumSq && !(c.maxNorm >= 0.0)) RA_REFUSE("%s: maxNorm %g with sumSq", fn, c.maxNorm);
  if (!aligned(c.stepPtr, 8) || !aligned(c.lrPtr, 4) || !aligned(c.sumSq, 8)) RA_REFUSE("%s: misaligned stepPtr, lrPtr or sumSq", fn);
  const bool mx = stateType == rcclAmdStateMx8;
  const size_t ps = raTypeSize(paramType), gs = raTypeSize(gradType), cs = isFloat(copyType) ? raTypeSize(copyType) : 1;
  bool copies = false;
  uint64_t all = 0;
  for (int i = 0; i < ntensors; i++) {
    const rcclAmdAdamWTensor_t& t = tensors[i];
    if (t.count == 0) continue;
    if (t.count > kMaxElements || (all += t.count) > kMaxElements) RA_REFUSE("%s: tensor %d: %zu elements, or too many in all", fn, i, t.count);
    if (!t.param || !t.grad || !t.expAvg || !t.expAvgSq || (mx && (!t.expAvgScale || !t.expAvgSqScale))) RA_REFUSE("%s: tensor %d has a null buffer", fn, i);
    // (what has scales has moments of one byte: taken for floats they would be read and written far past their end)
    if (!mx && (t.expAvgScale || t.expAvgSqScale)) RA_REFUSE("%s: tensor %d has scales, which 32-bit states have not", fn, i);
    if (!aligned(t.param, ps) || !aligned(t.grad, gs) || (!mx && (!aligned(t.expAvg, 4) || !aligned(t.expAvgSq, 4))) || !aligned(t.copy, cs))
      RA_REFUSE("%s: tensor %d has a buffer that is not aligned to its element type", fn, i);
    copies = copies || t.copy;
  }
  if (copies && !isFloat(copyType)) RA_REFUSE("%s: copy type %d is not float32, bfloat16 or float16", fn, (int)copyType);
  if (all) RA_CHECK(checkStream(fn, stream));

  RaAdamWArgs a;
  a.lr = c.lr; a.beta1 = c.beta1; a.beta2 = c.beta2; a.weightDecay = c.weightDecay; a.gradScale = c.gradScale; a.maxNorm = c.maxNorm;
  a.stepPtr = c.stepPtr; a.lrPtr = c.lrPtr; a.sumSq = c.sumSq; a.step = c.step; a.seed = c.seed;
  a.b1 = (float)c.beta1; a.omb1 = (float)(1.0 - c.beta1); a.b2 = (float)c.beta2; a.omb2 = (float)(1.0 - c.beta2); a.eps = (float)c.eps;
  a.decay = (float)(1.0 - c.lr * c.weightDecay);
  a.stepSize = (float)(c.lr / (1.0 - powN(c.beta1, c.step)));
  a.rootC2 = (float)(1.0 / sqrt(1.0 - powN(c.beta2, c.step)));
  a.coef = (float)c.gradScale;
  a.copyType = copies ? (int)copyType : -1;
  a.copyWord = copies ? (mx ? RA_W_VS + 1 : RA_W_V + 1) : -1;
  a.stride = (mx ? RA_W_VS : RA_W_V) + (copies ? 2 : 1);
  const uint32_t stride = a.stride;
  const int general = RA_ADAMW_WORDS / (int)stride < RA_ADAMW_MAX ? RA_ADAMW_WORDS / (int)stride : RA_ADAMW_MAX;
  const bool flat = ntensors > general && liesFlat(tensors, ntensors, mx, ps, gs, cs, a.flat.base);
  const int fit = flat ? RA_ADAMW_FLAT : general;
  if (flat) a.stride = 0;
  // A chunk is the work of one workgroup: a row for each wave (1024 elements), with 8-bit states up to two, or four where
  // parameter and gradient have 16 bits and there is no copy, where there is much to do (see the kernel).
  const uint64_t unit = RA_ADAMW_THREADS / 64 * RA_ADAMW_ROW, most = ps + gs + (copies ? cs : 0) > 4 ? 2 : 4;
  for (int lo = 0; lo < ntensors; lo += fit) {
    const int n = ntensors - lo < fit ? ntensors - lo : fit;
    uint64_t elements = 0, chunks = 0;
    for (int i = 0; i < n; i++) elements += tensors[lo + i].count;
    if (elements == 0) continue;
    uint64_t chunk = mx ? (elements / 4096 + unit - 1) / unit * unit : unit;
    chunk = chunk < unit ? unit : chunk > most * unit ? most * unit : chunk;
    while (elements / chunk > 1u << 22) chunk *= 2;       // (a launch has fewer than 2^32 threads)
    for (int i = 0; i < n; i++) {
      const rcclAmdAdamWTensor_t& t = tensors[lo + i];
      if (flat) {
        a.flat.offset[i] = t.count ? (uint32_t)(((uintptr_t)t.param - a.flat.base[RA_W_PARAM]) / ps) : 0;
        a.flat.count[i] = (uint32_t)t.count;
        a.flat.first[i] = (uint32_t)chunks;
      } else {
        describe(t, mx, copies, a.general.words + (size_t)i * stride);
        a.general.first[i] = (uint32_t)chunks;
      }
      chunks += (t.count + chunk - 1) / chunk;
    }
    a.n = (uint32_t)n; a.chunk = (uint32_t)chunk; a.ordinal = (uint32_t)lo;
    RA_LAUNCH(fn, raLaunchAdamW(a, paramType, gradType, mx, (uint32_t)chunks, stream));
  }
  return ncclSuccess;
}

RA_API ncclResult_t rcclAmdSumSquaresBytes(int ntensors, size_t* workspaceBytes) {
  if (ntensors < 0 || !workspaceBytes) RA_REFUSE("rcclAmdSumSquaresBytes: %d tensors, null argument", ntensors);
  *workspaceBytes = ntensors ? (8192 + (size_t)ntensors) * sizeof(double) : 0;
  return ncclSuccess;
}

RA_API ncclResult_t rcclAmdSumSquares(const void* const* tensors, const size_t* counts, int ntensors, ncclDataType_t datatype,
                                      double* out, int accumulate, void* workspace, size_t workspaceBytes, hipStream_t stream) {
  const char* fn = "rcclAmdSumSquares";
  if (ntensors < 0 || (ntensors > 0 && (!tensors || !counts)) || !out) RA_REFUSE("%s: %d tensors, null argument", fn, ntensors);
  if (!isFloat(datatype)) RA_REFUSE("%s: type %d is not float32, bfloat16 or float16", fn, (int)datatype);
  if (!aligned(out, 8) || !aligned(workspace, 16)) RA_REFUSE("%s: misaligned out or workspace", fn);
  size_t need = 0;
  RA_CHECK(rcclAmdSumSquaresBytes(ntensors, &need));
  if (workspaceBytes < need || (need && !workspace)) RA_REFUSE("%s: workspace of %zu bytes, %zu needed", fn, workspaceBytes, need);
  const size_t size = raTypeSize(datatype);
  uint64_t all = 0;
  for (int i = 0; i < ntensors; i++) {
    if (counts[i] > kMaxElements || (all += counts[i]) > kMaxElements) RA_REFUSE("%s: tensor %d: %zu elements, or too many in all", fn, i, counts[i]);
    if (counts[i] && (!tensors[i] || !aligned(tensors[i], size))) RA_REFUSE("%s: tensor %d is null or not aligned to its element type", fn, i);
  }
  RA_CHECK(checkStream(fn, stream));
  // Chunks: at most 4096 of equal size and one more for each tensor (and for each 2^31 elements of one, which is what an
  // entry of a launch holds), so the partial sums fit the workspace.
  const uint64_t unit = RA_SUMSQ_THREADS * 4 * 4, piece = 1ull << 31;
  uint64_t chunk = (all / 4096 + unit) / unit * unit;
  if (chunk > piece) chunk = piece;
  RaSumSqArgs a;
  a.chunk = (uint32_t)chunk; a.accumulate = accumulate != 0;
  const bool single = all <= chunk && ntensors == 1;
  uint64_t done = 0;                                      // chunks of earlier launches
  uint64_t chunks = 0;
  a.n = 0;
  for (int i = 0; i < ntensors; i++) {
    uint64_t at = 0;
    while (at < counts[i]) {
      const uint64_t len = counts[i] - at < piece ? counts[i] - at : piece;
      a.ptr[a.n] = (const char*)tensors[i] + at * size;
      a.count[a.n] = (uint32_t)len;
      a.first[a.n] = (uint32_t)chunks;
      chunks += (len + chunk - 1) / chunk;
      at += len;
      if (++a.n == RA_SUMSQ_MAX) {
        a.partial = (double*)workspace + done; a.out = nullptr;
        RA_LAUNCH(fn, raLaunchSumSq(a, datatype, (uint32_t)chunks, stream));
        done += chunks; chunks = 0; a.n = 0;
      }
    }
  }
  if (a.n) {
    a.partial = (double*)workspace + done; a.out = single ? out : nullptr;
    RA_LAUNCH(fn, raLaunchSumSq(a, datatype, (uint32_t)chunks, stream));
    done += chunks;
    if (single) return ncclSuccess;
  }
  RA_LAUNCH(fn, raLaunchSumSqJoin((const double*)workspace, (uint32_t)done, out, a.accumulate, stream));
  return ncclSuccess;
}

static ncclResult_t checkSlots(const char* fn, size_t tokens, int topk) {
  if (topk < 1 || topk > RA_ROWS_MAX_TOPK) RA_REFUSE("%s: topk %d, 1 .. %d supported", fn, topk, RA_ROWS_MAX_TOPK);
  if (tokens > 0x7FFFFFFFull / (unsigned)topk) RA_REFUSE("%s: %zu tokens of %d slots: 2^31 - 1 slots at most", fn, tokens, topk);
  return ncclSuccess;
}

RA_API ncclResult_t rcclAmdExpertSortBytes(size_t tokens, int topk, int nExperts, size_t* workspaceBytes) {
  const char* fn = "rcclAmdExpertSortBytes";
  RA_CHECK(checkSlots(fn, tokens, topk));
  if (nExperts < 1 || nExperts > RA_SORT_MAX_EXPERTS || !workspaceBytes) RA_REFUSE("%s: %d experts, 1 .. %d supported, or a null argument", fn, nExperts, RA_SORT_MAX_EXPERTS);
  const uint64_t tiles = raSortTiles((uint64_t)tokens * topk);
  *workspaceBytes = tiles > 1 ? (size_t)(tiles + 1) * nExperts * sizeof(int32_t) : 0;
  return ncclSuccess;
}

RA_API ncclResult_t rcclAmdExpertSort(const void* experts, ncclDataType_t expertType, size_t tokens, int topk, int64_t firstExpert,
                                      int nExperts, int rowAlign, int32_t* position, int32_t* source, int32_t* offsets,
                                      int32_t* counts, void* workspace, size_t workspaceBytes, hipStream_t stream) {
  const char* fn = "rcclAmdExpertSort";
  size_t need = 0;
  RA_CHECK(rcclAmdExpertSortBytes(tokens, topk, nExperts, &need));
  if (expertType != ncclInt32 && expertType != ncclInt64) RA_REFUSE("%s: expert type %d is not int32 or int64", fn, (int)expertType);
  if (rowAlign < 1 || rowAlign > 1024) RA_REFUSE("%s: rowAlign %d, 1 .. 1024 supported", fn, rowAlign);
  if (firstExpert < 0 || firstExpert > INT64_MAX - nExperts) RA_REFUSE("%s: first expert %lld", fn, (long long)firstExpert);
  const uint64_t slots = (uint64_t)tokens * topk, rows = slots + (uint64_t)nExperts * (rowAlign - 1);
  if (rows > 0x7FFFFFFF) RA_REFUSE("%s: %llu rows, 2^31 - 1 at most", fn, (unsigned long long)rows);
  if (slots && (!experts || !position)) RA_REFUSE("%s: null experts or position", fn);
  if (!aligned(experts, raTypeSize(expertType)) || !aligned(position, 4) || !aligned(source, 4) || !aligned(offsets, 4) || !aligned(counts, 4) || !aligned(workspace, 16))
    RA_REFUSE("%s: misaligned buffer", fn);
  if (workspaceBytes < need || (need && !workspace)) RA_REFUSE("%s: workspace of %zu bytes, %zu needed", fn, workspaceBytes, need);
  RA_CHECK(checkStream(fn, stream));
  RaSortArgs a;
  a.ids = experts; a.firstExpert = firstExpert; a.position = position; a.source = source; a.offsets = offsets; a.counts = counts;
  a.tileCounts = (int32_t*)workspace; a.slots = (uint32_t)slots; a.rows = (uint32_t)rows;
  a.tiles = slots ? (uint32_t)raSortTiles(slots) : 1;
  a.nExperts = nExperts; a.rowAlign = rowAlign; a.idBytes = (int)raTypeSize(expertType);
  a.scanned = raSortScanned(a.tiles, nExperts);
  RA_LAUNCH(fn, raLaunchSort(a, stream));
  return ncclSuccess;
}

// What the three row operators ask of their arguments alike.
static ncclResult_t checkRows(const char* fn, const RaRowsArgs& a, int datatype, size_t outRowsLimit) {
  RA_CHECK(checkSlots(fn, a.tokens, a.topk));
  if (!isFloat(datatype)) RA_REFUSE("%s: type %d is not float32, bfloat16 or float16", fn, datatype);
  const size_t s = raTypeSize(datatype);
  if (a.hidden < 1 || a.hidden > kMaxRow) RA_REFUSE("%s: rows of %zu elements", fn, a.hidden);
  if (a.rows > 0x7FFFFFFF) RA_REFUSE("%s: %zu rows, 2^31 - 1 at most", fn, a.rows);
  if (a.inStride < a.hidden || a.outStride < a.hidden || (a.z && a.zStride < a.hidden)) RA_REFUSE("%s: a stride is below the %zu elements of a row", fn, a.hidden);
  if (a.inStride > kMaxRow || a.outStride > kMaxRow || a.zStride > kMaxRow) RA_REFUSE("%s: a stride is too large", fn);
  if (!a.offsets != !a.counts) RA_REFUSE("%s: offsets and counts belong together", fn);
  if (a.offsets && (a.nExperts < 1 || a.nExperts > RA_SORT_MAX_EXPERTS)) RA_REFUSE("%s: %d experts, 1 .. %d supported", fn, a.nExperts, RA_SORT_MAX_EXPERTS);
  if (a.weightType >= 0 && !isFloat(a.weightType)) RA_REFUSE("%s: weight type %d is not float32, bfloat16 or float16", fn, a.weightType);
  if (a.tokens && (!a.position || !a.in)) RA_REFUSE("%s: null buffer", fn);
  if (outRowsLimit && !a.out) RA_REFUSE("%s: null output", fn);
  if (!aligned(a.in, s) || !aligned(a.z, s) || !aligned(a.out, s) || !aligned(a.position, 4) || !aligned(a.offsets, 4) || !aligned(a.counts, 4) ||
      (a.weightType >= 0 && (!aligned(a.weights, raTypeSize(a.weightType)) || !aligned(a.dweights, raTypeSize(a.weightType)))))
    RA_REFUSE("%s: a buffer is not aligned to its element type", fn);
  return ncclSuccess;
}

RA_API ncclResult_t rcclAmdExpertDispatch(const void* x, size_t xStride, void* out, size_t outStride, size_t rows,
                                          ncclDataType_t datatype, size_t tokens, int topk, size_t hidden, const int32_t* position,
                                          const int32_t* offsets, const int32_t* counts, int nExperts, hipStream_t stream) {
  const char* fn = "rcclAmdExpertDispatch";
  RaRowsArgs a = {x, nullptr, out, nullptr, nullptr, position, offsets, counts, xStride, 0, outStride, tokens, hidden, rows, topk, nExperts, -1};
  RA_CHECK(checkRows(fn, a, datatype, rows));
  if (rows && x == out) RA_REFUSE("%s: x and out are the same buffer", fn);
  if (rows == 0 || (tokens == 0 && !offsets)) return ncclSuccess;
  RA_CHECK(checkStream(fn, stream));
  RA_LAUNCH(fn, raLaunchDispatch(a, datatype, stream));
  return ncclSuccess;
}

RA_API ncclResult_t rcclAmdExpertCombine(const void* z, size_t zStride, size_t rows, const void* weights, ncclDataType_t weightType,
                                         void* y, size_t yStride, ncclDataType_t datatype, size_t tokens, int topk, size_t hidden,
                                         const int32_t* position, hipStream_t stream) {
  const char* fn = "rcclAmdExpertCombine";
  if (weights && !isFloat(weightType)) RA_REFUSE("%s: weight type %d is not float32, bfloat16 or float16", fn, (int)weightType);
  // without rows z is not read, and may be null
  RaRowsArgs a = {rows ? z : y, nullptr, y, weights, nullptr, position, nullptr, nullptr, zStride, 0, yStride, tokens, hidden, rows, topk, 0,
                  weights ? (int)weightType : -1};
  RA_CHECK(checkRows(fn, a, datatype, tokens));
  if (tokens && rows && z == y) RA_REFUSE("%s: z and y are the same buffer", fn);
  if (tokens == 0) return ncclSuccess;
  RA_CHECK(checkStream(fn, stream));
  RA_LAUNCH(fn, raLaunchCombine(a, datatype, stream));
  return ncclSuccess;
}

RA_API ncclResult_t rcclAmdExpertCombineBackward(const void* dy, size_t dyStride, const void* z, size_t zStride, size_t rows,
                                                 const void* weights, ncclDataType_t weightType, void* dz, size_t dzStride,
                                                 void* dweights, ncclDataType_t datatype, size_t tokens, int topk, size_t hidden,
                                                 const int32_t* position, const int32_t* offsets, const int32_t* counts,
                                                 int nExperts, hipStream_t stream) {
  const char* fn = "rcclAmdExpertCombineBackward";
  if (!isFloat(weightType)) RA_REFUSE("%s: weight type %d is not float32, bfloat16 or float16", fn, (int)weightType);
  RaRowsArgs a = {dy, z, dz, weights, dweights, position, offsets, counts, dyStride, zStride, dzStride, tokens, hidden, rows, topk, nExperts, (int)weightType};
  RA_CHECK(checkRows(fn, a, datatype, rows));
  if (tokens && (!weights || !dweights)) RA_REFUSE("%s: null weights or dweights", fn);
  if (rows && !z) RA_REFUSE("%s: null z", fn);
  if (rows && (dy == dz || dy == z || (z == dz && zStride != dzStride))) RA_REFUSE("%s: dy overlaps, or dz is z with another stride", fn);
  if (tokens && (dweights == weights)) RA_REFUSE("%s: weights and dweights are the same buffer", fn);
  if (tokens == 0 && (rows == 0 || !offsets)) return ncclSuccess;
  RA_CHECK(checkStream(fn, stream));
  RA_LAUNCH(fn, raLaunchCombineBackward(a, datatype, stream));
  return ncclSuccess;
}
