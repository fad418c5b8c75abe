// Host side shared by the row operators (rows.cu, row_sort.cu): argument
// checks, the widest access a set of rows allows, launch error handling.
#pragma once

#include "gpu_common.h"

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <initializer_list>

namespace nmb {
namespace rows {

inline int elemBytes(int type) { return type == GPUX_ELEM_F64 ? 8 : type == GPUX_ELEM_F32 ? 4 : 2; }

// The queue's stream with its device current; puts the caller's device back.
struct Stream {
  cudaStream_t stream = nullptr;
  int device = 0;
  bool ok = false;
  explicit Stream(void *queue) {
    if (cudaGetDevice(&before_) != cudaSuccess)
      (void)cudaGetLastError();
    QueueView qv;
    if (!queueView(queue, &qv))
      return;
    stream = static_cast<cudaStream_t>(qv.stream);
    device = qv.device;
    ok = true;
  }
  ~Stream() {
    if (ok && before_ >= 0 && before_ != device)
      (void)cudaSetDevice(before_);
  }

private:
  int before_ = -1;
};

// The workspace of one call: the caller's, or, where it gave none, memory of the
// stream-ordered pool that goes back behind the call's last kernel.  Recorded
// into a graph the two become nodes of that graph, so graphs share nothing.
class Workspace {
public:
  Workspace(const Stream &s, const char *who, void *given, size_t givenBytes, size_t need) : stream_(s.stream) {
    if (given) {
      if (reinterpret_cast<uintptr_t>(given) % 256 != 0 || givenBytes < need) {
        setError("%s: the workspace is not aligned to 256 bytes or holds %zu bytes of the %zu needed", who,
                 givenBytes, need);
        return;
      }
      data = given;
    } else if (need > 0) {
      keepPool(s.device);
      const cudaError_t e = cudaMallocAsync(&taken_, need, s.stream);
      if (e != cudaSuccess) {
        taken_ = nullptr;
        setError("%s: no workspace of %zu bytes: %s", who, need, cudaGetErrorString(e));
        (void)cudaGetLastError();
        return;
      }
      data = taken_;
    }
    ok = true;
  }
  ~Workspace() {
    if (taken_ && cudaFreeAsync(taken_, stream_) != cudaSuccess)
      (void)cudaGetLastError();
  }
  Workspace(const Workspace &) = delete;
  Workspace &operator=(const Workspace &) = delete;
  void *data = nullptr;
  bool ok = false;

private:
  // What gpuxQueueCreate sets for its device, for queues made over a foreign
  // stream: freed memory stays in the pool.
  static void keepPool(int device) {
    static std::atomic<bool> done[64];
    if (device < 0 || device >= 64 || done[device])
      return;
    cudaMemPool_t pool;
    if (cudaDeviceGetDefaultMemPool(&pool, device) == cudaSuccess) {
      uint64_t threshold = UINT64_MAX;
      cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &threshold);
    }
    (void)cudaGetLastError();
    done[device] = true;
  }
  cudaStream_t stream_;
  void *taken_ = nullptr;
};

// Reports a failed launch; counts a good one.
inline bool launched(const char *who) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    setError("%s: launch failed: %s", who, cudaGetErrorString(e));
    return false;
  }
  noteLaunch();
  return true;
}

// Launches a kernel that may begin while the kernel before it in the stream, one
// of the same call, is still running (it calls let_next_begin): its blocks are
// set up and then wait in wait_for_previous before they read what that kernel
// and those before it write.  Not `behind`: the stream's last work is not this
// call's, nobody knows what that in turn has waited for, and the kernel begins when
// all of it is done.
template <typename K, typename... Args>
inline void launchBehind(K kernel, dim3 grid, unsigned threads, size_t shared, cudaStream_t stream, bool behind,
                         Args... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = behind ? 1 : 0;
  (void)cudaLaunchKernelEx(&config, kernel, args...);
}
#ifdef __CUDACC__
// A kernel completes only when the one before it has, since each that is
// launched behind another waits for it: so a wait covers all kernels before.
__device__ __forceinline__ void let_next_begin() { cudaTriggerProgrammaticLaunchCompletion(); }
__device__ __forceinline__ void wait_for_previous() { cudaGridDependencySynchronize(); }
// What the kernels before this one of the same call have written.  This kernel's
// blocks may be on their multiprocessors while it is being written, so it is never
// read through the read-only path (__ldg, or a pointer that is const and
// __restrict__), which is for memory that nobody writes while the kernel lives.  An
// ordinary load: wait_for_previous makes those writes visible to it.  (Loads past
// L1 cost more where neighbours read the same words: dispatch of 30000 x 2 rows of
// 259 bf16 63.8 us against 41.1, the gradient of 60000 skewed ids of 32 bf16 57
// against 39.)
template <typename T> __device__ __forceinline__ T made(const T *p) { return *p; }
#endif

// Lets a kernel use more than 48 KB of shared memory; once per kernel and device.
template <typename K> inline bool allowShared(const char *who, K kernel, int bytes, std::atomic<bool> *ready, int device) {
  if (device >= 0 && device < 64 && ready[device])
    return true;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) {
    setError("%s: cudaFuncSetAttribute failed: %s", who, cudaGetErrorString(e));
    (void)cudaGetLastError();
    return false;
  }
  if (device >= 0 && device < 64)
    ready[device] = true;
  return true;
}

inline bool checkRows(const char *who, const char *name, const GPUXRows *r, bool result) {
  if (!r) {
    setError("%s: %s is null", who, name);
    return false;
  }
  if (r->type < GPUX_ELEM_F32 || r->type > GPUX_ELEM_BF16) {
    setError("%s: %s has an unknown element type %d", who, name, (int)r->type);
    return false;
  }
  if (r->rows < 0 || r->cols < 0 || r->rows >= (int64_t(1) << 40) || r->cols >= (int64_t(1) << 31)) {
    setError("%s: %s has an impossible shape", who, name);
    return false;
  }
  if (r->rows == 0 || r->cols == 0)
    return true;
  if (!r->data || reinterpret_cast<uintptr_t>(r->data) % (uintptr_t)elemBytes(r->type) != 0) {
    setError("%s: the data of %s is null or not aligned to its elements", who, name);
    return false;
  }
  if (result && r->rows > 1 && r->stride < r->cols && r->stride > -r->cols) {
    setError("%s: the rows of %s overlap", who, name);
    return false;
  }
  return true;
}

inline bool checkIndex(const char *who, const GPUXIndex *ids) {
  if (!ids || ids->count < 0 || (ids->bytes != 4 && ids->bytes != 8) ||
      (ids->count > 0 &&
       (!ids->data || reinterpret_cast<uintptr_t>(ids->data) % (uintptr_t)ids->bytes != 0))) {
    setError("%s: the indices must be aligned 4- or 8-byte integers", who);
    return false;
  }
  if (ids->count >= (int64_t(1) << 31)) {
    setError("%s: 2^31 indices or more", who);
    return false;
  }
  return true;
}

inline bool checkGroups(const char *who, const GPUXIndex *ids, int64_t groups, const int32_t *order,
                        const int32_t *place, const int32_t *offsets) {
  if (groups < 0 || groups >= 0x7fffffff) {
    setError("%s: the number of groups must be in 0 .. 2^31 - 2", who);
    return false;
  }
  if (!offsets || (ids->count > 0 && (!order || !place))) {
    setError("%s: null result", who);
    return false;
  }
  return true;
}

// Elements per access: the largest power of two up to `most` such that every
// row of every operand begins aligned for an access of that many of its
// elements (16 bytes and more need 16-byte alignment only) and the width is a
// multiple of it.
inline int accessElems(int64_t cols, int most, std::initializer_list<const GPUXRows *> operands) {
  for (int v = most; v > 1; v /= 2) {
    bool fits = cols % v == 0;
    for (const GPUXRows *r : operands) {
      const int64_t bytes = (int64_t)elemBytes(r->type) * v < 16 ? (int64_t)elemBytes(r->type) * v : 16;
      const int64_t step = r->rows > 1 ? r->stride * elemBytes(r->type) : 0;
      fits = fits && reinterpret_cast<uintptr_t>(r->data) % (uintptr_t)bytes == 0 && step % bytes == 0;
    }
    if (fits)
      return v;
  }
  return 1;
}

// log2 of the threads that share a row of `vecs` accesses: the next power of
// two, at most a block.
inline int laneBits(int64_t vecs, int most) {
  int b = 0;
  while ((int64_t(1) << b) < vecs && b < most)
    ++b;
  return b;
}

// Rows of a result that the sort's launches set to zero on the side, from the
// last one down: a sort keeps few multiprocessors busy.  `left` is the number of
// rows at the front that are not set yet.
struct Clearing {
  unsigned char *data = nullptr;
  int64_t left = 0;
  int64_t rowBytes = 0, stride = 0; // in bytes
  int unit = 1;                     // bytes per access: 16, 8, 4 or 2
};

// Stable sort of the indices by key, key = id inside [0, groups), groups for
// every other id.  Any of the results may be null: order[j] = entry at sorted
// position j, keys[j] its key, place[order[j]] = j, offsets[g] = position of
// the first key >= g for g <= groups.  `words` (the caller's, `wordCount` of them)
// are set to zero, and rows of `clearing`.
size_t sortBytes(int64_t count, int64_t groups);
bool sortByKey(const Stream &s, const char *who, const GPUXIndex &ids, int64_t groups, int32_t *order,
               uint32_t *keys, int32_t *place, int32_t *offsets, void *workspace, uint32_t *words = nullptr,
               int64_t wordCount = 0, Clearing *clearing = nullptr);

} // namespace rows
} // namespace nmb
