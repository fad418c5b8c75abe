// Rows picked, grouped and added by index: the embedding lookup and its
// gradient, tokens sorted by expert and back, and the gradients of both.
//
//   take         out[i,:]  = scale * table[ids[i],:]
//   take_grad    out[v,:]  = scale * sum of dout[i,:] over ids[i] == v
//   dispatch     out[place[t,j],:] = x[t,:]
//   combine      out[t,:]  = sum_j w[t,j] * ys[place[t,j],:]
//   combine_grad dys[place[t,j],:] = w[t,j] * dout[t,:],  dw[t,j] = dout[t,:] . ys[place[t,j],:]
//
// All of them move rows once and compute next to nothing, so memory bounds
// them: the layout is chosen for wide accesses and enough of them in flight.
// A narrow row is shared by a power of two of a block's threads (`lanes`), each
// thread moves `V` neighbouring elements per access (16 bytes where alignment
// and width allow), and blocks take several such rows.  Wide rows, and rows that
// do not begin on 16-byte boundaries, are brought into shared memory by bulk
// copies and read from there.  Arithmetic is float32 (float64 for float64 rows)
// and rounds once, on the way out.
#include "kernels/bulk_pipe.cuh"
#include "rows_host.h"

#include <atomic>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#define GPUX_EXPORT extern "C" __attribute__((visibility("default")))

namespace {

using nmb::rows::accessElems;
using nmb::rows::checkIndex;
using nmb::rows::checkRows;
using nmb::rows::elemBytes;
using nmb::rows::laneBits;
using nmb::rows::launched;
using nmb::rows::made;
using nmb::rows::Stream;

constexpr int kThreads = 256;
constexpr int kThreadBits = 8;
constexpr unsigned kAll = 0xffffffffu;

template <typename T> struct Acc { using type = float; };
template <> struct Acc<double> { using type = double; };

__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ double up(double v) { return v; }
__device__ __forceinline__ float up(__half v) { return __half2float(v); }
__device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
// one rounding to nearest even; a half past 65504 becomes an infinity
template <typename T, typename A> __device__ __forceinline__ T down(A v);
template <> __device__ __forceinline__ float down<float, float>(float v) { return v; }
template <> __device__ __forceinline__ double down<double, double>(double v) { return v; }
template <> __device__ __forceinline__ __half down<__half, float>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 down<__nv_bfloat16, float>(float v) {
  return __float2bfloat16_rn(v);
}
__device__ __forceinline__ float madd(float a, float b, float c) { return __fmaf_rn(a, b, c); }
__device__ __forceinline__ double madd(double a, double b, double c) { return __fma_rn(a, b, c); }

// Two neighbouring elements at a time: one instruction multiplies (and adds) a
// pair of float32, one rounds it to 16 bits.
__device__ __forceinline__ float2 up2(const float *p) { return make_float2(p[0], p[1]); }
__device__ __forceinline__ double2 up2(const double *p) { return make_double2(p[0], p[1]); }
__device__ __forceinline__ float2 up2(const __half *p) { return __half22float2(*reinterpret_cast<const __half2 *>(p)); }
__device__ __forceinline__ float2 up2(const __nv_bfloat16 *p) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(p));
}
__device__ __forceinline__ void down2(float *p, float2 v) { p[0] = v.x, p[1] = v.y; }
__device__ __forceinline__ void down2(double *p, double2 v) { p[0] = v.x, p[1] = v.y; }
__device__ __forceinline__ void down2(__half *p, float2 v) {
  *reinterpret_cast<__half2 *>(p) = __floats2half2_rn(v.x, v.y);
}
__device__ __forceinline__ void down2(__nv_bfloat16 *p, float2 v) {
  *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(v.x, v.y);
}
__device__ __forceinline__ uint64_t bits2(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 pair2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ float2 madd2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return pair2(r);
}
__device__ __forceinline__ double2 madd2(double2 a, double2 b, double2 c) {
  return make_double2(madd(a.x, b.x, c.x), madd(a.y, b.y, c.y));
}
__device__ __forceinline__ float2 mul2(float a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(make_float2(a, a))), "l"(bits2(b)));
  return pair2(r);
}
__device__ __forceinline__ double2 mul2(double a, double2 b) { return make_double2(a * b.x, a * b.y); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return pair2(r);
}
__device__ __forceinline__ double2 add2(double2 a, double2 b) { return make_double2(a.x + b.x, a.y + b.y); }
template <typename A> struct Two { using type = float2; };
template <> struct Two<double> { using type = double2; };

// V neighbouring elements, moved with 16-byte accesses where they fill one.
template <typename T, int V> struct alignas(sizeof(T) * V <= 16 ? sizeof(T) * V : 16) Pack {
  T v[V];
};
template <typename T, int V> __device__ __forceinline__ Pack<T, V> load(const T *p) {
  return *reinterpret_cast<const Pack<T, V> *>(p);
}
template <typename T, int V> __device__ __forceinline__ void store(T *p, const Pack<T, V> &x) {
  *reinterpret_cast<Pack<T, V> *>(p) = x;
}

// The same past L1, for what other blocks of the launch have written.
template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_l2(const T *p) {
  Pack<T, V> x;
  constexpr int bytes = (int)sizeof(T) * V;
  if constexpr (bytes >= 16) {
#pragma unroll
    for (int i = 0; i < bytes / 16; ++i)
      reinterpret_cast<int4 *>(&x)[i] = __ldcg(reinterpret_cast<const int4 *>(p) + i);
  } else if constexpr (bytes == 8) {
    *reinterpret_cast<int2 *>(&x) = __ldcg(reinterpret_cast<const int2 *>(p));
  } else {
    *reinterpret_cast<int *>(&x) = __ldcg(reinterpret_cast<const int *>(p));
  }
  return x;
}

// A signed index of 4 or 8 bytes.
__device__ __forceinline__ int64_t index_at(const void *ids, int bytes, int64_t i) {
  return bytes == 8 ? (int64_t)__ldg(static_cast<const long long *>(ids) + i)
                    : (int64_t)__ldg(static_cast<const int *>(ids) + i);
}

template <typename A> __device__ __forceinline__ A scalar_at(const void *p, int type, int64_t i) {
  if (type == GPUX_ELEM_F32)
    return (A) static_cast<const float *>(p)[i];
  if (type == GPUX_ELEM_F16)
    return (A)__half2float(static_cast<const __half *>(p)[i]);
  if (type == GPUX_ELEM_BF16)
    return (A)__bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
  return (A) static_cast<const double *>(p)[i];
}
template <typename A> __device__ __forceinline__ void set_scalar(void *p, int type, int64_t i, A v) {
  if (type == GPUX_ELEM_F32)
    static_cast<float *>(p)[i] = (float)v;
  else if (type == GPUX_ELEM_F16)
    static_cast<__half *>(p)[i] = __float2half_rn((float)v);
  else if (type == GPUX_ELEM_BF16)
    static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn((float)v);
  else
    static_cast<double *>(p)[i] = (double)v;
}

// Rows narrower than this are not fetched by bulk copies.
constexpr int kBulkLeast = 1024;

// The bound of the waits for bulk copies, and the queue's word that reports one
// that ran out.
struct Waits {
  uint32_t *status;
  uint32_t spins;
};

// Waits for the block's copies; all threads of the block come here.  Where the
// wait of one of them runs out the whole block gives up: that is reported in the
// queue's status word, the block stays for its copies (as long again at most), and
// what they were for is not written.  Behind it the threads also see what the
// others stored before it.
__device__ __forceinline__ bool bulk_arrived(uint64_t *bar, uint32_t phase, const Waits &waits) {
  const bool mine = nmb::mbar_wait(bar, phase, waits.spins);
  if (__syncthreads_and(mine))
    return true;
  if (!mine) {
    atomicExch(waits.status, (uint32_t)nmb::kStatusWaitTimeout);
    (void)nmb::mbar_wait(bar, phase);
  }
  return false;
}

// A row's way into shared memory, issued by one thread: a bulk copy starts and
// ends on 16-byte boundaries.  LOOSE rows do not: the words they lie in are copied
// as a whole, neighbours' elements included, as far as the operand's memory
// reaches; elements in the words at its very ends are copied one by one.  Those are
// ordinary stores: a thread that fetches into the same place again puts
// nmb::fence_async_smem in front, or the next copy may land before them.  Returns
// the place of the row's first element in `to`.
template <typename T> struct Bounds {
  const T *lo, *hi; // the operand's memory
};
template <bool LOOSE, typename T>
__device__ __forceinline__ int fetch_row(const T *from, int count, unsigned char *to, uint64_t *bar,
                                         const Bounds<T> &m) {
  if constexpr (!LOOSE) {
    nmb::mbar_expect_tx(bar, (uint32_t)count * (uint32_t)sizeof(T));
    nmb::bulk_load(to, from, (uint32_t)count * (uint32_t)sizeof(T), bar);
    return 0;
  } else {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(from), end = begin + (uintptr_t)count * sizeof(T);
    const uintptr_t base = begin & ~uintptr_t(15);
    uintptr_t a = base, b = (end + 15) & ~uintptr_t(15);
    if (a < reinterpret_cast<uintptr_t>(m.lo))
      a += 16;
    if (b > reinterpret_cast<uintptr_t>(m.hi))
      b -= 16;
    for (uintptr_t p = begin; p < min(a, end); p += sizeof(T))
      *reinterpret_cast<T *>(to + (p - base)) = *reinterpret_cast<const T *>(p);
    for (uintptr_t p = max(max(a, b), begin); p < end; p += sizeof(T))
      *reinterpret_cast<T *>(to + (p - base)) = *reinterpret_cast<const T *>(p);
    if (b > a) {
      nmb::mbar_expect_tx(bar, (uint32_t)(b - a));
      nmb::bulk_load(to + (a - base), reinterpret_cast<const void *>(a), (uint32_t)(b - a), bar);
    } else {
      nmb::mbar_arrive(bar);
    }
    return (int)((begin - base) / sizeof(T));
  }
}
// Bytes of shared memory for a row of `count` elements.
template <bool LOOSE, typename T> __host__ __device__ __forceinline__ int fetched_bytes(int count) {
  return ((int)sizeof(T) * count + 15) / 16 * 16 + (LOOSE ? 16 : 0);
}
// Elements per access of a row in shared memory.
template <bool LOOSE, typename T> constexpr int kBulkElems = LOOSE ? 1 : 16 / (int)sizeof(T);

// ------------------------------------------------------------------- take ---
// A thread has up to four accesses of a row in flight.
constexpr int kTakeBatch = 4;

template <typename I, typename O, int V>
__global__ void __launch_bounds__(kThreads)
    nmb_take_rows(const I *__restrict__ table, int64_t rows, int64_t stride, const void *__restrict__ ids, int id_bytes,
                  int64_t n, typename Acc<I>::type scale, O *__restrict__ out, int64_t out_stride, int64_t vecs,
                  int lane_bits) {
  using A = typename Acc<I>::type;
  const int lanes = 1 << lane_bits, lane = threadIdx.x & (lanes - 1);
  const int64_t i = (int64_t)blockIdx.x * (kThreads >> lane_bits) + (threadIdx.x >> lane_bits);
  if (i >= n)
    return;
  const int64_t id = index_at(ids, id_bytes, i);
  const bool inside = id >= 0 && id < rows;
  const I *src = table + (inside ? id : 0) * stride;
  O *dst = out + i * out_stride;
  for (int64_t c0 = lane; c0 < vecs; c0 += (int64_t)kTakeBatch * lanes) {
    Pack<I, V> x[kTakeBatch];
#pragma unroll
    for (int u = 0; u < kTakeBatch; ++u)
      if (inside && c0 + u * lanes < vecs)
        x[u] = load<I, V>(src + (c0 + u * lanes) * V);
#pragma unroll
    for (int u = 0; u < kTakeBatch; ++u)
      if (c0 + u * lanes < vecs) {
        Pack<O, V> y;
#pragma unroll
        for (int e = 0; e < V; ++e)
          y.v[e] = down<O, A>(inside ? up(x[u].v[e]) * scale : A(0));
        store<O, V>(dst + (c0 + u * lanes) * V, y);
      }
  }
}

// Wide rows by bulk copies: a block fetches `each` rows (a slab of each) into
// shared memory and scales them from there.  16384 bfloat16 rows of 4096 out of
// 131072 took 42.7 us (32.1 us where frequent rows repeat), through registers
// 50.7 us (40.7 us); below a few megabytes the two are alike.
constexpr int kTakeThreads = 128;
constexpr int kTakeRows = 16;          // most rows of a block
constexpr int kTakeBytes = 8192;       // most bytes in flight per block
constexpr int64_t kTakeBulkLeast = 8 << 20, kTakeLooseLeast = 1 << 20; // bytes from which on it pays

template <typename I, typename O, bool LOOSE>
__global__ void __launch_bounds__(kTakeThreads)
    nmb_take_rows_bulk(const I *__restrict__ table, int64_t rows, int64_t stride, const void *__restrict__ ids,
                       int id_bytes, int64_t n, typename Acc<I>::type scale, O *__restrict__ out, int64_t out_stride,
                       int64_t cols, int slab, int each, const Bounds<I> bounds, const Waits waits) {
  using A = typename Acc<I>::type;
  constexpr int V = kBulkElems<LOOSE, I>;
  extern __shared__ __align__(128) unsigned char memory[]; // [each] rows
  __shared__ uint64_t bar;
  __shared__ int at[kTakeRows]; // first element, -1: a row of zeros
  const int64_t i0 = (int64_t)blockIdx.x * each, first = (int64_t)blockIdx.y * slab;
  const int here = (int)min((int64_t)slab, cols - first), r = threadIdx.x, bytes = fetched_bytes<LOOSE, I>(slab);
  if (r == 0) {
    nmb::mbar_init(&bar, (uint32_t)each);
    nmb::mbar_init_fence();
  }
  __syncthreads();
  if (r < each) {
    const int64_t id = i0 + r < n ? index_at(ids, id_bytes, i0 + r) : -1;
    at[r] = -1;
    if (id >= 0 && id < rows)
      at[r] = fetch_row<LOOSE>(table + id * stride + first, here, memory + r * bytes, &bar, bounds);
    else
      nmb::mbar_arrive(&bar);
  }
  if (!bulk_arrived(&bar, 0, waits))
    return;
  const int live = (int)min((int64_t)each, n - i0);
  O *dst = out + i0 * out_stride + first;
  for (int j = 0; j < live; ++j, dst += out_stride) {
    const int begin = at[j];
    const I *src = reinterpret_cast<const I *>(memory + j * bytes) + max(begin, 0);
#pragma unroll 4
    for (int col = r * V; col < here; col += kTakeThreads * V) {
      if constexpr (LOOSE) {
        dst[col] = down<O, A>(begin < 0 ? A(0) : up(src[col]) * scale);
      } else {
        Pack<O, V> y{};
        if (begin >= 0) {
          const Pack<I, V> x = load<I, V>(src + col);
#pragma unroll
          for (int e = 0; e < V / 2; ++e)
            down2(y.v + 2 * e, mul2(scale, up2(x.v + 2 * e)));
        }
        store<O, V>(dst + col, y);
      }
    }
  }
}

// Threads per row: enough for four accesses each where there are rows enough to
// fill the multiprocessors that way, one access each otherwise.
int takeLaneBits(int64_t n, int64_t vecs) {
  const int wide = laneBits(vecs, kThreadBits);
  const int narrow = laneBits((vecs + kTakeBatch - 1) / kTakeBatch, kThreadBits);
  return n * (vecs / kTakeBatch) >= 148 * 2048 ? narrow : wide;
}

// -------------------------------------------------------------- take_grad ---
// The entries arrive sorted by row (keys, order), so a row's entries are a run
// of neighbours.  The sorted list is cut into chunks of `span` entries; a group
// of threads takes a chunk, a thread one access's width of columns, and adds up
// the runs that begin in the chunk.  Every incoming row is read once, every row
// of the result written once.  Rows of 1 KB and more come by bulk copies into
// shared memory, two turns of four rows in flight, and the group is a block;
// others come through registers, and a block holds several groups.
//
// A run that goes on past its chunk is finished by the group it began in, up
// to the first chunk that lies inside the run as a whole.  Those inner chunks
// add up their own entries, so a frequent token (padding, the end of a line)
// does not keep one group busy: all of the run's groups leave partial sums in
// the workspace, and the one that draws the last ticket adds them up in the
// order of the chunks (of 32 chunks at a time, then of those).  The order of
// additions is a function of the ids alone.
//
// Rows without entries are set to zero by blocks of their own, which look their
// rows up in the sorted keys, one row a lane.  The last rows (of a vocabulary:
// the rare tokens) have been cleared beside the sort, whether they have entries
// or not.
constexpr int kGradBatch = 4;   // incoming rows in flight per thread, through registers
constexpr int kTurnRows = 4;    // rows of a turn, by bulk copies
constexpr int kZeroRows = 32;   // rows looked up by a block that clears
constexpr int kBundle = 32;     // partial sums added up by one group

struct GradPlan {
  const int32_t *order;
  const uint32_t *keys;
  int64_t n;
  int span;
  unsigned slabs;          // groups side by side over the columns
  int slab;                // elements of a slab
  unsigned chunk_blocks;   // blocks over chunks
  unsigned period;         // one block of so many takes a chunk
  void *partials;          // [chunks][cols]
  uint32_t *tickets;       // [2][chunks][slabs], zero
  int64_t chunks;
  int64_t to_clear;        // rows that are not cleared yet, at the front
  int lane_bits;           // threads of a group, through registers
  Waits waits;
};

__device__ __forceinline__ int64_t lower_bound(const uint32_t *keys, int64_t lo, int64_t hi, uint32_t key) {
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (made(keys + mid) < key)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// The same for a warp that looks for one key: 32 places at a time, so four
// dependent reads where halving takes fifteen (an L2 access is about 0.4 us).
__device__ __forceinline__ int64_t warp_lower_bound(const uint32_t *keys, int64_t lo, int64_t hi, uint32_t key) {
  const int lane = threadIdx.x & 31;
  while (lo < hi) {
    const int64_t step = (hi - lo + 31) / 32, at = lo + lane * step;
    const int below = __popc(__ballot_sync(kAll, at < hi && made(keys + (at < hi ? at : lo)) < key));
    if (below == 0)
      return lo;
    hi = min(hi, lo + below * step);
    lo += (below - 1) * step + 1;
  }
  return lo;
}

// The end of the run of `key` that goes on at keys[at], and the begin of the one
// that keys[at - 1] belongs to, for the threads of a warp or for one.  Most runs
// end nearby: a warp looks at 1024 places first (two reads), a thread at ever
// longer steps.
__device__ __forceinline__ int64_t warp_run_end(const uint32_t *keys, int64_t at, int64_t n, uint32_t key) {
  const int64_t probe = at + (threadIdx.x & 31) * 32 + 31;
  const unsigned past = __ballot_sync(kAll, probe >= n || made(keys + (probe < n ? probe : at)) != key);
  if (past == 0)
    return warp_lower_bound(keys, at + 1024, n, key + 1);
  const int64_t first = at + (int64_t)(__ffs(past) - 1) * 32, place = first + (threadIdx.x & 31);
  return first + __popc(__ballot_sync(kAll, place < n && made(keys + (place < n ? place : at)) == key));
}
__device__ __forceinline__ int64_t warp_run_begin(const uint32_t *keys, int64_t at, uint32_t key) {
  const int64_t probe = at - 32 - (threadIdx.x & 31) * 32;
  const unsigned past = __ballot_sync(kAll, probe < 0 || made(keys + (probe < 0 ? at - 1 : probe)) != key);
  if (past == 0)
    return warp_lower_bound(keys, 0, at - 1024, key);
  const int64_t last = at - (int64_t)(__ffs(past) - 1) * 32, place = last - 1 - (threadIdx.x & 31);
  return last - __popc(__ballot_sync(kAll, place >= 0 && made(keys + (place < 0 ? at - 1 : place)) == key));
}
__device__ __forceinline__ int64_t run_end(const uint32_t *keys, int64_t at, int64_t n, uint32_t key) {
  int64_t step = 1;
  while (at + step < n && made(keys + at + step) == key) {
    at += step;
    step *= 2;
  }
  return lower_bound(keys, at, min(at + step, n), key + 1);
}
__device__ __forceinline__ int64_t run_begin(const uint32_t *keys, int64_t at, uint32_t key) {
  int64_t step = 1;
  while (at - step >= 0 && made(keys + at - step) == key) {
    at -= step;
    step *= 2;
  }
  return lower_bound(keys, max(at - step, (int64_t)0), at, key);
}

// The threads that share a chunk: a block, or 1 << bits of its threads.
template <bool BLOCK> struct Group {
  int bits, lanes, lane, number;
  __device__ __forceinline__ explicit Group(int lane_bits)
      : bits(lane_bits), lanes(BLOCK ? (int)blockDim.x : 1 << lane_bits),
        lane(BLOCK ? (int)threadIdx.x : threadIdx.x & ((1 << lane_bits) - 1)),
        number(BLOCK ? 0 : threadIdx.x >> lane_bits) {}
  __device__ __forceinline__ unsigned mask() const { // of a group inside a warp
    return bits >= 5 ? kAll : ((1u << lanes) - 1) << ((threadIdx.x & 31) & ~(lanes - 1));
  }
  __device__ __forceinline__ void sync() const {
    if (BLOCK)
      __syncthreads();
    else if (bits <= 5)
      __syncwarp(mask());
    else
      asm volatile("bar.sync %0, %1;" ::"r"(number + 1), "r"(lanes) : "memory");
  }
  // lane 0's value; `words` is shared, one word per group
  __device__ __forceinline__ uint32_t first(uint32_t v, uint32_t *words) const {
    if (!BLOCK && bits <= 5)
      return __shfl_sync(mask(), v, (threadIdx.x & 31) & ~(lanes - 1));
    if (lane == 0)
      words[number] = v;
    sync();
    v = words[number];
    sync();
    return v;
  }
  __device__ __forceinline__ int64_t find(const uint32_t *keys, int64_t lo, int64_t hi, uint32_t key) const {
    return BLOCK || bits >= 5 ? warp_lower_bound(keys, lo, hi, key) : lower_bound(keys, lo, hi, key);
  }
  __device__ __forceinline__ int64_t end_of(const uint32_t *keys, int64_t at, int64_t n, uint32_t key) const {
    return BLOCK || bits >= 5 ? warp_run_end(keys, at, n, key) : run_end(keys, at, n, key);
  }
  __device__ __forceinline__ int64_t begin_of(const uint32_t *keys, int64_t at, uint32_t key) const {
    return BLOCK || bits >= 5 ? warp_run_begin(keys, at, key) : run_begin(keys, at, key);
  }
};

// V sums, kept and added in pairs where there are pairs.
template <typename A, int V> struct Sums {
  static constexpr int kPairs = V / 2;
  typename Two<A>::type pair[kPairs > 0 ? kPairs : 1];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int e = 0; e < (kPairs > 0 ? kPairs : 1); ++e)
      pair[e].x = pair[e].y = A(0);
  }
  template <typename T> __device__ __forceinline__ void add(const Pack<T, V> &x) {
    if constexpr (V == 1) {
      pair[0].x += up(x.v[0]);
    } else {
#pragma unroll
      for (int e = 0; e < kPairs; ++e)
        pair[e] = add2(pair[e], up2(x.v + 2 * e));
    }
  }
  // scale * sum, or that added to `old`
  template <bool ADD, typename O> __device__ __forceinline__ Pack<O, V> result(A scale, const Pack<O, V> &old) const {
    Pack<O, V> y;
    if constexpr (V == 1) {
      y.v[0] = down<O, A>(ADD ? madd(scale, pair[0].x, up(old.v[0])) : scale * pair[0].x);
    } else {
      typename Two<A>::type s;
      s.x = s.y = scale;
#pragma unroll
      for (int e = 0; e < kPairs; ++e)
        down2(y.v + 2 * e, ADD ? madd2(s, pair[e], up2(old.v + 2 * e)) : mul2(scale, pair[e]));
    }
    return y;
  }
  __device__ __forceinline__ Pack<A, V> values() const {
    Pack<A, V> y;
    if constexpr (V == 1) {
      y.v[0] = pair[0].x;
    } else {
#pragma unroll
      for (int e = 0; e < kPairs; ++e)
        down2(y.v + 2 * e, pair[e]);
    }
    return y;
  }
};

// Sets a row to zero: 16-byte stores between its own boundaries.
template <typename O> __device__ __forceinline__ void clear_row(O *row, int64_t cols, int lane, int lanes) {
  const int64_t head =
      min(cols, (int64_t)((-reinterpret_cast<intptr_t>(row) & 15) / (int)sizeof(O)));
  const int64_t whole = (cols - head) * (int64_t)sizeof(O) / 16, tail = head + whole * (16 / (int)sizeof(O));
  int4 *words = reinterpret_cast<int4 *>(row + head);
  for (int64_t i = lane; i < whole; i += lanes)
    words[i] = make_int4(0, 0, 0, 0);
  for (int64_t i = lane; i < head; i += lanes)
    row[i] = O(0.0f);
  for (int64_t i = tail + lane; i < cols; i += lanes)
    row[i] = O(0.0f);
}

// A thread's columns of the result: V neighbouring ones, or, LOOSE, every step-th
// one.
template <typename O, int V, bool ADD, bool LOOSE, typename A> struct GradColumn {
  O *out;          // the thread's first column of row 0
  int64_t stride;
  A scale;
  bool active;     // threads without columns go along for the barriers
  int live, step;  // LOOSE: how many columns, how far apart
  __device__ __forceinline__ Pack<O, V> old(uint32_t row) const {
    Pack<O, V> v{};
    if constexpr (ADD && LOOSE) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < live)
          v.v[e] = out[(int64_t)row * stride + e * step];
    } else if (ADD && active) {
      v = load<O, V>(out + (int64_t)row * stride);
    }
    return v;
  }
  // A run's row: scale * sum, or that added to what the row holds.
  __device__ __forceinline__ void write(uint32_t row, const Sums<A, V> &sum, const Pack<O, V> &old) const {
    const Pack<O, V> y = sum.template result<ADD, O>(scale, old);
    if constexpr (LOOSE) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < live)
          out[(int64_t)row * stride + e * step] = y.v[e];
    } else if (active) {
      store<O, V>(out + (int64_t)row * stride, y);
    }
  }
};

// The entries that a group adds up: sorted positions [begin, middle), then
// [tail, end), which go on with the last run of the first part.
struct Walk {
  int64_t begin, middle, tail, end;
  __device__ __forceinline__ int64_t count() const { return middle - begin + end - tail; }
  __device__ __forceinline__ int64_t at(int64_t i) const {
    return i < middle - begin ? begin + i : tail + (i - (middle - begin));
  }
};

// Adds up one after another the rows of a batch of N entries, writing a run's
// row when the next begins.  Where the results are added to, the rows to be
// written are read for the whole batch first.
template <bool WHOLE, int N, typename I, typename O, int V, bool ADD, bool LOOSE, typename A>
__device__ __forceinline__ void add_rows(const Pack<I, V> (&x)[N], const uint32_t (&key)[N], int live,
                                         const GradColumn<O, V, ADD, LOOSE, A> &column, uint32_t &row, Sums<A, V> &sum) {
  Pack<O, V> old[ADD ? N : 1] = {};
  if constexpr (ADD) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const uint32_t before = u > 0 ? key[u > 0 ? u - 1 : 0] : row;
      if ((WHOLE || u < live) && key[u] != before)
        old[u] = column.old(before);
    }
  }
#pragma unroll
  for (int u = 0; u < N; ++u)
    if (WHOLE || u < live) {
      if (key[u] != row) {
        column.write(row, sum, old[ADD ? u : 0]);
        row = key[u];
        sum.clear();
      }
      sum.add(x[u]);
    }
}

// Through registers: the indices of the next batch are read along with the rows
// of this one.  The row and the sum of the last run stay behind.
template <typename I, typename O, int V, bool ADD, bool LOOSE, typename A>
__device__ __forceinline__ void walk_registers(const I *__restrict__ src, int64_t stride, const GradPlan &p,
                                               const Walk &w, const GradColumn<O, V, ADD, LOOSE, A> &column, uint32_t &row,
                                               Sums<A, V> &sum) {
  const int64_t count = w.count();
  int32_t at[kGradBatch] = {};
  uint32_t key[kGradBatch] = {}, next[kGradBatch];
#pragma unroll
  for (int u = 0; u < kGradBatch; ++u)
    if (u < count) {
      at[u] = made(p.order + w.at(u));
      key[u] = made(p.keys + w.at(u));
    }
  for (int64_t i = 0; i < count; i += kGradBatch) {
    Pack<I, V> x[kGradBatch];
#pragma unroll
    for (int u = 0; u < kGradBatch; ++u)
      if (i + u < count)
        x[u] = load<I, V>(src + (int64_t)at[u] * stride);
#pragma unroll
    for (int u = 0; u < kGradBatch; ++u) {
      next[u] = key[u];
      if (i + kGradBatch + u < count) {
        at[u] = made(p.order + w.at(i + kGradBatch + u));
        key[u] = made(p.keys + w.at(i + kGradBatch + u));
      }
    }
    add_rows<false>(x, next, (int)min((int64_t)kGradBatch, count - i), column, row, sum);
  }
}

// By bulk copies: while the threads add up one turn of rows the next is on its
// way.  The first threads fetch a row each.
struct Turns {
  uint64_t bar[2];
  uint32_t key[2][kTurnRows];
  int begin[2][kTurnRows];
};
template <typename I, typename O, int V, bool ADD, bool LOOSE, typename A>
__device__ __forceinline__ bool walk_bulk(const I *__restrict__ src, int64_t stride, const Bounds<I> &bounds,
                                          const GradPlan &p, const Walk &w, int here, unsigned char *memory, Turns &turns,
                                          const GradColumn<O, V, ADD, LOOSE, A> &column, uint32_t &row, Sums<A, V> &sum) {
  const int64_t count = w.count(), last = (count + kTurnRows - 1) / kTurnRows;
  const int r = threadIdx.x, mine = LOOSE ? r : (column.active ? r : 0) * V;
  const int bytes = fetched_bytes<LOOSE, I>(p.slab);
  if (r == 0) {
    nmb::mbar_init(&turns.bar[0], kTurnRows);
    nmb::mbar_init(&turns.bar[1], kTurnRows);
    nmb::mbar_init_fence();
  }
  int32_t at = 0;
  uint32_t key = 0;
  auto look = [&](int64_t turn) { // the entry that this thread fetches in a turn
    const int64_t i = turn * kTurnRows + r;
    if (r < kTurnRows && i < count) {
      at = made(p.order + w.at(i));
      key = made(p.keys + w.at(i));
    }
  };
  auto fetch = [&](int64_t turn) {
    if (r >= kTurnRows)
      return;
    const int b = (int)(turn & 1);
    if (LOOSE && turn > 1)
      nmb::fence_async_smem();
    if (turn * kTurnRows + r < count) {
      turns.key[b][r] = key;
      turns.begin[b][r] = fetch_row<LOOSE>(src + (int64_t)at * stride, here, memory + (b * kTurnRows + r) * bytes,
                                           &turns.bar[b], bounds);
    } else {
      nmb::mbar_arrive(&turns.bar[b]);
    }
  };
  look(0);
  __syncthreads();
  fetch(0);
  look(1);
  if (last > 1)
    fetch(1);
  look(2);
  for (int64_t turn = 0; turn < last; ++turn) {
    const int b = (int)(turn & 1);
    if (!bulk_arrived(&turns.bar[b], (uint32_t)(turn >> 1) & 1, p.waits)) {
      if (turn + 1 < last) // the next turn's copies are on their way, too
        (void)nmb::mbar_wait(&turns.bar[b ^ 1], (uint32_t)((turn + 1) >> 1) & 1);
      return false;
    }
    const int live = (int)min((int64_t)kTurnRows, count - turn * kTurnRows);
    Pack<I, V> x[kTurnRows];
    uint32_t keys[kTurnRows];
    auto take = [&](int u) {
      keys[u] = turns.key[b][u];
      const I *from = reinterpret_cast<const I *>(memory + (b * kTurnRows + u) * bytes) + mine;
      if constexpr (LOOSE) {
        from += turns.begin[b][u];
#pragma unroll
        for (int e = 0; e < V; ++e)
          x[u].v[e] = e < column.live ? from[e * column.step] : I(0.0f);
      } else {
        x[u] = load<I, V>(from);
      }
    };
    if (live == kTurnRows) {
#pragma unroll
      for (int u = 0; u < kTurnRows; ++u)
        take(u);
      add_rows<true>(x, keys, live, column, row, sum);
    } else {
#pragma unroll
      for (int u = 0; u < kTurnRows; ++u)
        if (u < live)
          take(u);
      add_rows<false>(x, keys, live, column, row, sum);
    }
    __syncthreads(); // the turn's memory is free again
    if (turn + 2 < last) {
      fetch(turn + 2);
      look(turn + 3);
    }
  }
  return true;
}

// Sum of `count` partial sums: at `first`, then at second, second + step, ...
template <bool LOOSE, int V, typename A, typename C>
__device__ __forceinline__ void add_partials(const A *partials, int64_t width, int64_t first, int64_t count,
                                             int64_t second, int64_t step, const C &column, Sums<A, V> &sum) {
  sum.clear();
#pragma unroll 4
  for (int64_t i = 0; i < count; ++i) {
    const A *from = partials + (i == 0 ? first : second + (i - 1) * step) * width;
    if constexpr (LOOSE) {
      Pack<A, V> x{};
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < column.live)
          x.v[e] = __ldcg(from + e * column.step);
      sum.add(x);
    } else {
      sum.add(load_l2<A, V>(from));
    }
  }
}

// BULK: the group is the block and V elements are 16 bytes of I; LOOSE: a
// thread's V columns are as many threads apart.
template <typename I, typename O, int V, bool ADD, bool BULK, bool LOOSE>
__global__ void __launch_bounds__(kThreads, BULK ? 4 : 3)
    nmb_take_rows_grad(const I *__restrict__ dout, int64_t stride, const GradPlan p, typename Acc<I>::type scale, O *out,
                       int64_t rows, int64_t out_stride, int64_t cols, const Bounds<I> bounds) {
  using A = typename Acc<I>::type;
  extern __shared__ __align__(128) unsigned char memory[]; // BULK: [2][kTurnRows] rows
  __shared__ uint32_t words[kThreads / 64 + 1];
  __shared__ Turns turns;
  const Group<BULK> group(p.lane_bits);
  nmb::rows::wait_for_previous(); // the sort

  // every `period`-th block takes a chunk as long as there are any: blocks that
  // clear are writes alone, the others mostly wait for reads
  const unsigned turn = blockIdx.x / p.period, work = p.chunk_blocks * p.slabs;
  if (blockIdx.x % p.period != 0 || turn >= work) { // rows without entries
    const int64_t first = (int64_t)(blockIdx.x - min(turn + 1, work)) * kZeroRows;
    if (threadIdx.x < 32) {
      const int64_t v = first + threadIdx.x;
      const int64_t lo = warp_lower_bound(p.keys, 0, p.n, (uint32_t)first);
      const int64_t hi = warp_lower_bound(p.keys, lo, p.n, (uint32_t)min(first + kZeroRows, p.to_clear));
      bool absent = v < p.to_clear;
      if (absent) {
        const int64_t at = lower_bound(p.keys, lo, hi, (uint32_t)v);
        absent = at >= hi || made(p.keys + at) != (uint32_t)v;
      }
      const uint32_t mask = __ballot_sync(kAll, absent);
      if (threadIdx.x == 0)
        words[0] = mask;
    }
    __syncthreads();
    const uint32_t mask = words[0];
    for (int r = group.number; r < kZeroRows; r += (int)blockDim.x / group.lanes)
      if (mask >> r & 1)
        clear_row(out + (first + r) * out_stride, cols, group.lane, group.lanes);
    return;
  }

  const unsigned slab = turn % p.slabs;
  const int64_t chunk = (int64_t)(turn / p.slabs) * (BULK ? 1 : kThreads >> p.lane_bits) + group.number;
  const int64_t slab_first = (int64_t)slab * p.slab;
  const int here = (int)min((int64_t)p.slab, cols - slab_first);
  const bool active = group.lane * (LOOSE ? 1 : V) < here;
  const int64_t col = slab_first + (active ? group.lane * (LOOSE ? 1 : V) : 0); // the thread's first
  const int mine = LOOSE ? (here - group.lane + group.lanes - 1) / group.lanes : 0; // how many, when apart
  const int64_t begin = chunk * p.span;
  if (begin >= p.n)
    return;
  const int64_t end = min(begin + p.span, p.n);
  const uint32_t first_key = made(p.keys + begin), last_key = made(p.keys + end - 1);
  const uint32_t prev_key = begin > 0 ? made(p.keys + begin - 1) : 0xffffffffu;
  const uint32_t next_key = end < p.n ? made(p.keys + end) : 0xffffffffu;
  if (first_key >= rows)
    return;
  const GradColumn<O, V, ADD, LOOSE, A> column{out + col, out_stride, scale, active, active ? mine : 0, group.lanes};

  int64_t owner = chunk, inner = 0; // where a long run began, its inner chunks
  Walk walk{begin, end, end, end};
  if (begin > 0 && prev_key == first_key && last_key == first_key && end - begin == p.span) {
    // inside a long run as a whole
    owner = group.begin_of(p.keys, begin, first_key) / p.span;
    const int64_t stop = next_key == first_key ? group.end_of(p.keys, end, p.n, first_key) : end;
    inner = (stop - (owner + 1) * p.span) / p.span;
  } else {
    // entries of a run that began before belong to the group it began in
    if (prev_key == first_key)
      walk.begin = group.find(p.keys, begin, end, first_key + 1);
    if (last_key >= rows)
      walk.middle = group.find(p.keys, walk.begin, end, (uint32_t)rows);
    if (walk.begin >= walk.middle)
      return;
    if (last_key < rows && next_key == last_key) {
      walk.end = group.end_of(p.keys, end, p.n, last_key);
      inner = (walk.end - end) / p.span;
      walk.tail = end + inner * p.span;
    }
  }
  uint32_t row = made(p.keys + walk.begin);
  Sums<A, V> sum;
  sum.clear();
  if constexpr (BULK) {
    if (!walk_bulk<I, O, V, ADD, LOOSE>(dout + slab_first, stride, bounds, p, walk, here, memory, turns, column, row, sum))
      return;
  } else {
    walk_registers<I, O, V, ADD, LOOSE>(dout + col, stride, p, walk, column, row, sum);
  }
  if (inner == 0) {
    column.write(row, sum, column.old(row));
    return;
  }

  // A long run: leave the partial sum.  The last group of a bundle of chunks
  // adds its bundle's up, the last of those groups the bundles'.
  A *partials = static_cast<A *>(p.partials) + col;
  auto leave_and_draw = [&](int64_t slot, uint32_t *ticket) {
    if constexpr (LOOSE) {
      const Pack<A, V> v = sum.values();
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < column.live)
          partials[slot * cols + e * column.step] = v.v[e];
    } else if (active) {
      store<A, V>(partials + slot * cols, sum.values());
    }
    __threadfence();
    group.sync();
    const uint32_t drawn = group.first(group.lane == 0 ? atomicAdd(ticket + slab, 1u) : 0, words);
    __threadfence();
    return drawn;
  };
  const int64_t last = owner + inner, bundle = chunk / kBundle;
  const int64_t first = max(owner, bundle * kBundle), count = min(last, bundle * kBundle + kBundle - 1) - first + 1;
  const int64_t bundles = last / kBundle - owner / kBundle + 1;
  if (leave_and_draw(chunk, p.tickets + first * p.slabs) != (uint32_t)(count - 1))
    return;
  add_partials<LOOSE>(partials, cols, first, count, first + 1, 1, column, sum);
  if (bundles > 1) {
    if (leave_and_draw(first, p.tickets + (p.chunks + owner) * p.slabs) != (uint32_t)(bundles - 1))
      return;
    add_partials<LOOSE>(partials, cols, owner, bundles, (owner / kBundle + 1) * kBundle, kBundle, column, sum);
  }
  column.write(row, sum, column.old(row));
}

// Entries per chunk: 32, or fewer (down to 4) where that leaves less than two
// blocks a multiprocessor.  With 777 entries of 1000 float32 chunks of 4 give
// 195 blocks, chunks of 32 only 25; 52004 entries of 248 bfloat16 took 29.4 us
// with two, 34.8 us with four (shorter chunks leave more partial sums).
int gradSpan(int64_t n, int64_t vecs) {
  const int bits = laneBits(vecs, kThreadBits);
  const int64_t slabs = (vecs + (int64_t(1) << bits) - 1) >> bits;
  int span = 32;
  while (span > 4 && (n / span >> (kThreadBits - bits)) * slabs < 148 * 2)
    span /= 2;
  return span;
}

// --------------------------------------------------------------- dispatch ---
// Bytes are copied, whatever they mean: U is an unsigned integer of an
// element's size.  A token's row is read once and written k times.
template <typename U, int V>
__global__ void __launch_bounds__(kThreads)
    nmb_dispatch_rows(const U *__restrict__ x, int64_t tokens, int64_t stride, int64_t k,
                      const int32_t *place, const int32_t *kept, U *__restrict__ out,
                      int64_t out_rows, int64_t out_stride, int64_t vecs, int lane_bits) {
  const int lane = threadIdx.x & ((1 << lane_bits) - 1);
  const int64_t t = (int64_t)blockIdx.x * (kThreads >> lane_bits) + (threadIdx.x >> lane_bits);
  nmb::rows::wait_for_previous();
  if (t >= tokens)
    return;
  const int64_t live = made(kept);
  for (int64_t c = lane; c < vecs; c += 1 << lane_bits) {
    const Pack<U, V> row = load<U, V>(x + t * stride + c * V);
#pragma unroll 4
    for (int64_t j = 0; j < k; ++j) {
      const int64_t at = place[t * k + j];
      if (at >= 0 && at < out_rows)
        store<U, V>(out + at * out_stride + c * V, at < live ? row : Pack<U, V>{});
    }
  }
}

// Rows that are not aligned to 16 bytes: a token's row goes into shared memory by
// a bulk copy, and from there element by element to its places.
constexpr int kCopyThreads = 128, kCopyBytes = 8192;
template <typename U>
__global__ void __launch_bounds__(kCopyThreads)
    nmb_dispatch_rows_bulk(const U *__restrict__ x, int64_t stride, int64_t k, const int32_t *place,
                           const int32_t *kept, U *__restrict__ out, int64_t out_rows, int64_t out_stride,
                           int64_t cols, int slab, const Bounds<U> bounds, const Waits waits) {
  extern __shared__ __align__(128) unsigned char memory[];
  __shared__ uint64_t bar;
  __shared__ int begin;
  const int64_t t = blockIdx.x, first = (int64_t)blockIdx.y * slab;
  const int here = (int)min((int64_t)slab, cols - first);
  nmb::rows::wait_for_previous();
  if (threadIdx.x == 0) {
    nmb::mbar_init(&bar, 1);
    nmb::mbar_init_fence();
    begin = fetch_row<true>(x + t * stride + first, here, memory, &bar, bounds);
  }
  __syncthreads();
  const int64_t live = made(kept);
  if (!bulk_arrived(&bar, 0, waits))
    return;
  const U *row = reinterpret_cast<const U *>(memory) + begin;
  for (int64_t j = 0; j < k; ++j) {
    const int64_t at = place[t * k + j];
    if (at < 0 || at >= out_rows)
      continue;
    U *to = out + at * out_stride + first;
#pragma unroll 4
    for (int col = threadIdx.x; col < here; col += kCopyThreads)
      to[col] = at < live ? row[col] : U(0);
  }
}

// Sort and copy in one launch for few entries.  A block takes a token, and a
// warp finds the place of one of its choices by counting: the entries of smaller
// keys and the earlier ones of the same key.  That is `entries` comparisons per
// entry, but no step waits for another block.  Rows of 2048 bfloat16, 8 of 64
// experts: 3.0 us for 4 tokens (4.6 us in two launches), 3.3 us for 128 (7.1),
// 10.0 us for 512 (12.5).  All blocks together look at tokens x entries ids, so
// tokens of few choices end it earlier.  In two launches against one, rows of 64
// and of 2048 bfloat16: 2048 tokens of one choice 6.5 and 10.5 against 6.6 and
// 7.6 us, 1024 of four 9.1 and 12.2 against 9.6 and 10.9 (both within the limit);
// 2048 of two 8.4 and 13.4 against 12.6 and 14.3, 4096 of one 8.4 and 16.7 against
// 19.2 and 21.6 (both past it, in one launch with room for more choices a block).  A block finds its token's choices by its eight
// warps, which ends it at 64 of them: one token of 64 of 1024 experts, rows of 64,
// 8.3 us against 9.7 in two launches, of 128 33.5 against 15.3, of 1024 146
// against 92.
constexpr int kCountEntries = 4096, kCountGroups = 1024, kCountChoices = 64;
constexpr int64_t kCountWork = int64_t(1) << 22; // tokens x entries

template <typename U, int V>
__global__ void __launch_bounds__(kThreads)
    nmb_sort_dispatch_rows(const U *__restrict__ x, int64_t stride, int k, const void *__restrict__ ids, int id_bytes,
                           int entries, int groups, int32_t *__restrict__ order, int32_t *__restrict__ place,
                           int32_t *__restrict__ offsets, U *__restrict__ out, int64_t out_stride, int64_t vecs) {
  __shared__ uint32_t keys[kCountEntries];
  __shared__ int32_t to[kCountChoices];
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kWarps = kThreads / 32;
  for (int i = threadIdx.x; i < entries; i += kThreads) {
    const int64_t id = index_at(ids, id_bytes, i);
    keys[i] = id >= 0 && id < groups ? (uint32_t)id : (uint32_t)groups;
  }
  __syncthreads();
  for (int j = warp; j < k; j += kWarps) {
    const int e = t * k + j;
    const uint32_t key = keys[e];
    int before = 0;
    for (int i = lane; i < entries; i += 32)
      before += keys[i] < key || (keys[i] == key && i < e);
    before = __reduce_add_sync(kAll, before);
    if (lane == 0) {
      to[j] = key < (uint32_t)groups ? before : ~before; // a dropped choice: the place of a zero row
      place[e] = before;
      order[before] = e;
    }
  }
  if (entries <= 64) {
    // few tokens may come with many groups: a thread per group
    for (int g = t * kThreads + (int)threadIdx.x; g <= groups; g += (int)gridDim.x * kThreads) {
      int before = 0;
      for (int i = 0; i < entries; ++i)
        before += keys[i] < (uint32_t)g;
      offsets[g] = before;
    }
  } else {
    for (int g = t * kWarps + warp; g <= groups; g += (int)gridDim.x * kWarps) {
      int before = 0;
      for (int i = lane; i < entries; i += 32)
        before += keys[i] < (uint32_t)g;
      before = __reduce_add_sync(kAll, before);
      if (lane == 0)
        offsets[g] = before;
    }
  }
  __syncthreads();
  for (int64_t c = threadIdx.x; c < vecs; c += kThreads) {
    const Pack<U, V> row = load<U, V>(x + (int64_t)t * stride + c * V);
#pragma unroll 4
    for (int j = 0; j < k; ++j) {
      const int at = to[j];
      store<U, V>(out + (int64_t)(at < 0 ? ~at : at) * out_stride + c * V, at < 0 ? Pack<U, V>{} : row);
    }
  }
}

// ---------------------------------------------------------------- combine ---
template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
    nmb_combine_rows(const T *__restrict__ ys, int64_t y_rows, int64_t stride, int64_t k,
                     const int32_t *__restrict__ place, const int32_t *__restrict__ kept, const void *weights,
                     int weight_type, T *__restrict__ out, int64_t tokens, int64_t out_stride, int64_t vecs,
                     int lane_bits) {
  using A = typename Acc<T>::type;
  const int lane = threadIdx.x & ((1 << lane_bits) - 1);
  const int64_t t = (int64_t)blockIdx.x * (kThreads >> lane_bits) + (threadIdx.x >> lane_bits);
  if (t >= tokens)
    return;
  const int64_t live = min((int64_t)*kept, y_rows);
  for (int64_t c = lane; c < vecs; c += 1 << lane_bits) {
    A sum[V] = {};
#pragma unroll 4
    for (int64_t j = 0; j < k; ++j) {
      const int64_t at = place[t * k + j];
      if (at >= 0 && at < live) {
        const Pack<T, V> y = load<T, V>(ys + at * stride + c * V);
        const A w = weights ? scalar_at<A>(weights, weight_type, t * k + j) : A(1);
#pragma unroll
        for (int e = 0; e < V; ++e)
          sum[e] = madd(w, up(y.v[e]), sum[e]);
      }
    }
    Pack<T, V> r;
#pragma unroll
    for (int e = 0; e < V; ++e)
      r.v[e] = down<T, A>(sum[e]);
    store<T, V>(out + t * out_stride + c * V, r);
  }
}

// The same with the rows fetched by bulk copies: a block takes a token, a few of
// narrow rows or a slab of its columns, brings the rows of all their choices into
// shared memory at once and adds them up from there.  Copies in flight cost no registers: with
// the rows in registers eight choices left room for one block a multiprocessor,
// and batches of four reached 4.5 of the 6.5 TB/s that a copy reaches.
constexpr int kBulkThreads = 128;
constexpr int kBulkBits = 7;
constexpr int kBulkChoices = 32;        // most choices of a token
// Most bytes in flight per block.  combine: 16384 tokens with eight rows of 4 KB
// took 92.1 us at 16 KB (two slabs a token), 95.8 us at 32 KB.  combine_grad: a
// token with eight such rows 173.5 us in one turn of 36 KB or in two of half of
// it; 30000 tokens with two rows of 2 KB, which share blocks where they fit,
// 49.8 us at 45 KB, 56.3 us at half.
constexpr int kBulkBytes = 16384, kBulkGradBytes = 46080;

// What the threads of a block share about a token's choices.
template <typename A> struct BulkChoices {
  uint64_t bar;
  int32_t at[kBulkChoices]; // where the row begins in shared memory, or where it goes; -1: left out
  A weight[kBulkChoices];
};

template <typename T, bool LOOSE>
__global__ void __launch_bounds__(kBulkThreads)
    nmb_combine_rows_bulk(const T *__restrict__ ys, int64_t y_rows, int64_t stride, int k,
                          const int32_t *__restrict__ place, const int32_t *__restrict__ kept,
                          const void *__restrict__ weights, int weight_type, T *__restrict__ out, int64_t tokens,
                          int64_t out_stride, int64_t cols, int slab, int each_bits, const Bounds<T> bounds,
                          const Waits waits) {
  using A = typename Acc<T>::type;
  constexpr int V = kBulkElems<LOOSE, T>;
  extern __shared__ __align__(128) unsigned char rows[]; // [1 << each_bits][k] rows
  __shared__ BulkChoices<A> c;
  const int64_t t0 = (int64_t)blockIdx.x << each_bits, first = (int64_t)blockIdx.y * slab;
  const int here = (int)min((int64_t)slab, cols - first), bytes = fetched_bytes<LOOSE, T>(slab);
  const int entries = k * (int)min((int64_t)1 << each_bits, tokens - t0);
  const int j = threadIdx.x;
  int32_t at = -1;
  if (j < entries) {
    at = __ldg(place + t0 * k + j);
    at = at < min((int64_t)__ldg(kept), y_rows) ? at : -1;
    c.weight[j] = weights ? scalar_at<A>(weights, weight_type, t0 * k + j) : A(1);
  }
  if (j == 0) {
    nmb::mbar_init(&c.bar, (uint32_t)entries);
    nmb::mbar_init_fence();
  }
  __syncthreads();
  if (j < entries) {
    c.at[j] = -1;
    if (at >= 0)
      c.at[j] = j * bytes + (int)sizeof(T) * fetch_row<LOOSE>(ys + at * stride + first, here, rows + j * bytes, &c.bar,
                                                              bounds);
    else
      nmb::mbar_arrive(&c.bar);
  }
  if (!bulk_arrived(&c.bar, 0, waits))
    return;
  const int bits = kBulkBits - each_bits, threads = 1 << bits, token = j >> bits; // a token's threads
  if (t0 + token >= tokens)
    return;
  const int32_t *begin = c.at + token * k;
  const A *weight = c.weight + token * k;
  T *dst = out + (t0 + token) * out_stride + first;
  for (int col = (j & (threads - 1)) * V; col < here; col += threads * V) {
    A sum[V] = {};
#pragma unroll 4
    for (int i = 0; i < k; ++i)
      if (begin[i] >= 0) {
        const Pack<T, V> y = load<T, V>(reinterpret_cast<const T *>(rows + begin[i]) + col);
#pragma unroll
        for (int e = 0; e < V; ++e)
          sum[e] = madd(weight[i], up(y.v[e]), sum[e]);
      }
    Pack<T, V> r;
#pragma unroll
    for (int e = 0; e < V; ++e)
      r.v[e] = down<T, A>(sum[e]);
    store<T, V>(dst + col, r);
  }
}

// Elements of a slab where `rows` rows share `most` bytes: equal shares of the
// row in as few slabs as that allows.  0: not by bulk copies (too many choices, or
// rows so narrow that the registers' kernels are as fast).  30000 tokens, combine
// and its gradient, registers against bulk: two rows of 512 bytes 9.4 and 17.6
// against 10.9 and 21.7 us, of 768 bytes 17.4 and 49.3 (by four) against 13.9 and
// 29.1; eight rows of 256 bytes 12.6 and 32.8 against 18.2 and 68.4, of 512 bytes
// 36.1 and 58.6 against 28.8 and 52.4.  Off the words, where the registers take an
// element at a time: two rows of 31 bf16 6.7 and 15.3 against 9.7 and 17.9, of 47
// 11.0 and 30.1 against 10.7 and 19.2, of 259 42.5 and 122.2 against 18.1 and 29.6.
int bulkSlab(int64_t cols, int type, bool loose, int64_t choices, int rows, int most) {
  const int size = elemBytes(type), step = loose ? 1 : 16 / size;
  if (choices < 1 || choices > kBulkChoices || (loose ? cols < 48 : cols * size < (choices <= 2 ? 768 : 512)))
    return 0;
  const int64_t room = most / rows - (loose ? 32 : 0); // bytes of a row
  const int64_t slabs = (cols * size + room - 1) / room;
  const int64_t slab = ((cols + slabs - 1) / slabs + step - 1) / step * step;
  return slabs <= 65535 ? (int)slab : 0;
}

// Tokens of a block (their log2) where their rows are so narrow that a block of
// one token is mostly its own beginning: up to four, as long as `most` bytes and
// the choices hold them and four blocks a multiprocessor are left.  30000 tokens
// with two rows of 1 KB: 15.6 us by four, 29.2 us by one.
int bulkTokens(int64_t tokens, int64_t bytesEach, int64_t choices, int most) {
  int bits = 2;
  while (bits > 0 && (bytesEach << bits > most || choices << bits > kBulkChoices || tokens >> bits < 148 * 4))
    --bits;
  return bits;
}

// ----------------------------------------------------------- combine_grad ---
// The threads of a token read dout once for up to N choices, whose rows are
// in flight together; each keeps its share of their dot products, which meet at
// the end in a fixed tree: shuffles that halve the values along with the lanes,
// then the token's warps in order.
//
// Two at a time for tokens of one or two choices, whose threads then hold half
// as much and leave room for more blocks: 30000 tokens with two rows of 512
// bytes 24.5 us by four, 17.6 us by two; with eight such rows 58.6 us by four,
// 62.1 us by two.
template <int N, typename A> struct Choices {
  int32_t at[N];
  A weight[N];
  __device__ __forceinline__ void read(const int32_t *__restrict__ place, const void *__restrict__ weights,
                                       int weight_type, int64_t entry, int64_t left) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      at[j] = j < left ? __ldg(place + entry + j) : -1;
      weight[j] = weights && j < left ? scalar_at<A>(weights, weight_type, entry + j) : A(1);
    }
  }
};

// Adds N values up over the lanes of a token (up to a warp).  The first log2(N)
// steps also halve the values a lane is left with: lane bit b picks bit
// log2(N) - 1 - b of the value.
template <int N, typename A> __device__ __forceinline__ void meet(A (&v)[N], int lanes) {
  const int lane = threadIdx.x & 31;
  int held = N;
#pragma unroll
  for (int step = 1; step <= 16; step <<= 1) {
    if (step >= lanes)
      break;
    if (held > 1) {
      held /= 2;
      const bool high = lane & step;
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        if (i < held) {
          const A give = high ? v[i] : v[i + held], keep = high ? v[i + held] : v[i];
          v[i] = keep + __shfl_xor_sync(kAll, give, step);
        }
    } else {
      v[0] += __shfl_xor_sync(kAll, v[0], step);
    }
  }
}

template <typename T, int V, int N>
__global__ void __launch_bounds__(kThreads, 4)
    nmb_combine_rows_grad(const T *__restrict__ dout, int64_t tokens, int64_t stride, const T *__restrict__ ys,
                          int64_t y_rows, int64_t y_stride, int64_t k, const int32_t *__restrict__ place,
                          const int32_t *__restrict__ kept, const void *__restrict__ weights, int weight_type,
                          T *__restrict__ dys, int64_t dy_rows, int64_t dy_stride, void *dweights, int64_t vecs,
                          int lane_bits) {
  static_assert(N == 2 || N == 4, "the lanes' halvings are written for these");
  constexpr int kBits = N / 2;
  using A = typename Acc<T>::type;
  __shared__ A parts[kThreads / 32][N];
  const int lanes = 1 << lane_bits;
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t t = (int64_t)blockIdx.x * (kThreads >> lane_bits) + (threadIdx.x >> lane_bits);
  const bool token = t < tokens; // every thread stays for the shuffles and barriers
  const int64_t live = min((int64_t)__ldg(kept), y_rows);
  Choices<N, A> c;
  for (int64_t j0 = 0; j0 < k; j0 += N) {
    c.read(place, weights, weight_type, t * k + j0, token ? k - j0 : 0);
    A dot[N] = {};
    for (int64_t col = token ? lane : vecs; col < vecs; col += lanes) {
      const Pack<T, V> d = load<T, V>(dout + t * stride + col * V);
      Pack<T, V> y[N];
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (c.at[j] >= 0 && c.at[j] < live)
          y[j] = load<T, V>(ys + c.at[j] * y_stride + col * V);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (c.at[j] >= 0 && c.at[j] < dy_rows) {
          Pack<T, V> r{};
          if (c.at[j] < live) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              dot[j] = madd(up(d.v[e]), up(y[j].v[e]), dot[j]);
              r.v[e] = down<T, A>(c.weight[j] * up(d.v[e]));
            }
          }
          store<T, V>(dys + c.at[j] * dy_stride + col * V, r);
        }
    }
    meet(dot, lanes);
    const int halvings = lane_bits < kBits ? lane_bits : kBits;
    int mine = 0; // the first of the values that this lane ends up with
    for (int b = 0; b < halvings; ++b)
      mine |= (lane >> b & 1) << (kBits - 1 - b);
    const int held = N >> halvings;
    if (lanes > 32) {
      const int warp = threadIdx.x >> 5;
      if ((threadIdx.x & 31) < N)
        parts[warp][mine] = dot[0];
      __syncthreads();
      if (lane < N) {
        A sum = A(0);
        for (int w = 0; w < lanes / 32; ++w)
          sum += parts[warp + w][lane];
        if (token && j0 + lane < k && dweights)
          set_scalar<A>(dweights, weight_type, t * k + j0 + lane, sum);
      }
      __syncthreads();
    } else if (token && lane < (1 << halvings) && dweights) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < held && j0 + mine + i < k)
          set_scalar<A>(dweights, weight_type, t * k + j0 + mine + i, dot[i]);
    }
  }
}

// The same with the rows fetched by bulk copies, dout's first.  A block takes
// whole tokens; columns beyond a slab come in turns through the same memory.
template <typename T, bool LOOSE>
__global__ void __launch_bounds__(kBulkThreads)
    nmb_combine_rows_grad_bulk(const T *__restrict__ dout, int64_t tokens, int64_t stride,
                               const T *__restrict__ ys, int64_t y_rows, int64_t y_stride, int k,
                               const int32_t *__restrict__ place, const int32_t *__restrict__ kept, const void *__restrict__ weights, int weight_type,
                               T *__restrict__ dys, int64_t dy_rows, int64_t dy_stride, void *dweights, int64_t cols,
                               int slab, int each_bits, const Bounds<T> dbounds, const Bounds<T> ybounds,
                               const Waits waits) {
  using A = typename Acc<T>::type;
  constexpr int V = kBulkElems<LOOSE, T>, kWarps = kBulkThreads / 32, kPairs = V > 1 ? V / 2 : 1;
  // Choices read against dout at a time: what more of them hold in registers is
  // blocks less on the way.  30000 tokens with eight rows of 1.5 KB took 149 us by
  // two, 162 us by four, 236 us by eight.
  constexpr int kTogether = 2;
  extern __shared__ __align__(128) unsigned char rows[]; // [1 << each_bits][1 + k] rows, dout's first
  __shared__ BulkChoices<A> c;
  __shared__ int begin[2 * kBulkChoices]; // where each row's first element is
  __shared__ A parts[kWarps][kBulkChoices];
  const int64_t t0 = (int64_t)blockIdx.x << each_bits;
  const int j = threadIdx.x, lane = j & 31, warp = j >> 5, bytes = fetched_bytes<LOOSE, T>(slab);
  const int here_tokens = (int)min((int64_t)1 << each_bits, tokens - t0), entries = here_tokens * k;
  const int bits = kBulkBits - each_bits, threads = 1 << bits; // a token's threads
  const int token = j >> bits, mine = j & (threads - 1);
  const int64_t live = min((int64_t)__ldg(kept), y_rows);
  // thread j fetches dout's row of a token or that of a choice
  const int fetches = here_tokens * (k + 1), ftoken = j / (k + 1), fchoice = j - ftoken * (k + 1) - 1;
  int32_t at = -1;
  if (j < fetches && fchoice >= 0) {
    const int e = ftoken * k + fchoice;
    at = __ldg(place + t0 * k + e);
    c.at[e] = at < dy_rows ? at : -1;
    c.weight[e] = weights ? scalar_at<A>(weights, weight_type, t0 * k + e) : A(1);
  }
  if (j == 0) {
    nmb::mbar_init(&c.bar, (uint32_t)fetches);
    nmb::mbar_init_fence();
  }
  for (int i = j; i < kWarps * kBulkChoices; i += kBulkThreads)
    (&parts[0][0])[i] = A(0);
  __syncthreads();
  uint32_t phase = 0;
  for (int64_t first = 0; first < cols; first += slab, phase ^= 1) {
    const int here = (int)min((int64_t)slab, cols - first);
    if (j < fetches) {
      unsigned char *to = rows + j * bytes;
      if (LOOSE && first > 0)
        nmb::fence_async_smem();
      if (fchoice < 0)
        begin[j] = fetch_row<LOOSE>(dout + (t0 + ftoken) * stride + first, here, to, &c.bar, dbounds);
      else if (at >= 0 && at < live)
        begin[j] = fetch_row<LOOSE>(ys + at * y_stride + first, here, to, &c.bar, ybounds);
      else
        nmb::mbar_arrive(&c.bar);
    }
    if (!bulk_arrived(&c.bar, phase, waits))
      return;
    const int row0 = token * (k + 1), entry0 = token * k;
    const T *drow = reinterpret_cast<const T *>(rows + row0 * bytes) + (LOOSE ? begin[row0] : 0);
    for (int j0 = 0; j0 < k && token < here_tokens; j0 += kTogether) {
      int32_t to[kTogether];
      A w[kTogether];
      const T *yrow[kTogether];
      typename Two<A>::type dots[kTogether] = {};
#pragma unroll
      for (int i = 0; i < kTogether; ++i) {
        to[i] = j0 + i < k ? c.at[entry0 + j0 + i] : -1;
        w[i] = j0 + i < k ? c.weight[entry0 + j0 + i] : A(0);
        yrow[i] = reinterpret_cast<const T *>(rows + (row0 + j0 + i + 1) * bytes);
        if (LOOSE && to[i] >= 0 && to[i] < live)
          yrow[i] += begin[row0 + j0 + i + 1];
      }
      for (int col = mine * V; col < here; col += threads * V) {
        const Pack<T, V> x = load<T, V>(drow + col);
        typename Two<A>::type d[kPairs];
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          if constexpr (V > 1)
            d[e] = up2(x.v + 2 * e);
          else
            d[e].x = up(x.v[0]);
        }
#pragma unroll
        for (int i = 0; i < kTogether; ++i)
          if (to[i] >= 0) {
            Pack<T, V> r{};
            if (to[i] < live) {
              const Pack<T, V> y = load<T, V>(yrow[i] + col);
              if constexpr (V > 1) {
#pragma unroll
                for (int e = 0; e < kPairs; ++e) {
                  dots[i] = madd2(d[e], up2(y.v + 2 * e), dots[i]);
                  down2(r.v + 2 * e, mul2(w[i], d[e]));
                }
              } else {
                dots[i].x = madd(d[0].x, up(y.v[0]), dots[i].x);
                r.v[0] = down<T, A>(w[i] * d[0].x);
              }
            }
            store<T, V>(dys + to[i] * dy_stride + first + col, r);
          }
      }
      A dot[kTogether];
#pragma unroll
      for (int i = 0; i < kTogether; ++i)
        dot[i] = dots[i].x + dots[i].y;
      meet(dot, 32);
      if (lane < kTogether && j0 + lane < k) // see meet
        parts[warp][j0 + lane] += dot[0];
    }
    __syncthreads(); // the slab's memory is free again, the sums are in place
  }
  if (j < entries && dweights) {
    // a token's warps in order
    const int of = j / k, warps = kWarps >> each_bits;
    A sum = A(0);
    for (int w = 0; w < warps; ++w)
      sum += parts[of * warps + w][j - of * k];
    set_scalar<A>(dweights, weight_type, t0 * k + j, sum);
  }
}

// ------------------------------------------------------------------- host ---
std::atomic<uint32_t> gSpins{nmb::kWaitSpins};

// `status` null: no word, with the error set.
Waits waitsOf(void *queue) { return {nmb::statusWord(queue), gSpins.load(std::memory_order_relaxed)}; }

unsigned blocksFor(int64_t rows, int lane_bits) {
  const int64_t per = kThreads >> lane_bits;
  return (unsigned)((rows + per - 1) / per);
}
// grids are one-dimensional
bool gridFits(const char *who, int64_t rows) {
  if (rows < (int64_t(1) << 31))
    return true;
  nmb::setError("%s: 2^31 rows or more", who);
  return false;
}

template <typename T> constexpr int mostElems() { return 16 / (int)sizeof(T); }

// Calls f(V constant) for the access width v.
template <int MOST, typename F> void withElems(int v, F &&f) {
  if constexpr (MOST >= 8)
    if (v == 8)
      return f(std::integral_constant<int, 8>());
  if constexpr (MOST >= 4)
    if (v == 4)
      return f(std::integral_constant<int, 4>());
  if constexpr (MOST >= 2)
    if (v == 2)
      return f(std::integral_constant<int, 2>());
  f(std::integral_constant<int, 1>());
}

// The memory that rows lie in.
template <typename T> Bounds<T> boundsOf(const GPUXRows *r) {
  const T *data = static_cast<const T *>(r->data);
  const int64_t far = r->rows > 1 ? (r->rows - 1) * r->stride : 0;
  return {data + (far < 0 ? far : 0), data + (far > 0 ? far : 0) + r->cols};
}

template <typename F> void withType(int type, F &&f) {
  if (type == GPUX_ELEM_F32)
    f(float());
  else if (type == GPUX_ELEM_F64)
    f(double());
  else if (type == GPUX_ELEM_F16)
    f(__half());
  else
    f(__nv_bfloat16());
}

// The pairs of types of take and take_grad: equal, or float32 and a 16-bit type.
bool pairAllowed(const char *who, int a, int b) {
  const bool wide = a == GPUX_ELEM_F32 || b == GPUX_ELEM_F32;
  if (a == b || (wide && a != GPUX_ELEM_F64 && b != GPUX_ELEM_F64))
    return true;
  nmb::setError("%s: the result has the operand's type, or one is float32 and the other 16 bits wide", who);
  return false;
}
template <typename F> void withPair(int a, int b, F &&f) {
  withType(a, [&](auto x) {
    using X = decltype(x);
    if (a == b)
      return f(x, x);
    if constexpr (std::is_same_v<X, float>) {
      if (b == GPUX_ELEM_F16)
        f(x, __half());
      else
        f(x, __nv_bfloat16());
    } else if constexpr (sizeof(X) == 2) {
      f(x, float());
    }
  });
}

bool sameWidth(const char *who, const GPUXRows *a, const GPUXRows *b) {
  if (a->cols == b->cols)
    return true;
  nmb::setError("%s: rows of %lld and %lld elements", who, (long long)a->cols, (long long)b->cols);
  return false;
}
bool sameType(const char *who, const GPUXRows *a, const GPUXRows *b) {
  if (a->type == b->type)
    return true;
  nmb::setError("%s: the rows have different types", who);
  return false;
}
bool checkPlaces(const char *who, int64_t tokens, int64_t k, const int32_t *place, const int32_t *kept) {
  if (k < 0 || (k > 0 && tokens > ((int64_t(1) << 31) - 1) / k)) {
    nmb::setError("%s: the number of entries must be below 2^31", who);
    return false;
  }
  if ((tokens * k > 0 && !place) || !kept) {
    nmb::setError("%s: null positions", who);
    return false;
  }
  return true;
}
bool checkWeights(const char *who, const void *weights, int type) {
  if (!weights)
    return true;
  if (type < GPUX_ELEM_F32 || type > GPUX_ELEM_BF16 ||
      reinterpret_cast<uintptr_t>(weights) % (uintptr_t)elemBytes(type) != 0) {
    nmb::setError("%s: the weights have an unknown type or are not aligned", who);
    return false;
  }
  return true;
}

size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }

} // namespace

// Test hook: polls after which the row operators' kernels give up waiting for
// their own copies (which are then waited for all the same); 0: at once.
GPUX_EXPORT void gpuxTestRowWaitSpins(uint32_t spins) { gSpins = spins < nmb::kWaitSpins ? spins : nmb::kWaitSpins; }

GPUX_EXPORT int _mlir_ciface_nmb_take_rows_device(void *queue, const GPUXRows *table, const GPUXIndex *ids,
                                                  double scale, const GPUXRows *out) {
  const char *who = "take_rows";
  if (!checkRows(who, "table", table, false) || !checkIndex(who, ids) || !checkRows(who, "out", out, true) ||
      !pairAllowed(who, table->type, out->type) || !sameWidth(who, table, out))
    return 1;
  if (out->rows != ids->count) {
    nmb::setError("%s: %lld rows for %lld indices", who, (long long)out->rows, (long long)ids->count);
    return 1;
  }
  if (out->rows == 0 || out->cols == 0)
    return 0;
  Stream s(queue);
  if (!s.ok)
    return 1;
  const Waits waits = waitsOf(queue);
  if (!waits.status)
    return 1;
  withPair(table->type, out->type, [&](auto i, auto o) {
    using I = decltype(i);
    using O = decltype(o);
    constexpr int most = mostElems<I>() > mostElems<O>() ? mostElems<I>() : mostElems<O>();
    const int v = accessElems(out->cols, most, {table, out});
    const int64_t vecs = out->cols / v;
    const int64_t row_bytes = out->cols * (int64_t)sizeof(I);
    const bool loose = v < mostElems<I>();
    if (row_bytes >= kBulkLeast && out->rows * row_bytes >= (loose ? kTakeLooseLeast : kTakeBulkLeast)) {
      // equal slabs of a row that does not fit, several rows that do
      const int64_t step = loose ? 1 : mostElems<I>(), slabs = (row_bytes + kTakeBytes - 1) / kTakeBytes;
      const int slab = (int)(((out->cols + slabs - 1) / slabs + step - 1) / step * step);
      const int bytes = loose ? fetched_bytes<true, I>(slab) : fetched_bytes<false, I>(slab);
      const int fit = kTakeBytes / bytes, each = fit < 1 ? 1 : fit < kTakeRows ? fit : kTakeRows;
      if (slabs <= 65535) {
        const auto kernel = loose ? nmb_take_rows_bulk<I, O, true> : nmb_take_rows_bulk<I, O, false>;
        kernel<<<dim3((unsigned)((out->rows + each - 1) / each), (unsigned)slabs), kTakeThreads, (size_t)each * bytes,
                 s.stream>>>(static_cast<const I *>(table->data), table->rows, table->stride, ids->data, ids->bytes,
                             ids->count, (typename Acc<I>::type)scale, static_cast<O *>(out->data), out->stride,
                             out->cols, slab, each, boundsOf<I>(table), waits);
        return;
      }
    }
    const int bits = takeLaneBits(out->rows, vecs);
    withElems<most>(v, [&](auto V) {
      nmb_take_rows<I, O, V.value><<<blocksFor(out->rows, bits), kThreads, 0, s.stream>>>(
          static_cast<const I *>(table->data), table->rows, table->stride, ids->data, ids->bytes, ids->count,
          (typename Acc<I>::type)scale, static_cast<O *>(out->data), out->stride, vecs, bits);
    });
  });
  return launched(who) ? 0 : 1;
}

namespace {
// The workspace of take_grad: order, sorted keys, tickets, partial sums, the
// sort's own.  It depends on the shape alone: the widest access (8 elements)
// gives the shortest chunks, the narrowest the most slabs.
struct GradMemory {
  size_t entries, tickets, partials, sort;
  GradMemory(int64_t n, int64_t rows, int64_t cols, int type) {
    const int span = gradSpan(n, (cols + 7) / 8);
    const int64_t chunks = (n + span - 1) / span;
    entries = padded((size_t)n * 4);
    tickets = padded((size_t)chunks * 2 * (size_t)((cols + kThreads - 1) / kThreads) * 4);
    partials = padded((size_t)chunks * (size_t)cols * (type == GPUX_ELEM_F64 ? 8 : 4));
    sort = nmb::rows::sortBytes(n, rows);
  }
  size_t total() const { return 2 * entries + tickets + partials + sort; }
};
} // namespace

GPUX_EXPORT size_t _mlir_ciface_nmb_take_rows_grad_workspace(int64_t count, int64_t rows, int64_t cols, int type) {
  const int64_t most = 0x7fffffff; // what the entry takes
  return count < 0 || count > most || rows < 0 || rows >= most || cols < 0 || cols > most
             ? 0
             : GradMemory(count, rows, cols, type).total();
}

GPUX_EXPORT int _mlir_ciface_nmb_take_rows_grad_device(void *queue, const GPUXRows *dout, const GPUXIndex *ids,
                                                       double scale, const GPUXRows *out, int accumulate,
                                                       void *workspace, size_t workspaceBytes) {
  const char *who = "take_rows_grad";
  if (!checkRows(who, "dout", dout, false) || !checkIndex(who, ids) || !checkRows(who, "out", out, true) ||
      !pairAllowed(who, dout->type, out->type) || !sameWidth(who, dout, out) || !gridFits(who, out->rows))
    return 1;
  if (dout->rows != ids->count || out->rows >= 0x7fffffff) {
    nmb::setError("%s: %lld rows for %lld indices, %lld rows of the table", who, (long long)dout->rows,
                  (long long)ids->count, (long long)out->rows);
    return 1;
  }
  if (out->rows == 0 || out->cols == 0 || (accumulate && ids->count == 0))
    return 0;
  Stream s(queue);
  if (!s.ok)
    return 1;
  const GradMemory need(ids->count, out->rows, out->cols, dout->type);
  nmb::rows::Workspace memory(s, who, workspace, workspaceBytes, need.total());
  if (!memory.ok)
    return 1;
  const Waits waits = waitsOf(queue);
  if (!waits.status)
    return 1;
  unsigned char *ws = static_cast<unsigned char *>(memory.data);
  int32_t *order = reinterpret_cast<int32_t *>(ws);
  uint32_t *keys = reinterpret_cast<uint32_t *>(ws + need.entries);
  uint32_t *tickets = reinterpret_cast<uint32_t *>(ws + 2 * need.entries);
  void *partials = ws + 2 * need.entries + need.tickets;
  bool ok = true;
  withPair(dout->type, out->type, [&](auto i, auto o) {
    using I = decltype(i);
    using O = decltype(o);
    constexpr int wide = mostElems<I>();
    const int v = accessElems(out->cols, wide, {dout, out});
    const bool bulk = out->cols * (int64_t)sizeof(I) >= kBulkLeast, loose = bulk && v < wide;
    const int64_t vecs = bulk ? (out->cols + wide - 1) / wide : out->cols / v;
    const int bits = laneBits(vecs, kThreadBits);
    const int span = gradSpan(ids->count, vecs);
    const int64_t chunks = (ids->count + span - 1) / span;
    const unsigned slabs = (unsigned)((vecs + (int64_t(1) << bits) - 1) >> bits);
    const int slab = (int)((vecs + slabs - 1) / slabs) * (bulk ? wide : v);
    const unsigned chunkBlocks = bulk ? (unsigned)chunks : blocksFor(chunks, bits);
    const int64_t work = (int64_t)chunkBlocks * slabs;
    if (work + (out->rows + kZeroRows - 1) / kZeroRows >= (int64_t(1) << 31)) {
      nmb::setError("%s: too many indices for their width", who);
      ok = false;
      return;
    }
    nmb::rows::Clearing clearing;
    clearing.data = static_cast<unsigned char *>(out->data);
    clearing.left = accumulate ? 0 : out->rows;
    clearing.rowBytes = out->cols * (int64_t)sizeof(O);
    clearing.stride = out->stride * (int64_t)sizeof(O);
    const int alone = accessElems(out->cols, mostElems<O>(), {out}); // elements per access of the result by itself
    clearing.unit = alone * (int)sizeof(O) < 16 ? alone * (int)sizeof(O) : 16;
    ok = nmb::rows::sortByKey(s, who, *ids, out->rows, order, keys, nullptr, nullptr,
                              ws + 2 * need.entries + need.tickets + need.partials, tickets, 2 * chunks * slabs,
                              &clearing);
    if (!ok)
      return;
    const int64_t blocks = work + (clearing.left + kZeroRows - 1) / kZeroRows;
    if (blocks == 0)
      return;
    const GradPlan plan{order,
                        keys,
                        ids->count,
                        span,
                        slabs,
                        slab,
                        chunkBlocks,
                        work > 0 ? (unsigned)(blocks / work) : 1,
                        partials,
                        tickets,
                        chunks,
                        clearing.left,
                        bits,
                        waits};
    // without entries there is no sort in front, and the kernel begins like any other
    const bool behind = ids->count > 0;
    auto go = [&](auto kernel, int threads, size_t shared) {
      nmb::rows::launchBehind(kernel, (unsigned)blocks, (unsigned)threads, shared, s.stream, behind,
                              static_cast<const I *>(dout->data), dout->stride, plan, (typename Acc<I>::type)scale,
                              static_cast<O *>(out->data), out->rows, out->stride, out->cols, boundsOf<I>(dout));
      ok = launched(who);
    };
    if (bulk) {
      auto launch = [&](auto LOOSE) {
        constexpr bool kLoose = LOOSE.value;
        const auto kernel = accumulate ? nmb_take_rows_grad<I, O, wide, true, true, kLoose>
                                       : nmb_take_rows_grad<I, O, wide, false, true, kLoose>;
        const size_t shared = (size_t)2 * kTurnRows * fetched_bytes<kLoose, I>(slab); // 33 KB at most
        go(kernel, (slab / wide + 31) / 32 * 32, shared);
      };
      if (loose)
        launch(std::true_type());
      else
        launch(std::false_type());
      return;
    }
    withElems<wide>(v, [&](auto V) {
      go(accumulate ? nmb_take_rows_grad<I, O, V.value, true, false, false>
                    : nmb_take_rows_grad<I, O, V.value, false, false, false>,
         kThreads, 0);
    });
  });
  return ok ? 0 : 1;
}

namespace {
// Calls f(U(), V constant, accesses per row) for copying rows of x to out.
template <typename F> void withCopy(const GPUXRows *x, const GPUXRows *out, F &&f) {
  auto go = [&](auto u) {
    using U = decltype(u);
    const int v = accessElems(x->cols, mostElems<U>(), {x, out});
    withElems<mostElems<U>()>(v, [&](auto V) { f(u, V, x->cols / v); });
  };
  if (elemBytes(x->type) == 2)
    go(uint16_t());
  else if (elemBytes(x->type) == 4)
    go(uint32_t());
  else
    go(uint64_t());
}
} // namespace

namespace {
// `behind`: right behind the sort that makes the places, nothing in between.
int dispatchRows(const Waits &waits, const Stream &s, const GPUXRows *x, int64_t k, const int32_t *place,
                 const int32_t *kept, const GPUXRows *out, bool behind) {
  if (x->rows == 0 || x->cols == 0 || k == 0 || out->rows == 0)
    return 0;
  withCopy(x, out, [&](auto u, auto V, int64_t vecs) {
    using U = decltype(u);
    const int64_t slabs = (x->cols * (int64_t)sizeof(U) + kCopyBytes - 1) / kCopyBytes;
    if (V.value < mostElems<U>() && x->cols * (int64_t)sizeof(U) >= kBulkLeast && slabs <= 65535) {
      const int slab = (int)((x->cols + slabs - 1) / slabs);
      const dim3 grid((unsigned)x->rows, (unsigned)slabs);
      const size_t shared = (size_t)fetched_bytes<true, U>(slab);
      const U *from = static_cast<const U *>(x->data);
      U *to = static_cast<U *>(out->data);
      nmb::rows::launchBehind(nmb_dispatch_rows_bulk<U>, grid, kCopyThreads, shared, s.stream, behind, from, x->stride,
                              k, place, kept, to, out->rows, out->stride, x->cols, slab, boundsOf<U>(x), waits);
      return;
    }
    const int bits = laneBits(vecs, kThreadBits);
    nmb::rows::launchBehind(nmb_dispatch_rows<U, V.value>, blocksFor(x->rows, bits), kThreads, 0, s.stream, behind,
                            static_cast<const U *>(x->data), x->rows, x->stride, k, place, kept,
                            static_cast<U *>(out->data), out->rows, out->stride, vecs, bits);
  });
  return launched("dispatch_rows") ? 0 : 1;
}
} // namespace

GPUX_EXPORT int _mlir_ciface_nmb_dispatch_rows_device(void *queue, const GPUXRows *x, int64_t k, const int32_t *place,
                                                      const int32_t *kept, const GPUXRows *out) {
  const char *who = "dispatch_rows";
  if (!checkRows(who, "x", x, false) || !checkRows(who, "out", out, true) || !sameType(who, x, out) ||
      !sameWidth(who, x, out) || !checkPlaces(who, x->rows, k, place, kept) || !gridFits(who, x->rows))
    return 1;
  Stream s(queue);
  if (!s.ok)
    return 1;
  const Waits waits = waitsOf(queue);
  return waits.status ? dispatchRows(waits, s, x, k, place, kept, out, false) : 1;
}

GPUX_EXPORT int _mlir_ciface_nmb_sort_dispatch_rows_device(void *queue, const GPUXRows *x, const GPUXIndex *ids,
                                                           int64_t groups, int32_t *order, int32_t *place,
                                                           int32_t *offsets, void *workspace, size_t workspaceBytes,
                                                           const GPUXRows *out) {
  const char *who = "dispatch_rows";
  if (!checkRows(who, "x", x, false) || !checkIndex(who, ids) || !checkRows(who, "out", out, true) ||
      !sameType(who, x, out) || !sameWidth(who, x, out) || !gridFits(who, x->rows))
    return 1;
  const int64_t k = x->rows > 0 ? ids->count / x->rows : 0;
  if (ids->count != k * x->rows || out->rows < ids->count) {
    nmb::setError("%s: %lld entries and %lld rows for %lld tokens", who, (long long)ids->count, (long long)out->rows,
                  (long long)x->rows);
    return 1;
  }
  if (!nmb::rows::checkGroups(who, ids, groups, order, place, offsets))
    return 1;
  if (ids->count > 0 && ids->count <= kCountEntries && groups <= kCountGroups && x->cols > 0 &&
      k <= kCountChoices && x->rows * ids->count <= kCountWork) {
    Stream s(queue);
    if (!s.ok)
      return 1;
    withCopy(x, out, [&](auto u, auto V, int64_t vecs) {
      using U = decltype(u);
      nmb_sort_dispatch_rows<U, V.value><<<(unsigned)x->rows, kThreads, 0, s.stream>>>(
          static_cast<const U *>(x->data), x->stride, (int)k, ids->data, ids->bytes, (int)ids->count, (int)groups,
          order, place, offsets, static_cast<U *>(out->data), out->stride, vecs);
    });
    return launched(who) ? 0 : 1;
  }
  Stream s(queue);
  if (!s.ok)
    return 1;
  const Waits waits = waitsOf(queue);
  if (!waits.status)
    return 1;
  nmb::rows::Workspace ws(s, who, workspace, workspaceBytes, nmb::rows::sortBytes(ids->count, groups));
  if (!ws.ok || !nmb::rows::sortByKey(s, who, *ids, groups, order, nullptr, place, offsets, ws.data))
    return 1;
  // groups of several passes end with a kernel that lets nothing begin early
  return dispatchRows(waits, s, x, k, place, offsets + groups, out, ids->count > 0);
}

GPUX_EXPORT int _mlir_ciface_nmb_combine_rows_device(void *queue, const GPUXRows *ys, int64_t k, const int32_t *place,
                                                     const int32_t *kept, const void *weights, int weightType,
                                                     const GPUXRows *out) {
  const char *who = "combine_rows";
  if (!checkRows(who, "ys", ys, false) || !checkRows(who, "out", out, true) || !sameType(who, ys, out) ||
      !sameWidth(who, ys, out) || !checkPlaces(who, out->rows, k, place, kept) ||
      !checkWeights(who, weights, weightType) || !gridFits(who, out->rows))
    return 1;
  if (out->rows == 0 || out->cols == 0)
    return 0;
  Stream s(queue);
  if (!s.ok)
    return 1;
  const Waits waits = waitsOf(queue);
  if (!waits.status)
    return 1;
  withType(ys->type, [&](auto e) {
    using T = decltype(e);
    const int v = accessElems(out->cols, mostElems<T>(), {ys, out});
    const int64_t vecs = out->cols / v;
    const int bits = laneBits(vecs, kThreadBits);
    const bool loose = v < mostElems<T>();
    if (const int slab = bulkSlab(out->cols, out->type, loose, k, (int)k, kBulkBytes)) {
      const auto kernel = loose ? nmb_combine_rows_bulk<T, true> : nmb_combine_rows_bulk<T, false>;
      const int64_t bytes = k * (loose ? fetched_bytes<true, T>(slab) : fetched_bytes<false, T>(slab));
      const int many = slab >= out->cols ? bulkTokens(out->rows, bytes, k, kBulkBytes) : 0;
      const dim3 grid((unsigned)((out->rows + (1 << many) - 1) >> many), (unsigned)((out->cols + slab - 1) / slab));
      kernel<<<grid, kBulkThreads, (size_t)(bytes << many), s.stream>>>(
          static_cast<const T *>(ys->data), ys->rows, ys->stride, (int)k, place, kept, weights, weightType,
          static_cast<T *>(out->data), out->rows, out->stride, out->cols, slab, many, boundsOf<T>(ys), waits);
      return;
    }
    withElems<mostElems<T>()>(v, [&](auto V) {
      nmb_combine_rows<T, V.value><<<blocksFor(out->rows, bits), kThreads, 0, s.stream>>>(
          static_cast<const T *>(ys->data), ys->rows, ys->stride, k, place, kept, weights, weightType,
          static_cast<T *>(out->data), out->rows, out->stride, vecs, bits);
    });
  });
  return launched(who) ? 0 : 1;
}

GPUX_EXPORT int _mlir_ciface_nmb_combine_rows_grad_device(void *queue, const GPUXRows *dout, const GPUXRows *ys,
                                                          int64_t k, const int32_t *place, const int32_t *kept,
                                                          const void *weights, int weightType, const GPUXRows *dys,
                                                          void *dweights) {
  const char *who = "combine_rows_grad";
  if (!checkRows(who, "dout", dout, false) || !checkRows(who, "ys", ys, false) || !checkRows(who, "dys", dys, true) ||
      !sameType(who, dout, ys) || !sameType(who, dout, dys) || !sameWidth(who, dout, ys) ||
      !sameWidth(who, dout, dys) || !checkPlaces(who, dout->rows, k, place, kept) ||
      !checkWeights(who, weights, weightType) || !checkWeights(who, dweights, weightType) ||
      !gridFits(who, dout->rows))
    return 1;
  if (dout->rows == 0 || k == 0)
    return 0;
  Stream s(queue);
  if (!s.ok)
    return 1;
  const Waits waits = waitsOf(queue);
  if (!waits.status)
    return 1;
  withType(ys->type, [&](auto e) {
    using T = decltype(e);
    const int v = dout->cols ? accessElems(dout->cols, mostElems<T>(), {dout, ys, dys}) : 1;
    const int64_t vecs = dout->cols / v;
    const int bits = laneBits(vecs, kThreadBits);
    const bool loose = v < mostElems<T>();
    if (const int slab = bulkSlab(dout->cols, dout->type, loose, k, (int)k + 1, kBulkGradBytes)) {
      const auto kernel = loose ? nmb_combine_rows_grad_bulk<T, true> : nmb_combine_rows_grad_bulk<T, false>;
      const int64_t bytes = (k + 1) * (loose ? fetched_bytes<true, T>(slab) : fetched_bytes<false, T>(slab));
      // Off the words, where blocks have more to compute, half the memory and more
      // blocks: 30000 tokens with eight rows of 1027 bf16 271 us, 313 us with all
      // of it.  On them 164 us (rows of 1024) with all, 166 us with half.
      const int many = slab >= dout->cols ? bulkTokens(dout->rows, bytes, k, kBulkGradBytes / (loose ? 2 : 1)) : 0;
      kernel<<<(unsigned)((dout->rows + (1 << many) - 1) >> many), kBulkThreads, (size_t)(bytes << many), s.stream>>>(
          static_cast<const T *>(dout->data), dout->rows, dout->stride, static_cast<const T *>(ys->data), ys->rows,
          ys->stride, (int)k, place, kept, weights, weightType, static_cast<T *>(dys->data), dys->rows, dys->stride,
          dweights, dout->cols, slab, many, boundsOf<T>(dout), boundsOf<T>(ys), waits);
      return;
    }
    withElems<mostElems<T>()>(v, [&](auto V) {
      const auto kernel = k <= 2 ? nmb_combine_rows_grad<T, V.value, 2> : nmb_combine_rows_grad<T, V.value, 4>;
      kernel<<<blocksFor(dout->rows, bits), kThreads, 0, s.stream>>>(
          static_cast<const T *>(dout->data), dout->rows, dout->stride, static_cast<const T *>(ys->data), ys->rows,
          ys->stride, k, place, kept, weights, weightType, static_cast<T *>(dys->data), dys->rows, dys->stride,
          dweights, vecs, bits);
    });
  });
  return launched(who) ? 0 : 1;
}
