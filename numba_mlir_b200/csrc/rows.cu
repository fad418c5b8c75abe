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
// A row is shared by a power of two of a block's threads (`lanes`), each thread
// moves `V` neighbouring elements per access (16 bytes where alignment and
// width allow), and blocks take several short rows or one long one.  Arithmetic
// is float32 (float64 for float64 rows) and rounds once, on the way out.
#include "rows_host.h"

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

// ------------------------------------------------------------------- take ---
template <typename I, typename O, int V>
__global__ void __launch_bounds__(kThreads)
    nmb_take_rows(const I *__restrict__ table, int64_t rows, int64_t stride, const void *__restrict__ ids, int id_bytes,
                  int64_t n, typename Acc<I>::type scale, O *__restrict__ out, int64_t out_stride, int64_t vecs,
                  int lane_bits) {
  using A = typename Acc<I>::type;
  const int lane = threadIdx.x & ((1 << lane_bits) - 1);
  const int64_t i = (int64_t)blockIdx.x * (kThreads >> lane_bits) + (threadIdx.x >> lane_bits);
  if (i >= n)
    return;
  const int64_t id = index_at(ids, id_bytes, i);
  const bool inside = id >= 0 && id < rows;
  const I *src = table + (inside ? id : 0) * stride;
  O *dst = out + i * out_stride;
#pragma unroll 4
  for (int64_t c = lane; c < vecs; c += 1 << lane_bits) {
    Pack<O, V> y;
    if (inside) {
      const Pack<I, V> x = load<I, V>(src + c * V);
#pragma unroll
      for (int e = 0; e < V; ++e)
        y.v[e] = down<O, A>(up(x.v[e]) * scale);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        y.v[e] = down<O, A>(A(0));
    }
    store<O, V>(dst + c * V, y);
  }
}

// -------------------------------------------------------------- take_grad ---
// The entries arrive sorted by row (order, keys), so a row's entries are
// neighbours: the threads of a row find them with a binary search and add them
// up in order.  A row without entries becomes zero.
__device__ __forceinline__ int64_t lower_bound(const uint32_t *keys, int64_t n, uint32_t key) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (keys[mid] < key)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

template <typename I, typename O, int V>
__global__ void __launch_bounds__(kThreads)
    nmb_take_rows_grad(const I *__restrict__ dout, int64_t stride, const int32_t *__restrict__ order,
                       const uint32_t *__restrict__ keys, int64_t n, typename Acc<I>::type scale, O *out, int64_t rows,
                       int64_t out_stride, int accumulate, int64_t vecs, int lane_bits) {
  using A = typename Acc<I>::type;
  const int lane = threadIdx.x & ((1 << lane_bits) - 1);
  const int64_t v = (int64_t)blockIdx.x * (kThreads >> lane_bits) + (threadIdx.x >> lane_bits);
  if (v >= rows)
    return;
  const int64_t begin = lower_bound(keys, n, (uint32_t)v);
  O *dst = out + v * out_stride;
  if (accumulate && (begin >= n || keys[begin] != (uint32_t)v))
    return;
  for (int64_t c = lane; c < vecs; c += 1 << lane_bits) {
    A sum[V] = {};
    for (int64_t j = begin; j < n && keys[j] == (uint32_t)v; ++j) {
      const Pack<I, V> x = load<I, V>(dout + (int64_t)order[j] * stride + c * V);
#pragma unroll
      for (int e = 0; e < V; ++e)
        sum[e] += up(x.v[e]);
    }
    Pack<O, V> y;
    if (accumulate) {
      y = load<O, V>(dst + c * V);
#pragma unroll
      for (int e = 0; e < V; ++e)
        y.v[e] = down<O, A>(madd(scale, sum[e], up(y.v[e])));
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        y.v[e] = down<O, A>(scale * sum[e]);
    }
    store<O, V>(dst + c * V, y);
  }
}

// --------------------------------------------------------------- dispatch ---
// Bytes are copied, whatever they mean: U is an unsigned integer of an
// element's size.  A token's row is read once and written k times.
template <typename U, int V>
__global__ void __launch_bounds__(kThreads)
    nmb_dispatch_rows(const U *__restrict__ x, int64_t tokens, int64_t stride, int64_t k,
                      const int32_t *__restrict__ place, const int32_t *__restrict__ kept, U *__restrict__ out,
                      int64_t out_rows, int64_t out_stride, int64_t vecs, int lane_bits) {
  const int lane = threadIdx.x & ((1 << lane_bits) - 1);
  const int64_t t = (int64_t)blockIdx.x * (kThreads >> lane_bits) + (threadIdx.x >> lane_bits);
  if (t >= tokens)
    return;
  const int64_t live = *kept;
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

// ----------------------------------------------------------- combine_grad ---
// The threads of a token go over its choices one by one; the products of a
// choice meet in a fixed tree (shuffles, then the warps in order).
template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
    nmb_combine_rows_grad(const T *__restrict__ dout, int64_t tokens, int64_t stride, const T *__restrict__ ys,
                          int64_t y_rows, int64_t y_stride, int64_t k, const int32_t *__restrict__ place,
                          const int32_t *__restrict__ kept, const void *weights, int weight_type, T *__restrict__ dys,
                          int64_t dy_rows, int64_t dy_stride, void *dweights, int64_t vecs, int lane_bits) {
  using A = typename Acc<T>::type;
  __shared__ A parts[kThreads / 32];
  const int lanes = 1 << lane_bits;
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t t = (int64_t)blockIdx.x * (kThreads >> lane_bits) + (threadIdx.x >> lane_bits);
  const bool token = t < tokens; // every thread stays for the barriers
  const int64_t live = min((int64_t)*kept, y_rows);
  for (int64_t j = 0; j < k; ++j) {
    const int64_t at = token ? place[t * k + j] : -1;
    const bool inside = at >= 0 && at < live;
    const A w = inside ? (weights ? scalar_at<A>(weights, weight_type, t * k + j) : A(1)) : A(0);
    A dot = A(0);
    if (at >= 0 && at < dy_rows) {
      for (int64_t c = lane; c < vecs; c += lanes) {
        Pack<T, V> r{};
        if (inside) {
          const Pack<T, V> d = load<T, V>(dout + t * stride + c * V);
          const Pack<T, V> y = load<T, V>(ys + at * y_stride + c * V);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            dot = madd(up(d.v[e]), up(y.v[e]), dot);
            r.v[e] = down<T, A>(w * up(d.v[e]));
          }
        }
        store<T, V>(dys + at * dy_stride + c * V, r);
      }
    }
    for (int s = min(lanes, 32) / 2; s > 0; s >>= 1)
      dot += __shfl_xor_sync(kAll, dot, s);
    if (lanes > 32) {
      if ((threadIdx.x & 31) == 0)
        parts[threadIdx.x >> 5] = dot;
      __syncthreads();
      if (lane == 0) {
        dot = A(0);
        for (int i = 0; i < lanes / 32; ++i)
          dot += parts[(threadIdx.x >> 5) + i];
      }
      __syncthreads();
    }
    if (token && lane == 0 && dweights)
      set_scalar<A>(dweights, weight_type, t * k + j, dot);
  }
}

// ------------------------------------------------------------------- host ---
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
  withPair(table->type, out->type, [&](auto i, auto o) {
    using I = decltype(i);
    using O = decltype(o);
    constexpr int most = mostElems<I>() > mostElems<O>() ? mostElems<I>() : mostElems<O>();
    const int v = accessElems(out->cols, most, {table, out});
    const int64_t vecs = out->cols / v;
    const int bits = laneBits(vecs, kThreadBits);
    withElems<most>(v, [&](auto V) {
      nmb_take_rows<I, O, V.value><<<blocksFor(out->rows, bits), kThreads, 0, s.stream>>>(
          static_cast<const I *>(table->data), table->rows, table->stride, ids->data, ids->bytes, ids->count,
          (typename Acc<I>::type)scale, static_cast<O *>(out->data), out->stride, vecs, bits);
    });
  });
  return launched(who) ? 0 : 1;
}

GPUX_EXPORT size_t _mlir_ciface_nmb_take_rows_grad_workspace(int64_t count, int64_t rows, int64_t cols, int type) {
  (void)cols;
  (void)type;
  return count < 0 ? 0 : 2 * padded((size_t)count * 4) + nmb::rows::sortBytes(count, rows);
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
  if (out->rows == 0 || out->cols == 0)
    return 0;
  Stream s(queue);
  if (!s.ok)
    return 1;
  nmb::rows::Workspace memory(
      s, who, workspace, workspaceBytes,
      _mlir_ciface_nmb_take_rows_grad_workspace(ids->count, out->rows, out->cols, dout->type));
  if (!memory.ok)
    return 1;
  const size_t entries = padded((size_t)ids->count * 4);
  unsigned char *ws = static_cast<unsigned char *>(memory.data);
  int32_t *order = reinterpret_cast<int32_t *>(ws);
  uint32_t *keys = reinterpret_cast<uint32_t *>(ws + entries);
  if (!nmb::rows::sortByKey(s, who, *ids, out->rows, order, keys, nullptr, nullptr, ws + 2 * entries))
    return 1;
  withPair(dout->type, out->type, [&](auto i, auto o) {
    using I = decltype(i);
    using O = decltype(o);
    constexpr int most = mostElems<I>() > mostElems<O>() ? mostElems<I>() : mostElems<O>();
    const int v = accessElems(out->cols, most, {dout, out});
    const int64_t vecs = out->cols / v;
    const int bits = laneBits(vecs, kThreadBits);
    withElems<most>(v, [&](auto V) {
      nmb_take_rows_grad<I, O, V.value><<<blocksFor(out->rows, bits), kThreads, 0, s.stream>>>(
          static_cast<const I *>(dout->data), dout->stride, order, keys, ids->count, (typename Acc<I>::type)scale,
          static_cast<O *>(out->data), out->rows, out->stride, accumulate, vecs, bits);
    });
  });
  return launched(who) ? 0 : 1;
}

GPUX_EXPORT int _mlir_ciface_nmb_dispatch_rows_device(void *queue, const GPUXRows *x, int64_t k, const int32_t *place,
                                                      const int32_t *kept, const GPUXRows *out) {
  const char *who = "dispatch_rows";
  if (!checkRows(who, "x", x, false) || !checkRows(who, "out", out, true) || !sameType(who, x, out) ||
      !sameWidth(who, x, out) || !checkPlaces(who, x->rows, k, place, kept) || !gridFits(who, x->rows))
    return 1;
  if (x->rows == 0 || x->cols == 0 || k == 0 || out->rows == 0)
    return 0;
  Stream s(queue);
  if (!s.ok)
    return 1;
  auto go = [&](auto u) {
    using U = decltype(u);
    const int v = accessElems(x->cols, mostElems<U>(), {x, out});
    const int64_t vecs = x->cols / v;
    const int bits = laneBits(vecs, kThreadBits);
    withElems<mostElems<U>()>(v, [&](auto V) {
      nmb_dispatch_rows<U, V.value><<<blocksFor(x->rows, bits), kThreads, 0, s.stream>>>(
          static_cast<const U *>(x->data), x->rows, x->stride, k, place, kept, static_cast<U *>(out->data), out->rows,
          out->stride, vecs, bits);
    });
  };
  if (elemBytes(x->type) == 2)
    go(uint16_t());
  else if (elemBytes(x->type) == 4)
    go(uint32_t());
  else
    go(uint64_t());
  return launched(who) ? 0 : 1;
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
  withType(ys->type, [&](auto e) {
    using T = decltype(e);
    const int v = accessElems(out->cols, mostElems<T>(), {ys, out});
    const int64_t vecs = out->cols / v;
    const int bits = laneBits(vecs, kThreadBits);
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
  withType(ys->type, [&](auto e) {
    using T = decltype(e);
    const int v = dout->cols ? accessElems(dout->cols, mostElems<T>(), {dout, ys, dys}) : 1;
    const int64_t vecs = dout->cols / v;
    const int bits = laneBits(vecs, kThreadBits);
    withElems<mostElems<T>()>(v, [&](auto V) {
      nmb_combine_rows_grad<T, V.value><<<blocksFor(dout->rows, bits), kThreads, 0, s.stream>>>(
          static_cast<const T *>(dout->data), dout->rows, dout->stride, static_cast<const T *>(ys->data), ys->rows,
          ys->stride, k, place, kept, weights, weightType, static_cast<T *>(dys->data), dys->rows, dys->stride,
          dweights, vecs, bits);
    });
  });
  return launched(who) ? 0 : 1;
}
