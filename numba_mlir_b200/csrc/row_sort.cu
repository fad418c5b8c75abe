// Entries sorted by group: the stable order of the row operators (rows.cu).
//
// A least-significant-digit radix sort of (key, entry) pairs, key = id for an
// id inside [0, groups) and `groups` for every other one, over
// bits(groups) bits in the fewest passes of at most 10 bits each: one pass up
// to 1023 groups (experts), two up to a million (a vocabulary).  Nothing
// depends on the order in which blocks or atomics run: a block counts its own
// entries, counts are added up in block order, and the rank of an entry among
// the equal digits of its warp's 32 comes from a match over the warp.
//
// What it costs is latency, not bandwidth (an entry is 8 bytes).  Up to 8192
// entries stay in one block's shared memory for all passes: one launch.  More
// take three launches a pass: blocks count tiles of 4096 entries, a warp per
// digit adds the counts up over the blocks, blocks scatter their tiles.
#include "rows_host.h"

#include <atomic>

#define GPUX_EXPORT extern "C" __attribute__((visibility("default")))

namespace {

constexpr int kMaxDigitBits = 10;
constexpr int kBins = 1 << kMaxDigitBits;
constexpr unsigned kAll = 0xffffffffu;

struct Ids {
  const void *data;
  int bytes;
  uint32_t groups;
  __device__ __forceinline__ uint32_t key(int64_t i) const {
    const int64_t id = bytes == 8 ? __ldg(static_cast<const long long *>(data) + i)
                                  : (int64_t)__ldg(static_cast<const int *>(data) + i);
    return id >= 0 && id < (int64_t)groups ? (uint32_t)id : groups;
  }
};

// Rank of this lane's digit among the equal digits of the lanes before it, and
// the running count of that digit in `count` (one word per digit, this warp's
// own): the first lane of each set of equals adds the set's size.
__device__ __forceinline__ uint32_t warp_rank(uint32_t digit, bool live, uint32_t *count) {
  const int lane = threadIdx.x & 31;
  const unsigned peers = __match_any_sync(kAll, live ? digit : 0xffffffffu);
  const int first = __ffs(peers) - 1;
  uint32_t base = 0;
  if (live && lane == first) {
    base = count[digit];
    count[digit] = base + __popc(peers);
  }
  base = __shfl_sync(kAll, base, first);
  return base + __popc(peers & ((1u << lane) - 1));
}

// Exclusive prefix of v over the block's threads (blockDim.x a multiple of 32);
// `sums` holds 32 words.
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t *sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint32_t inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t t = __shfl_up_sync(kAll, inc, d);
    if (lane >= d)
      inc += t;
  }
  if (lane == 31)
    sums[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const uint32_t mine = lane < warps ? sums[lane] : 0;
    uint32_t s = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t t = __shfl_up_sync(kAll, s, d);
      if (lane >= d)
        s += t;
    }
    sums[lane] = s - mine;
  }
  __syncthreads();
  const uint32_t before = sums[warp] + inc - v;
  __syncthreads();
  return before;
}

// ---- one block ----------------------------------------------------------------
constexpr int kOneThreads = 1024;
constexpr int kOnePerThread = 8;
constexpr int kOneMax = kOneThreads * kOnePerThread;
constexpr int kOneSmem = (32 * kBins + 2 * kOneMax + 32 + 1) * 4; // counts, keys, entries, prefix sums, total

struct Results {
  int32_t *order;
  uint32_t *keys;
  int32_t *place;
  int32_t *offsets;
};

// Words of the caller's that the first kernel sets to zero.
struct Clear {
  uint32_t *words;
  int64_t count;
  __device__ __forceinline__ void run() const {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += (int64_t)gridDim.x * blockDim.x)
      words[i] = 0;
  }
};

__global__ void __launch_bounds__(kOneThreads)
    nmb_sort_one(const Ids ids, int n, int bits, int passes, const Results res, const Clear clear) {
  clear.run();
  extern __shared__ uint32_t smem[];
  uint32_t *counts = smem;                 // [warps][bins]
  uint32_t *keys = smem + 32 * kBins;      // [n]
  uint32_t *entries = keys + kOneMax;      // [n]
  uint32_t *sums = entries + kOneMax;      // [32]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int warps = blockDim.x >> 5;
  const int digit_bits = (bits + passes - 1) / passes, bins = 1 << digit_bits;
  // a warp owns a contiguous run of `span` entries, 32 at a time
  const int span = ((n + warps - 1) / warps + 31) / 32 * 32;
  const int begin = warp * span;

  for (int i = tid; i < n; i += blockDim.x) {
    keys[i] = ids.key(i);
    entries[i] = i;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digit_bits;
    for (int i = tid; i < warps * bins; i += blockDim.x)
      counts[i] = 0;
    __syncthreads();
    uint32_t key[kOnePerThread], entry[kOnePerThread], rank[kOnePerThread];
#pragma unroll
    for (int u = 0; u < kOnePerThread; ++u) {
      const int i = begin + u * 32 + lane;
      if (u * 32 < span) { // the same for all lanes
        const bool live = i < n;
        key[u] = live ? keys[i] : 0;
        entry[u] = live ? entries[i] : 0;
        rank[u] = warp_rank((key[u] >> shift) & (bins - 1), live, counts + warp * bins);
        __syncwarp();
      }
    }
    __syncthreads();
    // counts[w][d] <- entries of digit d in the warps before w; the digits'
    // totals go through a prefix over the block, up to `per` digits a thread
    const int per = (bins + blockDim.x - 1) / blockDim.x;
    uint32_t total = 0;
    for (int b = tid * per; b < min((tid + 1) * per, bins); ++b) {
      for (int w = 0; w < warps; ++w) {
        const uint32_t c = counts[w * bins + b];
        counts[w * bins + b] = total;
        total += c;
      }
    }
    const uint32_t before = block_prefix(total, sums);
    for (int b = tid * per; b < min((tid + 1) * per, bins); ++b) {
      for (int w = 0; w < warps; ++w)
        counts[w * bins + b] += before;
      if (passes == 1 && res.offsets && b <= (int)ids.groups)
        res.offsets[b] = (int32_t)counts[b];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kOnePerThread; ++u) {
      const int i = begin + u * 32 + lane;
      if (u * 32 < span && i < n) {
        const uint32_t at = counts[warp * bins + ((key[u] >> shift) & (bins - 1))] + rank[u];
        keys[at] = key[u];
        entries[at] = entry[u];
      }
    }
    __syncthreads();
  }
  for (int i = tid; i < n; i += blockDim.x) {
    const uint32_t e = entries[i];
    if (res.order)
      res.order[i] = (int32_t)e;
    if (res.keys)
      res.keys[i] = keys[i];
    if (res.place)
      res.place[e] = i;
  }
}

// ---- many blocks --------------------------------------------------------------
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPerThread = 16;
constexpr int kTile = kThreads * kPerThread;

struct Pass {
  Ids ids;                 // the first pass reads its keys here (keysIn == nullptr)
  const uint32_t *keysIn;
  const int32_t *entriesIn;
  uint32_t *counts;        // [bins][blocks]
  uint32_t *totals;        // [bins]
  int64_t n;
  int blocks, shift, bins;
  __device__ __forceinline__ uint32_t key(int64_t i) const { return keysIn ? keysIn[i] : ids.key(i); }
  __device__ __forceinline__ uint32_t digit(uint32_t k) const { return (k >> shift) & (uint32_t)(bins - 1); }
};

__global__ void __launch_bounds__(kThreads) nmb_sort_count(const Pass p, const Clear clear) {
  clear.run();
  __shared__ uint32_t count[kBins];
  for (int b = threadIdx.x; b < p.bins; b += kThreads)
    count[b] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kTile;
#pragma unroll 4
  for (int u = 0; u < kPerThread; ++u) {
    const int64_t i = base + u * kThreads + threadIdx.x;
    if (i < p.n)
      atomicAdd(&count[p.digit(p.key(i))], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < p.bins; b += kThreads)
    p.counts[(int64_t)b * p.blocks + blockIdx.x] = count[b];
}

// A warp per digit: counts[d][b] <- sum of counts[d][0..b), totals[d] <- the sum.
__global__ void __launch_bounds__(kThreads) nmb_sort_prefix(uint32_t *counts, uint32_t *totals, int blocks, int bins) {
  const int lane = threadIdx.x & 31;
  const int d = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (d >= bins)
    return;
  uint32_t *row = counts + (int64_t)d * blocks;
  uint32_t carry = 0;
  for (int b0 = 0; b0 < blocks; b0 += 32) {
    const int b = b0 + lane;
    const uint32_t v = b < blocks ? row[b] : 0;
    uint32_t inc = v;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const uint32_t t = __shfl_up_sync(kAll, inc, s);
      if (lane >= s)
        inc += t;
    }
    if (b < blocks)
      row[b] = carry + inc - v;
    carry += __shfl_sync(kAll, inc, 31);
  }
  if (lane == 0)
    totals[d] = carry;
}

__global__ void __launch_bounds__(kThreads)
    nmb_sort_scatter(const Pass p, uint32_t *keysOut, int32_t *entriesOut, int32_t *place, int32_t *offsets) {
  __shared__ uint32_t counts[kWarps][kBins];
  __shared__ uint32_t start[kBins];
  __shared__ uint32_t sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kWarps * kBins; i += kThreads)
    (&counts[0][0])[i] = 0;
  // where each digit's entries begin in the output: prefix of the totals
  {
    constexpr int kPer = kBins / kThreads;
    uint32_t mine[kPer], sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int d = threadIdx.x * kPer + j;
      mine[j] = sum;
      sum += d < p.bins ? p.totals[d] : 0;
    }
    const uint32_t before = block_prefix(sum, sums);
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      start[threadIdx.x * kPer + j] = before + mine[j];
  }
  __syncthreads();
  if (offsets && blockIdx.x == 0)
    for (int d = threadIdx.x; d <= (int)p.ids.groups; d += kThreads)
      offsets[d] = (int32_t)start[d];
  // a warp owns 512 consecutive entries of the tile, 32 at a time
  const int64_t base = (int64_t)blockIdx.x * kTile + warp * (kTile / kWarps);
  uint32_t key[kPerThread], rank[kPerThread];
#pragma unroll
  for (int u = 0; u < kPerThread; ++u) {
    const int64_t i = base + u * 32 + lane;
    key[u] = i < p.n ? p.key(i) : 0;
  }
#pragma unroll
  for (int u = 0; u < kPerThread; ++u) {
    rank[u] = warp_rank(p.digit(key[u]), base + u * 32 + lane < p.n, counts[warp]);
    __syncwarp();
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.bins; d += kThreads) {
    uint32_t at = start[d] + p.counts[(int64_t)d * p.blocks + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const uint32_t c = counts[w][d];
      counts[w][d] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kPerThread; ++u) {
    const int64_t i = base + u * 32 + lane;
    if (i < p.n) {
      const uint32_t at = counts[warp][p.digit(key[u])] + rank[u];
      const int32_t e = p.entriesIn ? p.entriesIn[i] : (int32_t)i;
      if (keysOut)
        keysOut[at] = key[u];
      if (entriesOut)
        entriesOut[at] = e;
      if (place)
        place[e] = (int32_t)at;
    }
  }
}

// offsets[g] = position of the first key >= g, for the sorts of several passes.
__global__ void __launch_bounds__(kThreads)
    nmb_sort_offsets(const uint32_t *keys, int64_t n, int64_t groups, int32_t *offsets) {
  const int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (g > groups)
    return;
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (keys[mid] < (uint32_t)g)
      lo = mid + 1;
    else
      hi = mid;
  }
  offsets[g] = (int32_t)lo;
}

__global__ void __launch_bounds__(kThreads) nmb_sort_nothing(int64_t groups, int32_t *offsets) {
  const int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (g <= groups)
    offsets[g] = 0;
}

int bitsOf(int64_t groups) {
  int b = 1;
  while ((int64_t(1) << b) <= groups)
    ++b;
  return b; // keys are 0 .. groups
}

size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }

int64_t tiles(int64_t n) { return (n + kTile - 1) / kTile; }

bool fitsOneBlock(int64_t n) { return n <= kOneMax; }

} // namespace

namespace nmb {
namespace rows {

// Two (key, entry) buffers, the counts and the digits' totals.  A sort of several
// passes whose caller does not ask for the sorted keys keeps them in the first
// buffer, for the offsets.
size_t sortBytes(int64_t count, int64_t groups) {
  const size_t pairs = padded((size_t)count * 4);
  if (fitsOneBlock(count))
    return bitsOf(groups) > kMaxDigitBits ? pairs : 0; // the sorted keys, for the offsets
  return 4 * pairs + padded((size_t)kBins * (size_t)tiles(count) * 4) + padded(kBins * 4);
}

bool sortByKey(const Stream &s, const char *who, const GPUXIndex &ids, int64_t groups, int32_t *order,
               uint32_t *keys, int32_t *place, int32_t *offsets, void *workspace, uint32_t *clear,
               int64_t clearWords) {
  const int64_t n = ids.count;
  const Ids in{ids.data, ids.bytes, (uint32_t)groups};
  const int bits = bitsOf(groups), passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
  const unsigned offsetBlocks = (unsigned)((groups + kThreads) / kThreads);
  if (n == 0) {
    if (!offsets)
      return true;
    nmb_sort_nothing<<<offsetBlocks, kThreads, 0, s.stream>>>(groups, offsets);
    return launched(who);
  }
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  const size_t pairs = padded((size_t)n * 4);
  if (passes > 1 && offsets && !keys)
    keys = reinterpret_cast<uint32_t *>(ws); // the sorted keys, wanted for the offsets below
  if (fitsOneBlock(n)) {
    static std::atomic<bool> ready[64]; // per device; setting it twice is harmless
    if (s.device < 0 || s.device >= 64 || !ready[s.device]) {
      const cudaError_t e =
          cudaFuncSetAttribute(nmb_sort_one, cudaFuncAttributeMaxDynamicSharedMemorySize, kOneSmem);
      if (e != cudaSuccess) {
        setError("%s: cudaFuncSetAttribute failed: %s", who, cudaGetErrorString(e));
        (void)cudaGetLastError();
        return false;
      }
      if (s.device >= 0 && s.device < 64)
        ready[s.device] = true;
    }
    // as many warps as there are rows of 32 entries
    const int warps = (int)(n + 31) / 32 < 32 ? (int)(n + 31) / 32 : 32;
    nmb_sort_one<<<1, warps * 32, kOneSmem, s.stream>>>(in, (int)n, bits, passes,
                                                        Results{order, keys, place, passes == 1 ? offsets : nullptr},
                                                        Clear{clear, clearWords});
    if (!launched(who))
      return false;
  } else {
    const int64_t blocks = tiles(n);
    uint32_t *keyBuf[2] = {reinterpret_cast<uint32_t *>(ws), reinterpret_cast<uint32_t *>(ws + pairs)};
    int32_t *entryBuf[2] = {reinterpret_cast<int32_t *>(ws + 2 * pairs), reinterpret_cast<int32_t *>(ws + 3 * pairs)};
    uint32_t *counts = reinterpret_cast<uint32_t *>(ws + 4 * pairs);
    uint32_t *totals =
        reinterpret_cast<uint32_t *>(ws + 4 * pairs + padded((size_t)kBins * (size_t)blocks * 4));
    const int digitBits = (bits + passes - 1) / passes;
    Pass p{in, nullptr, nullptr, counts, totals, n, (int)blocks, 0, 1 << digitBits};
    for (int pass = 0; pass < passes; ++pass) {
      const bool last = pass + 1 == passes;
      // the passes alternate between the buffers so that the last one may write
      // sorted keys into buffer 0 (see above)
      const int to = (passes - 1 - pass) & 1;
      p.shift = pass * digitBits;
      nmb_sort_count<<<(unsigned)blocks, kThreads, 0, s.stream>>>(p, Clear{clear, pass == 0 ? clearWords : 0});
      if (!launched(who))
        return false;
      nmb_sort_prefix<<<(unsigned)((p.bins + kWarps - 1) / kWarps), kThreads, 0, s.stream>>>(counts, totals,
                                                                                             (int)blocks, p.bins);
      if (!launched(who))
        return false;
      nmb_sort_scatter<<<(unsigned)blocks, kThreads, 0, s.stream>>>(
          p, last ? keys : keyBuf[to], last ? order : entryBuf[to], last ? place : nullptr,
          passes == 1 ? offsets : nullptr);
      if (!launched(who))
        return false;
      p.keysIn = keyBuf[to];
      p.entriesIn = entryBuf[to];
    }
  }
  if (offsets && passes > 1) {
    nmb_sort_offsets<<<offsetBlocks, kThreads, 0, s.stream>>>(keys, n, groups, offsets);
    return launched(who);
  }
  return true;
}

} // namespace rows
} // namespace nmb

GPUX_EXPORT size_t _mlir_ciface_nmb_group_rows_workspace(int64_t count, int64_t groups) {
  return count < 0 ? 0 : nmb::rows::sortBytes(count, groups);
}

GPUX_EXPORT int _mlir_ciface_nmb_group_rows_device(void *queue, const GPUXIndex *ids, int64_t groups, int32_t *order,
                                                   int32_t *place, int32_t *offsets, void *workspace,
                                                   size_t workspaceBytes) {
  const char *who = "group_rows";
  if (!nmb::rows::checkIndex(who, ids))
    return 1;
  if (groups < 0 || groups >= 0x7fffffff) {
    nmb::setError("%s: the number of groups must be in 0 .. 2^31 - 2", who);
    return 1;
  }
  if (!offsets || (ids->count > 0 && (!order || !place))) {
    nmb::setError("%s: null result", who);
    return 1;
  }
  nmb::rows::Stream s(queue);
  if (!s.ok)
    return 1;
  nmb::rows::Workspace ws(s, who, workspace, workspaceBytes, nmb::rows::sortBytes(ids->count, groups));
  if (!ws.ok)
    return 1;
  return nmb::rows::sortByKey(s, who, *ids, groups, order, nullptr, place, offsets, ws.data) ? 0 : 1;
}
